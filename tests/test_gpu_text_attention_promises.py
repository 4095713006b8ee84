"""What the documents say and other tests do not reach: calls one after another without a wait between them, threads, streams, many
samples, the self-check word."""
import threading

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao                      # noqa: E402
import causal_oracle as co                         # noqa: E402
from test_gpu_cached_attention import check, make, random_tree   # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _generate(A, x, f, prompt, drafts, wait, window, dtype):
    """A prompt, then `drafts` tokens at a time; every call's inputs are made by the calls before it."""
    b, n, heads, dim = x.shape
    hk, page = 2, 16
    hq = heads - 2 * hk
    kp = torch.zeros((b * 20, page, hk, dim), dtype=dtype, device="cuda")
    vp = torch.zeros_like(kp)
    table = torch.arange(b * 20, device="cuda").view(b, 20).to(torch.int32)
    held = torch.zeros(b, dtype=torch.int32, device="cuda")
    outs, at = [], 0
    carry = torch.zeros((b, 1, hq, dim), dtype=dtype, device="cuda")
    while at < n:
        c = min(prompt if at == 0 else drafts, n - at)
        q, k, v = (x[:, at:at + c, s] for s in (slice(0, hq), slice(hq, hq + hk), slice(hq + hk, heads)))
        q = q + carry                                # the next call reads the last one's result
        q = A.append_rotary(q, k, v, None, f, (dim // 2,), kp, vp, table, held)
        out = A.cached_attention(q, kp, vp, table, held, window=window, sinks=2)
        held += c
        carry = out[:, -1:].clone()
        outs.append(out)
        at += c
        if wait:
            torch.cuda.synchronize()
    return torch.cat(outs, 1), kp, vp


@pytest.mark.parametrize("prompt,drafts", [(150, 1), (33, 5), (64, 20), (7, 3)])
@pytest.mark.parametrize("window", [None, 40])
def test_calls_behind_one_another(pkg, prompt, drafts, window):
    """Kernels begin beside the end of those before them: the same bits as with a wait after every step."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    x = torch.randn((2, 240, 12, 128), generator=gen, device="cuda").to(BF16)
    f = 10000.0 ** (-torch.arange(64, device="cuda") / 64)
    want = _generate(pkg.attention, x, f, prompt, drafts, True, window, BF16)
    for _ in range(3):
        got = _generate(pkg.attention, x, f, prompt, drafts, False, window, BF16)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_training_steps_behind_one_another(pkg):
    """Layers whose inputs are the results of the layers before, forward and back, with and without waits."""
    A = pkg.attention
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    x0 = torch.randn((1, 700, 4, 64), generator=gen, device="cuda").to(BF16)

    def run(wait):
        x = x0.clone().requires_grad_()
        y = x
        for i in range(4):
            y = A.window_attention(y, y[:, :, :2], y[:, :, 2:] * 2, window=64 if i % 2 else None, sinks=3)
            if wait:
                torch.cuda.synchronize()
        y.backward(x0)
        if wait:
            torch.cuda.synchronize()
        return y.detach(), x.grad

    want = run(True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(False), want))


def test_two_streams_and_two_threads_at_once(pkg):
    A = pkg.attention
    cases = [make(BF16, 2, 1, 8, 2, 128, 16, [900, 333], seed=i) for i in range(2)]
    long = [tuple(torch.randn((1, 500, h, 64), device="cuda").to(F16) for h in (4, 2, 2)) for _ in range(2)]
    want = [(A.cached_attention(*c), A.window_attention(*w, window=90, return_lse=True)) for c, w in zip(cases, long)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(40):
                    a, (b, lse) = A.cached_attention(*cases[i]), A.window_attention(*long[i], window=90, return_lse=True)
                    g = A.window_attention_backward(b, *long[i], b, lse, window=90)
                torch.cuda.current_stream().synchronize()
            if not (torch.equal(a, want[i][0]) and torch.equal(b, want[i][1][0]) and torch.equal(lse, want[i][1][1]) and torch.isfinite(g[1]).all()):
                bad.append(i)
        except Exception as e:   # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("tokens", [1, 3])
def test_many_samples(pkg, tokens):
    """More samples than the kernel for few rows takes in one grid."""
    rng = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 40, (1100,), generator=rng).tolist()
    check(pkg, *make(F16, 1100, tokens, 4, 2, 64, 8, lengths), window=16, sinks=2)


@pytest.mark.parametrize("tokens", [1, 4, 30])
def test_the_same_pages_for_several_samples(pkg, tokens):
    """Samples that share the pages of a common beginning, and a page that a sample's table names twice."""
    q, kp, vp, table, held = make(BF16, 3, tokens, 8, 2, 64, 16, [64, 64, 64])
    kp, vp = kp.nan_to_num(), vp.nan_to_num()
    table[1, :3] = table[0, :3]
    table[2, 1] = table[2, 0]
    check(pkg, q, kp, vp, table, held)


def test_wide_tables(pkg):
    """A table with room for far more than a sample holds: the work goes by what it holds."""
    q, kp, vp, table, held = make(BF16, 2, 1, 8, 2, 128, 16, [100, 37])
    wide = torch.full((2, 60000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    want = pkg.attention.cached_attention(q, kp, vp, table, held)
    got = pkg.attention.cached_attention(q, kp, vp, wide, held)
    k, v = co.gathered(kp, table), co.gathered(vp, table)
    read = co.cached_read(1, table, kp.shape[0], 16, held)
    scale = float(torch.tensor(128 ** -0.5))
    out, _, p = co.attention(q, k, v, read, scale)
    for x in (want, got):
        ao.within(x, out, co.bound(q, k, v, out, p, read, scale))


def test_strided_queries_and_trees(pkg):
    """q as a view of a joint projection, one that is copied for its alignment, a tree with other strides."""
    q, kp, vp, table, held = make(BF16, 2, 9, 4, 2, 64, 32, [70, 5])
    tree = random_tree(9, 1, 2)
    want = pkg.attention.cached_attention(q, kp, vp, table, held, tree=tree)
    joint = torch.zeros((2, 9, 8, 64), dtype=BF16, device="cuda")
    joint[:, :, 2:6] = q
    assert torch.equal(pkg.attention.cached_attention(joint[:, :, 2:6], kp, vp, table, held, tree=tree), want)
    odd = torch.zeros(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(pkg.attention.cached_attention(odd, kp, vp, table, held, tree=tree.transpose(1, 2).contiguous().transpose(1, 2)), want)
    grown = torch.zeros((2, 12, 11), dtype=torch.bool, device="cuda")
    grown[:, 3:, 1:10] = tree
    assert torch.equal(pkg.attention.cached_attention(q, kp, vp, table, held, tree=grown[:, 3:, 1:10]), want)


def test_self_check_word_is_clean(pkg):
    assert pkg._capi.attention_status(0, torch.cuda.current_stream().cuda_stream) == 0
