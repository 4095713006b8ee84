"""Attention of sequences to themselves, forward and backward, against float64."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402
import causal_oracle as co      # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def make(dtype, batch, tokens, hq, hk, dim, seed=0, packed=False):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def rand(heads):
        return torch.randn((batch, tokens, heads, dim), generator=gen, device="cuda").to(dtype)

    if packed:
        x = rand(hq + 2 * hk)
        return x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:], rand(hq)
    return rand(hq), rand(hk), rand(hk), rand(hq)


def check(pkg, q, k, v, dout, lengths=None, window=None, sinks=0, scale=None, lse_grad=None):
    A, how = pkg.attention, dict(window=window, sinks=sinks, lengths=lengths, scale=scale)
    scale = scale or float(torch.tensor(1 / math.sqrt(q.shape[-1])))
    read = co.window_read(q.shape[0], q.shape[1], window, sinks, lengths)
    out, lse = A.window_attention(q, k, v, return_lse=True, **how)
    want, want_lse, p = co.attention(q, k, v, read, scale)
    ao.within(out, want, co.bound(q, k, v, want, p, read, scale))
    ao.within(lse, want_lse, co.lse_bound(q, k, read, want_lse, scale))
    assert torch.equal(A.window_attention(q, k, v, **how), out)
    got = A.window_attention_backward(dout, q, k, v, out, lse, lse_grad=lse_grad, **how)
    for x, w, b in zip(got, *co.gradients(q, k, v, dout, read, scale, lse_grad)):
        ao.within(x, w, b)
    again = A.window_attention_backward(dout, q, k, v, out, lse, lse_grad=lse_grad, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    return out, lse, got


SHAPES = [
    # dtype, batch, tokens, q heads, kv heads, dim, window, sinks
    (BF16, 1, 1, 1, 1, 8, None, 0),
    (F16, 2, 2, 2, 1, 64, 1, 0),
    (BF16, 2, 31, 3, 3, 40, 7, 2),
    (F16, 1, 127, 4, 1, 128, None, 0),
    (BF16, 1, 128, 4, 2, 128, 128, 0),
    (F16, 1, 129, 2, 2, 72, 64, 1),
    (BF16, 3, 200, 7, 1, 64, 33, 5),
    (BF16, 1, 257, 8, 2, 96, 128, 130),
    (F16, 2, 300, 6, 6, 80, None, 0),
    (BF16, 1, 640, 4, 4, 128, 129, 4),
    (F16, 1, 700, 14, 2, 64, 250, 16),
    (BF16, 1, 513, 5, 1, 128, 1, 3),
    (BF16, 1, 400, 1, 1, 128, 1000, 7),
    (BF16, 1, 1100, 2, 1, 64, 300, 300),
    (F16, 1, 260, 48, 1, 64, 60, 4),
    (BF16, 1, 65, 130, 1, 32, 20, 1),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("how", ["plain", "packed", "lengths"])
def test_against_float64(pkg, shape, how):
    dtype, batch, tokens, hq, hk, dim, window, sinks = shape
    q, k, v, dout = make(dtype, batch, tokens, hq, hk, dim, seed=tokens, packed=how == "packed")
    lengths = None
    if how == "lengths":
        rng = torch.Generator().manual_seed(tokens)
        lengths = torch.randint(0, tokens + 1, (batch,), generator=rng).to("cuda")
        if batch > 1:
            lengths[0], lengths[-1] = tokens + 5, -3           # taken as the nearest
        for b in range(batch):
            n = max(0, int(lengths[b]))
            for x in (q, k, v, dout):
                x[b, n:] = math.nan                            # whatever lies there
    check(pkg, q, k, v, dout, lengths, window, sinks)


def test_scale_and_gradient_of_lse(pkg):
    q, k, v, dout = make(BF16, 2, 150, 4, 2, 64)
    lse_grad = torch.randn(2, 4, 150, device="cuda")
    lengths = torch.tensor([150, 70], dtype=torch.int32, device="cuda")
    lse_grad[1, :, 70:] = math.nan
    check(pkg, q, k, v, dout, lengths, 40, 3, scale=0.3, lse_grad=lse_grad)


def test_autograd(pkg):
    A = pkg.attention
    q, k, v, dout = make(BF16, 2, 190, 4, 2, 64)
    how = dict(window=50, sinks=2, lengths=torch.tensor([190, 100], device="cuda"))
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    out, lse = A.window_attention(*x, return_lse=True, **how)
    dlse = torch.randn_like(lse)
    dlse[1, :, 100:] = 0
    torch.autograd.backward((out, lse), (dout, dlse))
    want = A.window_attention_backward(dout, q, k, v, out.detach(), lse.detach(), lse_grad=dlse, **how)
    assert all(torch.equal(t.grad, w) for t, w in zip(x, want))
    x[1].grad = None
    A.window_attention(q, x[1], v, **how).backward(dout)
    want = A.window_attention_backward(dout, q, k, v, out.detach(), lse.detach(), **how)
    assert torch.equal(x[1].grad, want[1])
    # keys and values that all batches share
    s = torch.randn(1, 190, 2, 64, device="cuda").to(BF16).requires_grad_()
    A.window_attention(q, s.expand(2, -1, -1, -1), s.expand(2, -1, -1, -1), **how).backward(dout)
    kk = s.detach().expand(2, -1, -1, -1)
    o, l = A.window_attention(q, kk, kk, return_lse=True, **how)
    g = A.window_attention_backward(dout, q, kk, kk, o, l, **how)
    assert torch.allclose(s.grad.float(), (g[1].float() + g[2].float()).sum(0, keepdim=True), rtol=2.0 ** -6, atol=0.05)


def test_gradients_against_differences(pkg):
    """d/dx of sum(out g) along a direction, by central differences of the operator itself in float16."""
    A = pkg.attention
    q, k, v, g = make(F16, 1, 96, 2, 1, 64, seed=5)
    how = dict(window=30, sinks=2)
    out, lse = A.window_attention(q, k, v, return_lse=True, **how)
    grads = A.window_attention_backward(g, q, k, v, out, lse, **how)
    for i, x in enumerate((q, k, v)):
        d = torch.randn_like(x, dtype=torch.float32).to(F16)
        h = 2.0 ** -3                                        # x + h d is rounded, so the step that was taken is worked out
        plus, minus = (x + h * d).clone(), (x - h * d).clone()
        step = (plus.double() - minus.double())
        read = co.window_read(1, 96, 30, 2)
        scale = float(torch.tensor(1 / 8.0))
        args = [[q, k, v], [q, k, v]]
        args[0][i], args[1][i] = plus, minus
        f = [(A.window_attention(*a, **how).double() * g.double()).sum().item() for a in args]
        e = [(co.attention(*a, read, scale)[0] * g.double()).sum().item() for a in args]
        along = (grads[i].double() * step).sum().item()
        # the operator's two values are off by its rounding, the difference from the derivative by the third order; both are measured
        # on the float64 form
        want = (co.gradients(q, k, v, g, read, scale)[0][i] * step).sum().item()
        third = abs((e[0] - e[1]) - want)
        rounding = sum(abs(a - b) for a, b in zip(f, e))
        bound = (co.gradients(q, k, v, g, read, scale)[1][i] * step.abs()).sum().item()
        assert abs((f[0] - f[1]) - along) <= third + rounding + bound
        assert abs(along) > 3 * (third + rounding)           # the comparison says something


def test_rows_that_are_not_numbers_stay_where_they_are(pkg):
    """NaN in a query reaches its own row alone; in a key, the rows that read it."""
    A = pkg.attention
    q, k, v, _ = make(BF16, 1, 300, 2, 2, 64)
    clean = A.window_attention(q, k, v, window=40)
    q2 = q.clone()
    q2[0, 77] = math.nan
    out = A.window_attention(q2, k, v, window=40)
    assert out[0, 77].isnan().all()
    keep = torch.arange(300) != 77
    assert torch.equal(out[0, keep], clean[0, keep])
    k2 = k.clone()
    k2[0, 100] = math.nan
    out, lse = A.window_attention(q, k2, v, window=40, return_lse=True)
    hit = (torch.arange(300) >= 100) & (torch.arange(300) < 140)
    assert out[0, hit].isnan().all() and lse[0, :, hit].isnan().all() and torch.equal(out[0, ~hit], clean[0, ~hit])


def test_far_scores(pkg):
    """Scores that differ by thousands, and rows whose scores are all -infinity."""
    q, k, v, dout = make(BF16, 1, 200, 2, 2, 64)
    check(pkg, q * 30, k * 30, v, dout, None, 64, 1)
    q, k, v, dout = make(F16, 1, 140, 1, 1, 64)
    k[0, :, :, 0] = -math.inf
    q[...] = 0
    q[..., 0] = 1
    out, lse = pkg.attention.window_attention(q, k, v, window=10, return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    got = pkg.attention.window_attention_backward(dout, q, k, v, out, lse, window=10)
    assert not got[2].any()            # no weights


def test_captured_and_on_another_stream(pkg):
    A = pkg.attention
    q, k, v, dout = make(BF16, 1, 300, 4, 2, 128)
    how = dict(window=100, sinks=4)

    def both():
        out, lse = A.window_attention(q, k, v, return_lse=True, **how)
        return [out, lse, *A.window_attention_backward(dout, q, k, v, out, lse, **how)]

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    q.mul_(-1)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, both()))


def test_long_sequence_by_its_parts(pkg):
    """16384 tokens: the rows of some stretches against float64, every gradient of some keys."""
    A = pkg.attention
    n, window, sinks = 16384, 700, 3
    q, k, v, dout = make(BF16, 1, n, 2, 1, 128)
    out, lse = A.window_attention(q, k, v, window=window, sinks=sinks, return_lse=True)
    dq, dk, dv = A.window_attention_backward(dout, q, k, v, out, lse, window=window, sinks=sinks)
    scale = float(torch.tensor(1 / math.sqrt(128)))
    # stretches of queries with all keys they read: their rows and dq; the keys between them that nobody else reads: dk and dv
    for first in (0, 5000, n - 2000):
        rows = torch.arange(first, first + 2000, device="cuda")
        keys = torch.arange(max(0, first - window + 1), first + 2000, device="cuda")
        if first:
            keys = torch.cat((torch.arange(sinks, device="cuda"), keys))
        read = torch.zeros((1, 2000, len(keys)), dtype=torch.bool, device="cuda")
        read[0] = (keys <= rows[:, None]) & ((rows[:, None] - keys < window) | (keys < sinks))
        a = (q[:, rows], k[:, keys], v[:, keys])
        want, want_lse, p = co.attention(*a, read, scale)
        ao.within(out[:, rows], want, co.bound(*a, want, p, read, scale))
        ao.within(lse[:, :, rows], want_lse, co.lse_bound(a[0], a[1], read, want_lse, scale))
        grads, bounds = co.gradients(*a, dout[:, rows], read, scale)
        ao.within(dq[:, rows], grads[0], bounds[0])
        whole = (keys >= (first if first else sinks)) & (keys + window <= first + 2000) if first < n - 2000 else keys >= first
        for x, w, b in ((dk, grads[1], bounds[1]), (dv, grads[2], bounds[2])):
            ao.within(x[:, keys[whole]], w[:, whole], b[:, whole])


def test_refusals(pkg):
    A = pkg.attention
    q, k, v, dout = make(BF16, 2, 10, 4, 2, 64)
    out, lse = A.window_attention(q, k, v, return_lse=True)
    for text, args, how in (
            ("must be .batch, tokens", (q, k[:, :5], v[:, :5]), {}), ("shape of k", (q, k, v[:, :5]), {}),
            ("bfloat16 or float16", (q.float(), k.float(), v.float()), {}), ("type and device", (q, k.half(), v), {}),
            ("multiple of kv_heads", (q[:, :, :3], k, v), {}), ("head_dim", (q[..., :60], k[..., :60], v[..., :60]), {}),
            ("window must be at least 1", (q, k, v), dict(window=0)), ("window must be", (q, k, v), dict(window=2.5)),
            ("sinks must not be negative", (q, k, v), dict(sinks=-1)), ("scale", (q, k, v), dict(scale=0.0)),
            ("scale", (q, k, v), dict(scale=math.nan)), ("lengths must be", (q, k, v), dict(lengths=torch.zeros(3, device="cuda"))),
            ("no CPU path", (q, k.cpu(), v), {}), ("must be a torch tensor", (q, k, None), {})):
        with pytest.raises(ValueError, match=text):
            A.window_attention(*args, **how)
        if len(how) or "tensor" in text:
            with pytest.raises(ValueError, match=text):
                A.window_attention_backward(dout, *args, out, lse, **how)
    for text, change in (("lse must be", dict(lse=lse[:, :2])), ("lse_grad", dict(lse_grad=lse[:1])), ("dout must have", dict(dout=dout[:1])),
                         ("out must have", dict(out=out.float()))):
        a = dict(dout=dout, q=q, k=k, v=v, out=out, lse=lse)
        a.update(change)
        with pytest.raises(ValueError, match=text):
            A.window_attention_backward(**a)
    x = q.clone().requires_grad_()
    with pytest.raises(ValueError, match="scale has no gradient"):
        A.window_attention(x, k, v, scale=torch.tensor(0.1, requires_grad=True))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,window", [(1, None), (1, 5), (700, 1)])
def test_single_keys_have_no_gradient_of_scores(pkg, dtype, tokens, window):
    """A query that reads one key has the weight 1 whatever the score: dq and dk are exactly 0, and a gradient of lse comes through alone."""
    A = pkg.attention
    q, k, v, dout = make(dtype, 3, tokens, 8, 2, 128, seed=2)
    out, lse = A.window_attention(q, k, v, window=window, return_lse=True)
    assert torch.equal(out, v.repeat_interleave(4, 2))
    dq, dk, dv = A.window_attention_backward(dout, q, k, v, out, lse, window=window)
    assert not dq.any() and not dk.any()
    want = dout.double().view(3, tokens, 2, 4, 128)
    ao.within(dv, want.sum(3), co.U[dtype] * 1.01 * want.sum(3).abs() + 8 * co.F32 * want.abs().sum(3) + co.TINY[dtype])
