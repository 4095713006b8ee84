"""Cross attention against float64 forms: lengths from none to several tiles, masks that leave nothing, garbage where nothing
is read, grouped heads, head sizes, views, gradients against the formulas' and against differences."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
# batch, tokens, keys, q heads, kv heads, head_dim
SHAPES = [
    (1, 1, 1, 1, 1, 8),
    (1, 1, 1601, 32, 8, 128),
    (2, 1, 129, 8, 1, 64),
    (3, 1, 700, 7, 7, 80),
    (2, 2, 300, 12, 2, 96),
    (1, 5, 2050, 16, 2, 128),
    (1, 17, 127, 3, 1, 72),
    (2, 128, 128, 2, 2, 128),
    (1, 129, 255, 4, 2, 128),
    (2, 257, 385, 3, 3, 64),
    (1, 300, 77, 6, 2, 40),
    (1, 64, 4, 2, 1, 16),
    (1, 513, 1025, 2, 1, 128),
    (5, 33, 65, 5, 5, 32),
]


def _inputs(shape, dtype, seed=0, peak=2.0):
    b, t, n, hq, hk, d = shape
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def rand(*s, scale=1.0):
        return (torch.randn(s, generator=gen, device="cuda") * scale).to(dtype)

    return rand(b, t, hq, d, scale=peak), rand(b, n, hk, d), rand(b, n, hk, d), rand(b, t, hq, d)


def _masks(shape, kind, seed=0):
    """(arguments, which keys are read)."""
    b, _, n, *_ = shape
    gen = torch.Generator()
    gen.manual_seed(seed)
    all_read = torch.ones(b, n, dtype=torch.bool, device="cuda")
    if kind == "full":
        return {}, all_read
    lengths = torch.randint(0, n + 1, (b,), generator=gen)
    if kind == "lengths":
        lengths[0] = n // 2
        return dict(lengths=lengths.int().cuda()), torch.arange(n, device="cuda") < lengths.cuda()[:, None]
    mask = (torch.rand(b, n, generator=gen) < 0.6).cuda()
    if kind == "mask":
        return dict(key_mask=mask), mask
    if kind == "both":
        return dict(key_mask=mask, lengths=lengths.cuda()), mask & (torch.arange(n, device="cuda") < lengths.cuda()[:, None])
    assert kind == "nothing"
    mask[b // 2] = False
    return dict(key_mask=mask), mask


def _forward(pkg, q, k, v, args, read, scale=None):
    s = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    out, lse = pkg.attention.cross_attention(q, k, v, return_lse=True, scale=scale, **args)
    want, want_lse, p = ao.attention(q, k, v, read, s)
    assert out.dtype == q.dtype and out.is_contiguous() and lse.shape == want_lse.shape
    ao.within(out, want, ao.attention_bound(q, k, v, want, p, read, s))
    k64 = torch.where(read[:, :, None, None], k.double(), 0.0)
    ao.within(lse, want_lse, 2 * ao.score_error(q, k64, s) + k.shape[1] * ao.F32 + 4 * ao.F32 * torch.where(want_lse.isinf(), 0.0, want_lse.abs()))
    return out, lse


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind", ["full", "lengths", "mask", "both", "nothing"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(pkg, shape, kind, dtype):
    args, read = _masks(shape, kind)
    out, _ = _forward(pkg, *_inputs(shape, dtype)[:3], args, read)
    assert torch.equal(out, pkg.attention.cross_attention(*_inputs(shape, dtype)[:3], **args))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind", ["full", "lengths", "both", "nothing"])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(pkg, shape, kind, dtype):
    args, read = _masks(shape, kind)
    q, k, v, dout = _inputs(shape, dtype)
    out, lse = pkg.attention.cross_attention(q, k, v, return_lse=True, **args)
    got = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, **args)
    again = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, **args)
    want, bounds = ao.attention_gradients(q, k, v, dout, read, 1 / math.sqrt(q.shape[-1]))
    for g, a, w, b in zip(got, again, want, bounds):
        assert g.dtype == dtype and torch.equal(g, a)
        ao.within(g, w, b)
    assert not got[1][~read].any() and not got[2][~read].any()


@pytest.mark.parametrize("length", [0, 1, 2, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 383, 384])
@pytest.mark.parametrize("tokens", [1, 130])
def test_every_end_of_a_tile(pkg, length, tokens):
    """What lies behind the length is not a number, in either tensor."""
    shape = (2, tokens, 384, 4, 2, 128)
    q, k, v, dout = _inputs(shape, BF16)
    lengths = torch.tensor([length, 384 - length], device="cuda")
    read = torch.arange(384, device="cuda") < lengths[:, None]
    for junk in (math.nan, math.inf, -math.inf):
        k[~read] = junk
        v[~read] = junk
        out, lse = _forward(pkg, q, k, v, dict(lengths=lengths), read)
    got = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, lengths=lengths)
    want, bounds = ao.attention_gradients(q, k, v, dout, read, 1 / math.sqrt(128))
    for g, w, b in zip(got, want, bounds):
        ao.within(g, w, b)


@pytest.mark.parametrize("tokens", [1, 3, 40, 200])
def test_garbage_under_the_mask(pkg, tokens):
    shape = (2, tokens, 520, 4, 4, 64)
    q, k, v, dout = _inputs(shape, F16)
    args, read = _masks(shape, "mask", seed=5)
    k[~read] = math.nan
    v[~read] = math.inf
    out, lse = _forward(pkg, q, k, v, args, read)
    got = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, **args)
    want, bounds = ao.attention_gradients(q, k, v, dout, read, 1 / 8)
    for g, w, b in zip(got, want, bounds):
        ao.within(g, w, b)


@pytest.mark.parametrize("tokens", [1, 70])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_that_differ_by_thousands(pkg, tokens, dtype):
    """Rows whose largest score comes last, first, and far above the others: the running maximum moves by more than the
    exponential's range."""
    shape = (1, tokens, 600, 2, 1, 64)
    q, k, v, _ = _inputs(shape, dtype)
    q, k = q.sign() * 4, k.sign() * torch.linspace(0.125, 8, 600, device="cuda")[None, :, None, None].to(dtype)
    k = k.to(dtype)
    read = torch.ones(1, 600, dtype=torch.bool, device="cuda")
    for keys in (k, k.flip(1)):
        out = pkg.attention.cross_attention(q, keys, v, scale=1.0)
        want, _, p = ao.attention(q, keys, v, read, 1.0)
        ao.within(out, want, ao.attention_bound(q, keys, v, want, p, read, 1.0))


def test_lengths_out_of_range_are_the_nearest(pkg):
    shape = (3, 9, 100, 2, 2, 32)
    q, k, v, _ = _inputs(shape, BF16)
    got = pkg.attention.cross_attention(q, k, v, lengths=torch.tensor([-5, 1 << 40, 100], device="cuda"))
    want = pkg.attention.cross_attention(q, k, v, lengths=torch.tensor([0, 100, 100], device="cuda"))
    assert torch.equal(got, want)


@pytest.mark.parametrize("tokens", [1, 150])
def test_views_and_other_layouts(pkg, tokens):
    b, n, hq, hk, d = 2, 260, 4, 2, 64
    q, k, v, dout = _inputs((b, tokens, n, hq, hk, d), BF16)
    out, lse = pkg.attention.cross_attention(q, k, v, return_lse=True)
    grads = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse)
    joint = torch.stack((k, v), 2)
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    room = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")
    off = room[1:].view(q.shape)
    off.copy_(q)
    wide = torch.empty(b, n, hk, d + 4, dtype=BF16, device="cuda")[..., :d]   # rows that do not start on 16 bytes
    wide.copy_(k)
    every_second = torch.empty(b, 2 * n, hk, d, dtype=BF16, device="cuda")[:, ::2]
    every_second.copy_(v)
    for x, y, z in ((heads_first, joint[:, :, 0], joint[:, :, 1]), (off, wide, every_second)):
        assert torch.equal(pkg.attention.cross_attention(x, y, z), out)
        got = pkg.attention.cross_attention_backward(dout.transpose(1, 2).contiguous().transpose(1, 2), x, y, z, out, lse)
        assert all(torch.equal(g, w) for g, w in zip(got, grads))
    shared = k[:1].expand(b, -1, -1, -1)     # one image for every sample
    one = pkg.attention.cross_attention(q, shared, shared)
    assert torch.equal(one, pkg.attention.cross_attention(q, shared.contiguous(), shared.contiguous()))
    mask = torch.rand(b, 2 * n, device="cuda")[:, ::2] < 0.5
    assert torch.equal(pkg.attention.cross_attention(q, k, v, key_mask=mask), pkg.attention.cross_attention(q, k, v, key_mask=mask.contiguous()))


def test_empty_tensors(pkg):
    q, k, v, dout = _inputs((2, 4, 6, 2, 2, 64), BF16)
    out, lse = pkg.attention.cross_attention(q, k[:, :0], v[:, :0], return_lse=True)
    assert not out.any() and torch.equal(lse, torch.full_like(lse, -math.inf))
    dq, dk, dv = pkg.attention.cross_attention_backward(dout, q, k[:, :0], v[:, :0], out, lse)
    assert not dq.any() and dk.shape == (2, 0, 2, 64)
    out, lse = pkg.attention.cross_attention(q[:, :0], k, v, return_lse=True)
    assert out.shape == (2, 0, 2, 64)
    dq, dk, dv = pkg.attention.cross_attention_backward(dout[:, :0], q[:, :0], k, v, out, lse)
    assert dq.shape == (2, 0, 2, 64) and not dk.any() and not dv.any()


def test_gradients_against_differences(pkg):
    shape = (2, 19, 150, 4, 2, 32)
    q, k, v, dout = _inputs(shape, F16)
    args, read = _masks(shape, "both", seed=3)
    scale = 0.25
    out, lse = pkg.attention.cross_attention(q, k, v, return_lse=True, scale=scale, **args)
    grads = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, scale=scale, **args)
    _, bounds = ao.attention_gradients(q, k, v, dout, read, scale)
    at = [x.double() for x in (q, k, v)]

    def value(*x):
        return (ao.attention(*x, read, scale)[0] * dout.double()).sum()

    for i, (g, b) in enumerate(zip(grads, bounds)):
        d = torch.randn_like(at[i])
        step = 1e-5
        up, down = [list(at) for _ in range(2)]
        up[i], down[i] = at[i] + step * d, at[i] - step * d
        slope = (value(*up) - value(*down)) / (2 * step)
        assert (slope - (g.double() * d).sum()).abs() <= (b * d.abs()).sum() + 1e-6


def test_autograd_is_the_backward_pass(pkg):
    shape = (2, 40, 90, 4, 2, 64)
    q, k, v, dout = _inputs(shape, BF16)
    args, _ = _masks(shape, "both")
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    out = pkg.attention.cross_attention(*leaves, **args)
    out.backward(dout)
    o, lse = pkg.attention.cross_attention(q, k, v, return_lse=True, **args)
    want = pkg.attention.cross_attention_backward(dout, q, k, v, o, lse, **args)
    assert torch.equal(out, o) and all(torch.equal(x.grad, w) for x, w in zip(leaves, want))


@pytest.mark.parametrize("tokens", [1, 200])
def test_other_streams_and_graphs(pkg, tokens):
    shape = (2, tokens, 900, 8, 2, 128)
    q, k, v, dout = _inputs(shape, BF16)
    args, _ = _masks(shape, "both")
    want, lse = pkg.attention.cross_attention(q, k, v, return_lse=True, **args)
    grads = pkg.attention.cross_attention_backward(dout, q, k, v, want, lse, **args)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:                      # calls beside one another
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            late = k * 1
            got.append(pkg.attention.cross_attention(q, late, v, **args))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    held = torch.zeros_like(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        y, l = pkg.attention.cross_attention(q, held, v, return_lse=True, **args)
        g = pkg.attention.cross_attention_backward(dout, q, held, v, y, l, **args)
    for _ in range(2):
        held.copy_(k)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(g, grads))
        held.zero_()


@pytest.mark.parametrize("tokens", [1, 140])
def test_offsets_beyond_32_bits(pkg, tokens):
    apart = (1 << 31) + 64
    room = torch.empty(apart + 200 * 2 * 64, dtype=BF16, device="cuda")
    k = room.as_strided((2, 200, 2, 64), (apart, 128, 64, 1))
    q, k0, v, _ = _inputs((2, tokens, 200, 4, 2, 64), BF16)
    k.copy_(k0)
    assert torch.equal(pkg.attention.cross_attention(q, k, v), pkg.attention.cross_attention(q, k0, v))
