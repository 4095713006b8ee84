"""Rotary positions with several axes, alone and behind the norm of every head, against float64 forms: head sizes and
layouts, odd numbers of tokens and heads, views of a joint projection, types of positions and weights, gradients against
the formulas' and against differences."""
import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# batch, tokens, q heads, k heads, head_dim, sections, adjacent, interleaved
SHAPES = [
    (1, 1, 1, 1, 2, (1,), False, False),
    (1, 1, 32, 8, 128, (16, 24, 24), False, False),
    (2, 3, 5, 1, 128, (24, 20, 20), False, True),
    (3, 37, 7, 7, 64, (8, 10, 10), True, False),
    (1, 130, 2, 3, 80, (20, 20), True, True),
    (2, 65, 3, 1, 72, (12, 12, 12), False, False),      # rows of 9 units of 16 bytes
    (1, 33, 4, 2, 96, (8, 8, 8), False, False),         # half of the head passes through
    (1, 17, 3, 2, 96, (5, 3, 1, 2), True, True),
    (2, 9, 2, 1, 256, (128,), False, False),
    (1, 11, 2, 2, 256, (40, 40, 48), True, False),
    (1, 5, 3, 3, 6, (1, 1), False, True),
    (1, 7, 2, 1, 34, (0, 9, 8), False, False),          # an axis without pairs, rows of odd units
    (4, 1000, 3, 1, 32, (4, 6, 6), False, False),
]


def _inputs(shape, dtype, seed=0, pos=torch.int64, packed=False):
    b, t, hq, hk, d, sections, _, _ = shape
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def rand(*s):
        return torch.randn(s, generator=gen, device="cuda").to(dtype)

    if packed:
        joint = rand(b, t, hq + 2 * hk, d)
        q, k = joint[:, :, :hq], joint[:, :, hq:hq + hk]
    else:
        q, k = rand(b, t, hq, d), rand(b, t, hk, d)
    positions = torch.randint(0, 5000, (len(sections), b, t), generator=gen, device="cuda").to(pos)
    pairs = sum(sections)
    frequencies = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=F32) / pairs)
    return q, k, positions, frequencies, rand


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("packed", [False, True])
def test_rotary(pkg, shape, dtype, packed):
    sections, adjacent, interleaved = shape[5:]
    q, k, positions, frequencies, _ = _inputs(shape, dtype, packed=packed)
    for inverse in (False, True):
        got = pkg.attention.rotary(q, k, positions, frequencies, sections, inverse=inverse, adjacent=adjacent, interleaved=interleaved)
        for x, y in zip((q, k), got):
            want = ao.rotary(x.double(), positions, frequencies, sections, inverse, adjacent, interleaved)
            assert y.dtype == dtype and y.is_contiguous()
            ao.within(y, want, ao.rotary_bound(want, x.double(), sum(sections), adjacent, dtype))


@pytest.mark.parametrize("pos", [torch.int32, torch.int64, torch.float32])
def test_position_types_and_strides(pkg, pos):
    shape = (2, 19, 3, 2, 64, (10, 11, 11), False, False)
    q, k, positions, frequencies, _ = _inputs(shape, BF16, pos=pos)
    if pos is torch.float32:
        positions = positions + 0.37
    want = pkg.attention.rotary(q, k, positions, frequencies, shape[5])
    ref = ao.rotary(q.double(), positions, frequencies, shape[5])
    ao.within(want[0], ref, ao.rotary_bound(ref, q.double(), 32, False, BF16))
    across = positions.permute(1, 2, 0).contiguous().permute(2, 0, 1)        # axes next to one another in memory
    one = positions[:, :1].expand(-1, 2, -1)                                 # the same places for every sample
    for p in (across, one):
        got = pkg.attention.rotary(q, k, p, frequencies, shape[5])
        again = pkg.attention.rotary(q, k, p.contiguous(), frequencies, shape[5])
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    flat = pkg.attention.rotary(q[0], k[0], positions[:, 0], frequencies, shape[5])
    assert torch.equal(flat[0], want[0][0]) and torch.equal(flat[1], want[1][0])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_layouts_that_no_wide_load_fits(pkg, dtype):
    """Rows that start anywhere, heads ahead of tokens, elements that are not neighbours."""
    shape = (2, 21, 4, 2, 64, (16, 16), False, False)
    q, k, positions, frequencies, rand = _inputs(shape, dtype)
    want = pkg.attention.rotary(q, k, positions, frequencies, shape[5])
    room = rand(2 * 21 * 4 * 64 + 1)
    off = room[1:].view(2, 21, 4, 64)
    off.copy_(q)
    heads_first = k.transpose(1, 2).contiguous().transpose(1, 2)
    spread = rand(2, 21, 4, 128)[..., ::2]
    spread.copy_(q)
    odd = rand(2, 21, 4, 67)[..., :64]
    odd.copy_(q)
    for a in (off, spread, odd):
        got = pkg.attention.rotary(a, heads_first, positions, frequencies, shape[5])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_without_k_and_empty(pkg):
    shape = (2, 5, 3, 2, 64, (16, 16), False, False)
    q, k, positions, frequencies, _ = _inputs(shape, BF16)
    got = pkg.attention.rotary(q, None, positions, frequencies, shape[5])
    assert got[1] is None and torch.equal(got[0], pkg.attention.rotary(q, k, positions, frequencies, shape[5])[0])
    none = pkg.attention.rotary(q[:, :0], k[:, :0], positions[:, :, :0], frequencies, shape[5])
    assert none[0].shape == (2, 0, 3, 64)
    w = torch.ones(64, device="cuda")
    grads = pkg.attention.qk_norm_rotary_backward(q[:, :0], k[:, :0], q[:, :0], k[:, :0], positions[:, :, :0], frequencies, shape[5], w, w)
    assert grads[0].shape == (2, 0, 3, 64) and torch.equal(grads[2], torch.zeros_like(w))


def test_large_angles(pkg):
    """Positions up to 2^24: the angle is still the float32 product, its cosine still right."""
    q = torch.randn(1, 64, 2, 64, device="cuda")
    positions = torch.randint(1 << 20, 1 << 24, (1, 1, 64), device="cuda")
    frequencies = 10000.0 ** (-torch.arange(32, device="cuda", dtype=F32) / 32)
    got = pkg.attention.rotary(q, None, positions, frequencies, (32,))[0]
    want = ao.rotary(q.double(), positions, frequencies, (32,))
    ao.within(got, want, ao.rotary_bound(want, q.double(), 32, False, F32))


def _norm_bound(want, turned, pairs, adjacent, dtype, dim):
    return ao.rotary_bound(want, turned, pairs, adjacent, dtype, ao.norm_error(dim))


@pytest.mark.parametrize("dtype,wdtype", [(BF16, F32), (BF16, BF16), (F16, F16), (F32, F32), (F16, None)])
@pytest.mark.parametrize("shape", SHAPES)
def test_qk_norm_rotary(pkg, shape, dtype, wdtype):
    dim, sections, adjacent, interleaved = shape[4:]
    q, k, positions, frequencies, rand = _inputs(shape, dtype, packed=True)
    wq, wk = (None, None) if wdtype is None else ((1 + 0.3 * rand(dim)).to(wdtype), (1 + 0.3 * rand(dim)).to(wdtype))
    got = pkg.attention.qk_norm_rotary(q, k, positions, frequencies, sections, wq, wk, 1e-5, adjacent=adjacent, interleaved=interleaved)
    for x, w, y in zip((q, k), (wq, wk), got):
        n = ao.norm(x.double(), w, 1e-5)
        want = ao.rotary(n, positions, frequencies, sections, False, adjacent, interleaved)
        ao.within(y, want, _norm_bound(want, n, sum(sections), adjacent, dtype, dim))


@pytest.mark.parametrize("dtype,wdtype", [(BF16, F32), (BF16, BF16), (F16, F16), (F32, F32), (F32, None)])
@pytest.mark.parametrize("shape", SHAPES + [(3, 701, 6, 2, 128, (24, 20, 20), False, True)])
def test_qk_norm_rotary_backward(pkg, shape, dtype, wdtype):
    b, t, hq, hk, dim, sections, adjacent, interleaved = shape
    q, k, positions, frequencies, rand = _inputs(shape, dtype, packed=True)
    wq, wk = (None, None) if wdtype is None else ((1 + 0.3 * rand(dim)).to(wdtype), (1 + 0.3 * rand(dim)).to(wdtype))
    gq, gk = rand(*q.shape), rand(*k.shape)
    how = dict(adjacent=adjacent, interleaved=interleaved)
    got = pkg.attention.qk_norm_rotary_backward(gq, gk, q, k, positions, frequencies, sections, wq, wk, 1e-5, **how)
    again = pkg.attention.qk_norm_rotary_backward(gq, gk, q, k, positions, frequencies, sections, wq, wk, 1e-5, **how)
    for x, w, dy, dx, dw, dx2, dw2 in zip((q, k), (wq, wk), (gq, gk), got[:2], got[2:], again[:2], again[2:]):
        assert torch.equal(dx, dx2) and (dw is None) == (w is None)
        x64 = x.double()
        r = (x64.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        n = x64 * r
        g = ao.rotary(dy.double(), positions, frequencies, sections, True, adjacent, interleaved)
        size = ao.pair_size(dy.double(), sum(sections), adjacent)     # |terms| of which g is a sum
        w64 = torch.ones(dim, dtype=torch.float64, device="cuda") if w is None else w.double()
        dot = (g * w64 * n).mean(-1, keepdim=True)
        want = r * (g * w64 - n * dot)
        e = ao.norm_error(dim)
        terms = r * (size * w64.abs() + n.abs() * (size * w64.abs() * n.abs()).mean(-1, keepdim=True))
        ao.within(dx, want, ao.U[dtype] * 1.01 * want.abs() + (3 * e + 16 * ao.F32 + dim * ao.F32) * terms + ao.TINY[dtype])
        if w is not None:
            assert dw.dtype == wdtype and torch.equal(dw, dw2)
            want = (g * n).sum((0, 1, 2))
            rows = b * t * x.shape[2]
            bound = ao.U[wdtype] * 1.01 * want.abs() + (e + 16 * ao.F32 + min(rows, 4096) * ao.F32) * (size * n.abs()).sum((0, 1, 2))
            ao.within(dw, want, bound + ao.TINY[wdtype])


def test_gradients_against_differences(pkg):
    shape = (2, 13, 3, 2, 48, (8, 8, 6), True, True)
    dim, sections = shape[4], shape[5]
    q, k, positions, frequencies, rand = _inputs(shape, F32)
    wq, wk = 1 + 0.3 * rand(dim), 1 + 0.3 * rand(dim)
    gq, gk = rand(*q.shape), rand(*k.shape)
    how = dict(adjacent=True, interleaved=True)

    def value(q, k, wq, wk):   # float64, independent of the kernels
        return sum((ao.rotary(ao.norm(x, w, 1e-6), positions, frequencies, sections, False, True, True) * g.double()).sum()
                   for x, w, g in ((q, wq, gq), (k, wk, gk)))

    grads = pkg.attention.qk_norm_rotary_backward(gq, gk, q, k, positions, frequencies, sections, wq, wk, **how)
    at = [x.double() for x in (q, k, wq, wk)]
    for i, g in enumerate(grads):
        d = torch.randn_like(at[i])
        step = 1e-5
        up, down = [list(at) for _ in range(2)]
        up[i] = at[i] + step * d
        down[i] = at[i] - step * d
        slope = (value(*up) - value(*down)) / (2 * step)
        # the difference quotient is good to 1e-9 or so, the float32 gradient to a few units of its largest terms
        bound = 1e-5 * (g.double().abs() * d.abs()).sum() + 1e-6
        assert (slope - (g.double() * d).sum()).abs() <= bound


def test_autograd_is_the_backward_pass(pkg):
    shape = (2, 9, 4, 2, 64, (16, 8, 8), False, False)
    q, k, positions, frequencies, rand = _inputs(shape, BF16)
    wq, wk = 1 + 0.3 * rand(64).float(), 1 + 0.3 * rand(64).float()
    gq, gk = rand(*q.shape), rand(*k.shape)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, wq, wk)]
    out = pkg.attention.qk_norm_rotary(leaves[0], leaves[1], positions, frequencies, shape[5], leaves[2], leaves[3])
    torch.autograd.backward(out, (gq, gk))
    want = pkg.attention.qk_norm_rotary_backward(gq, gk, q, k, positions, frequencies, shape[5], wq, wk)
    assert all(torch.equal(x.grad, w) for x, w in zip(leaves, want))
    x = q.detach().clone().requires_grad_()
    y, none = pkg.attention.rotary(x, None, positions, frequencies, shape[5])
    y.backward(gq)
    assert none is None and torch.equal(x.grad, pkg.attention.rotary(gq, None, positions, frequencies, shape[5], inverse=True)[0])


def test_infinities_stay_in_their_pairs(pkg):
    shape = (1, 4, 2, 1, 64, (32,), False, False)
    q, k, positions, frequencies, _ = _inputs(shape, F32)
    clean = pkg.attention.rotary(q, k, positions, frequencies, shape[5])[0]
    q[0, 1, 0, 3] = float("inf")
    got = pkg.attention.rotary(q, k, positions, frequencies, shape[5])[0]
    touched = torch.zeros_like(got, dtype=torch.bool)
    touched[0, 1, 0, 3] = touched[0, 1, 0, 35] = True
    assert torch.equal(got[~touched], clean[~touched])


def test_other_streams_and_graphs(pkg):
    shape = (2, 100, 4, 2, 128, (24, 20, 20), False, False)
    q, k, positions, frequencies, rand = _inputs(shape, BF16)
    w = 1 + 0.3 * rand(128).float()
    want = pkg.attention.qk_norm_rotary(q, k, positions, frequencies, shape[5], w, w)
    grads = pkg.attention.qk_norm_rotary_backward(*want, q, k, positions, frequencies, shape[5], w, w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        late = q * 1
        got = pkg.attention.qk_norm_rotary(late, k, positions, frequencies, shape[5], w, w)
    stream.synchronize()
    assert torch.equal(got[0], want[0])
    held = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = pkg.attention.qk_norm_rotary(held, k, positions, frequencies, shape[5], w, w)
        g = pkg.attention.qk_norm_rotary_backward(*y, held, k, positions, frequencies, shape[5], w, w)
    held.copy_(q)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(y + g, want + grads))


def test_offsets_beyond_32_bits(pkg):
    """Two samples further apart than 2^31 elements."""
    apart = (1 << 31) + 64
    room = torch.empty(apart + 3 * 2 * 64, dtype=BF16, device="cuda")
    q = room.as_strided((2, 3, 2, 64), (apart, 128, 64, 1))
    q.copy_(torch.randn(2, 3, 2, 64, device="cuda"))
    positions = torch.arange(6, device="cuda").view(1, 2, 3)
    frequencies = torch.rand(32, device="cuda")
    got = pkg.attention.rotary(q, None, positions, frequencies, (32,))[0]
    assert torch.equal(got, pkg.attention.rotary(q.contiguous(), None, positions, frequencies, (32,))[0])
