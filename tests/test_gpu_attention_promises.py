"""What the header and the docstrings say and other tests do not reach: rotation in place, gradients of any layout, stretches of keys
longer than usual, gradients where scores differ by thousands, first calls under capture."""
import ctypes
import math
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _heads(capi, x):
    return capi.Heads(x.data_ptr(), x.stride(0), x.stride(1), x.stride(2))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("shape", [(2, 37, 7, 3, 64, 32), (1, 1, 32, 8, 128, 64), (1, 9, 2, 2, 34, 5), (2, 300, 5, 5, 80, 20)])
def test_rotation_in_place(pkg, shape, norm, adjacent, dtype):
    """q_out and k_out are q and k, inside a joint projection whose other values stay."""
    capi, lib = pkg._capi, pkg._capi.load()
    b, t, hq, hk, dim, pairs = shape
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    joint = torch.randn((b, t, hq + 2 * hk, dim), generator=gen, device="cuda").to(dtype)
    q, k, rest = joint[:, :, :hq], joint[:, :, hq:hq + hk], joint[:, :, hq + hk:].clone()
    positions = torch.randint(0, 900, (1, b, t), generator=gen, device="cuda")
    frequencies = torch.rand(pairs, generator=gen, device="cuda")
    weight = 1 + torch.rand(dim, generator=gen, device="cuda")
    if norm:
        want = pkg.attention.qk_norm_rotary(q, k, positions, frequencies, (pairs,), weight, weight, adjacent=adjacent)
    else:
        want = pkg.attention.rotary(q, k, positions, frequencies, (pairs,), adjacent=adjacent)
    d = capi.RotaryDesc(dtype={BF16: capi.BF16, F16: capi.F16, F32: capi.F32}[dtype], batch=b, tokens=t, q_heads=hq, k_heads=hk, head_dim=dim,
                        q=_heads(capi, q), k=_heads(capi, k), q_out=_heads(capi, q), k_out=_heads(capi, k), positions=positions.data_ptr(),
                        positions_dtype=capi.I64, positions_stride_axis=b * t, positions_stride_batch=t, positions_stride_token=1,
                        frequencies=frequencies.data_ptr(), n_axes=1, adjacent=adjacent, q_weight=weight.data_ptr(),
                        k_weight=weight.data_ptr(), weight_dtype=capi.F32, eps=1e-6)
    d.sections[0] = pairs
    entry = lib.mlxd_qk_norm_rotary if norm else lib.mlxd_rotary
    assert entry(0, torch.cuda.current_stream().cuda_stream, ctypes.byref(d)) == capi.OK
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(joint[:, :, hq + hk:], rest)


def test_gradients_of_other_layouts(pkg):
    dtype, shape = BF16, (2, 21, 4, 64)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    q, dy = (torch.randn(shape, generator=gen, device="cuda").to(dtype) for _ in range(2))
    positions = torch.randint(0, 900, (1, 2, 21), generator=gen, device="cuda")
    frequencies, w = torch.rand(32, generator=gen, device="cuda"), 1 + torch.rand(64, generator=gen, device="cuda")

    def both(g):
        turned = pkg.attention.rotary(g, None, positions, frequencies, (32,), inverse=True)[:1]
        return turned + pkg.attention.qk_norm_rotary_backward(g, g, q, q, positions, frequencies, (32,), w, w)

    want = both(dy)
    off = torch.empty(dy.numel() + 1, dtype=dtype, device="cuda")[1:].view(shape)
    wide = torch.empty(2, 21, 4, 67, dtype=dtype, device="cuda")[..., :64]
    spread = torch.empty(2, 21, 4, 128, dtype=dtype, device="cuda")[..., ::2]
    heads_first = torch.empty(2, 4, 21, 64, dtype=dtype, device="cuda").transpose(1, 2)
    for g in (off, wide, spread, heads_first):
        g.copy_(dy)
        for a, b in zip(both(g), want):
            assert a.dtype == b.dtype
            # sums of the weights' gradients go in another order where vectors are of another length
            assert torch.equal(a, b) if a.dim() == 4 else torch.allclose(a, b, rtol=1e-5, atol=1e-4)
    one = torch.ones((), dtype=dtype, device="cuda").expand(shape)            # what sum().backward() hands down
    for a, b in zip(both(one), both(torch.ones(shape, dtype=dtype, device="cuda"))):
        assert torch.equal(a, b)
    few = dy[:, :, :1].expand(shape)                                           # one head's gradient for all
    for a, b in zip(both(few), both(few.contiguous())):
        assert torch.equal(a, b)


def test_gradients_of_other_layouts_in_float32(pkg):
    """Where vectors are of another length the sums over a head go in another order: each layout against the formula."""
    b, t, h, dim = shape = (2, 21, 4, 64)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    q, dy = (torch.randn(shape, generator=gen, device="cuda") for _ in range(2))
    positions = torch.randint(0, 900, (1, b, t), generator=gen, device="cuda")
    frequencies, w = torch.rand(32, generator=gen, device="cuda"), 1 + torch.rand(dim, generator=gen, device="cuda")
    layouts = [torch.empty(dy.numel() + 1, device="cuda")[1:].view(shape), torch.empty(b, t, h, dim + 3, device="cuda")[..., :dim],
               torch.empty(b, t, h, 2 * dim, device="cuda")[..., ::2], torch.empty(b, h, t, dim, device="cuda").transpose(1, 2),
               torch.empty(b, t, 1, dim, device="cuda").expand(shape)]
    x, w64 = q.double(), w.double()
    r = (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    n = x * r
    for layout in layouts:
        g = layout
        g[:, :, :1].copy_(dy[:, :, :1])
        if g.stride(2):
            g.copy_(dy)
        size = ao.pair_size(g.double(), 32, False)
        turned = ao.rotary(g.double(), positions, frequencies, (32,), True)
        got = pkg.attention.rotary(g, None, positions, frequencies, (32,), inverse=True)[0]
        ao.within(got, turned, ao.rotary_bound(turned, g.double(), 32, False, F32))
        dx, _, dw, _ = pkg.attention.qk_norm_rotary_backward(g, None, q, None, positions, frequencies, (32,), w)
        want = r * (turned * w64 - n * (turned * w64 * n).mean(-1, keepdim=True))
        e = ao.norm_error(dim)
        terms = r * (size * w64 + n.abs() * (size * w64 * n.abs()).mean(-1, keepdim=True))
        ao.within(dx, want, ao.U[F32] * 1.01 * want.abs() + (3 * e + 16 * ao.F32 + dim * ao.F32) * terms + ao.TINY[F32])
        want = (turned * n).sum((0, 1, 2))
        ao.within(dw, want, ao.U[F32] * 1.01 * want.abs() + (e + 16 * ao.F32 + b * t * h * ao.F32) * (size * n.abs()).sum((0, 1, 2)) + ao.TINY[F32])


@pytest.mark.parametrize("kind", ["full", "lengths", "mask"])
def test_stretches_longer_than_usual(pkg, kind):
    """So many keys that a row would have over 64 parts while CTAs are plenty: stretches of 4096."""
    b, n, h, d = 2, 150001, 4, 64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    q = 2 * torch.randn((b, 1, h, d), generator=gen, device="cuda")
    q, (k, v) = q.to(BF16), (torch.randn((b, n, h, d), generator=gen, device="cuda").to(BF16) for _ in range(2))
    read, args = torch.ones((b, n), dtype=torch.bool, device="cuda"), {}
    if kind == "lengths":
        lengths = torch.tensor([n - 5, 70001], device="cuda")
        args, read = dict(lengths=lengths), torch.arange(n, device="cuda") < lengths[:, None]
    if kind == "mask":
        read = torch.rand((b, n), generator=gen, device="cuda") < 0.5
        read[1, :140000] = False
        args = dict(key_mask=read)
    out, lse = pkg.attention.cross_attention(q, k, v, return_lse=True, **args)
    want, want_lse, p = ao.attention(q, k, v, read, 1 / 8)
    ao.within(out, want, ao.attention_bound(q, k, v, want, p, read, 1 / 8))
    k64 = torch.where(read[:, :, None, None], k.double(), 0.0)
    ao.within(lse, want_lse, 2 * ao.score_error(q, k64, 1 / 8) + n * ao.F32 + 4 * ao.F32 * want_lse.abs())


@pytest.mark.parametrize("tokens", [1, 70, 200])
def test_gradients_where_scores_differ_by_thousands(pkg, tokens):
    dtype = F16
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    q, k, v, dout = (torch.randn((1, n, h, 64), generator=gen, device="cuda").to(dtype) for n, h in ((tokens, 2), (600, 1), (600, 1), (tokens, 2)))
    q = q.sign() * 4
    k = (k.sign() * torch.linspace(0.125, 8, 600, device="cuda")[None, :, None, None]).to(dtype)
    read = torch.ones(1, 600, dtype=torch.bool, device="cuda")
    for keys in (k, k.flip(1)):
        out, lse = pkg.attention.cross_attention(q, keys, v, scale=1.0, return_lse=True)
        got = pkg.attention.cross_attention_backward(dout, q, keys, v, out, lse, scale=1.0)
        want, bounds = ao.attention_gradients(q, keys, v, dout, read, 1.0)
        for g, w, b in zip(got, want, bounds):
            ao.within(g, w, b)


FIRST_CALL = """
import sys, torch
from __graft_entry__ import load_package
A = load_package().attention
n = 1 if sys.argv[1] == "step" else 300
q, k = (torch.randn(2, x, 4, 64, device="cuda").to(torch.bfloat16) for x in (n, 900))
f, p, w = torch.ones(32, device="cuda"), torch.zeros(1, 2, n, device="cuda"), torch.ones(64, device="cuda")
lse = torch.zeros(2, 4, n, device="cuda")
call = dict(rotary=lambda: A.rotary(q, q, p, f, (32,)), norm=lambda: A.qk_norm_rotary_backward(q, q, q, q, p, f, (32,), w, w),
            step=lambda: A.cross_attention(q, k, k), forward=lambda: A.cross_attention(q, k, k),
            backward=lambda: A.cross_attention_backward(q, q, k, k, q, lse))[sys.argv[1]]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = call()
graph.replay()
want = call()
torch.cuda.synchronize()
pairs = zip(got, want) if isinstance(got, tuple) else [(got, want)]
assert all(torch.equal(a, b) for a, b in pairs)
"""


@pytest.mark.parametrize("which", ["rotary", "norm", "step", "forward", "backward"])
def test_first_call_of_a_process_under_capture(which):
    r = subprocess.run([sys.executable, "-c", FIRST_CALL, which], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_the_same_call_gives_the_same_bits(pkg):
    """Also beside other work that changes the order in which CTAs run."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    q, k, v = (torch.randn((2, n, h, 128), generator=gen, device="cuda").to(BF16) for n, h in ((500, 8), (3000, 2), (3000, 2)))
    want = pkg.attention.cross_attention(q, k, v, return_lse=True)
    grads = pkg.attention.cross_attention_backward(q, q, k, v, *want)
    step = pkg.attention.cross_attention(q[:, :1], k, v)
    other = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(other):
            busy @ busy
        assert all(torch.equal(a, b) for a, b in zip(pkg.attention.cross_attention(q, k, v, return_lse=True), want))
        assert all(torch.equal(a, b) for a, b in zip(pkg.attention.cross_attention_backward(q, q, k, v, *want), grads))
        assert torch.equal(pkg.attention.cross_attention(q[:, :1], k, v), step)
    assert math.isfinite(want[1].sum().item())
