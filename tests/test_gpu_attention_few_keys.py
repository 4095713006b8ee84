"""Gradients where few keys have weights, whose dS is a small difference: to the precision of 16-bit operands, without what the rounding of
the result would add.

Bound of dS = P (dP - delta) with delta = sum(P dP) / sum(P) in float32: its rounding to 16 bits and P's own error e (twice, as in the
oracle's bounds), dP's sums of `dim` products, and delta's of at most 128 of these, weighted."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402

pytestmark = pytest.mark.gpu


def _gradients(q, k, v, dout, read, scale):
    dtype, group, dim = q.dtype, q.shape[2] // k.shape[2], q.shape[-1]
    _, _, p = ao.attention(q, k, v, read, scale)
    q64, do = q.double(), dout.double()
    k64, v64 = (torch.where(read[:, :, None, None], x.double(), 0.0).repeat_interleave(group, 2) for x in (k, v))
    dp = torch.einsum("bshd,bnhd->bhsn", do, v64)
    size = torch.einsum("bshd,bnhd->bhsn", do.abs(), v64.abs())
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    u, e, n = ao.U[dtype] * 1.01, ao.score_error(q, k64, scale), k.shape[1]
    delta_off = (p * (2 * dim * ao.F32 * size + (4 * e + 2 * n * ao.F32) * dp.abs())).sum(-1, keepdim=True)
    off = ds.abs() * (u + 2 * e) + p * (2 * dim * ao.F32 * size + delta_off) + ao.TINY[dtype]

    def shared(x):
        return x.view(*x.shape[:2], -1, group, dim).sum(3)

    dq = torch.einsum("bhsn,bnhd->bshd", ds, k64) * scale
    dk = shared(torch.einsum("bhsn,bshd->bnhd", ds, q64)) * scale
    bq = u * dq.abs() + scale * torch.einsum("bhsn,bnhd->bshd", off, k64.abs()) * (1 + n * ao.F32) + ao.TINY[dtype]
    bk = u * dk.abs() + scale * shared(torch.einsum("bhsn,bshd->bnhd", off, q64.abs())) * (1 + q.shape[1] * group * ao.F32) + ao.TINY[dtype]
    return (dq, dk), (bq, bk)


def _inputs(keys, dtype, heads=(4, 2), dim=64, tokens=150, batch=2):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(keys)
    q, k, v, dout = (torch.randn((batch, n, h, dim), generator=gen, device="cuda")
                     for n, h in ((tokens, heads[0]), (keys, heads[1]), (keys, heads[1]), (tokens, heads[0])))
    return (2 * q).to(dtype), k.to(dtype), v.to(dtype), dout.to(dtype)


def _run(pkg, q, k, v, dout, **args):
    out, lse = pkg.attention.cross_attention(q, k, v, return_lse=True, **args)
    return pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, **args)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 64, 80, 128])
@pytest.mark.parametrize("keys", [1, 2, 3, 5, 17, 64, 65, 127, 128])
def test_all_keys_of_one_tile(pkg, keys, dim, dtype):
    q, k, v, dout = _inputs(keys, dtype, dim=dim)
    read = torch.ones(2, keys, dtype=torch.bool, device="cuda")
    got = _run(pkg, q, k, v, dout)
    want, bounds = _gradients(q, k, v, dout, read, 1 / math.sqrt(dim))
    for g, w, b in zip(got, want, bounds):
        ao.within(g, w, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["lengths", "mask"])
def test_few_of_many_keys(pkg, kind, dtype):
    """A sample of few keys beside one of several tiles; those of the other sample are checked elsewhere."""
    q, k, v, dout = _inputs(400, dtype)
    for few in (1, 2, 7, 128):
        read = torch.zeros(2, 400, dtype=torch.bool, device="cuda")
        read[0, :300] = True
        if kind == "lengths":
            read[1, :few] = True
            args = dict(lengths=torch.tensor([300, few], device="cuda"))
        else:
            read[1, 127 - torch.arange(few, device="cuda") * 127 // few] = True
            args = dict(key_mask=read)
        got = _run(pkg, q, k, v, dout, **args)
        want, bounds = _gradients(q, k, v, dout, read, 1 / 8)
        for g, w, b in zip(got, want, bounds):
            ao.within(g[1:], w[1:], b[1:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 64, 72, 128])
@pytest.mark.parametrize("tokens", [1, 128, 300])
def test_a_single_key_has_no_gradient(pkg, tokens, dim, dtype):
    """Its weight is 1 whatever the score: dQ and dK are 0, dV is the sum of dout."""
    for keys, at in ((1, 0), (5, 3), (200, 100)):
        q, k, v, dout = _inputs(keys, dtype, dim=dim, tokens=tokens)
        mask = torch.zeros(2, keys, dtype=torch.bool, device="cuda")
        mask[:, at] = True
        calls = [dict(key_mask=mask)] + ([dict(lengths=torch.tensor([1, 1], device="cuda"))] if at == 0 else [])
        for args in calls + ([{}] if keys == 1 else []):
            dq, dk, dv = _run(pkg, q, k, v, dout, **args)
            assert not dq.any() and not dk.any()
            want = dout.double().unflatten(2, (2, 2)).sum((1, 3))
            size = dout.double().abs().unflatten(2, (2, 2)).sum((1, 3))
            e = ao.score_error(q, k.double(), 1 / math.sqrt(dim))
            ao.within(dv[:, at], want, ao.U[dtype] * 1.01 * want.abs() + (ao.U[dtype] * 1.01 + 2 * e + 2 * tokens * ao.F32) * size + ao.TINY[dtype])
