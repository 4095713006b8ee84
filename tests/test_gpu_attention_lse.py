"""The gradient of lse: against the formula's, against differences, and through autograd, where calls are joined by their lse."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402

pytestmark = pytest.mark.gpu

# batch, tokens, keys, q heads, kv heads, head_dim
SHAPES = [(1, 1, 1, 1, 1, 8), (2, 1, 129, 8, 1, 64), (2, 130, 300, 12, 2, 96), (1, 257, 385, 3, 3, 64), (1, 128, 1025, 4, 2, 128)]


def _inputs(shape, dtype):
    b, t, n, hq, hk, d = shape
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    q, k, v, dout = (torch.randn(s, generator=gen, device="cuda").to(dtype)
                     for s in ((b, t, hq, d), (b, n, hk, d), (b, n, hk, d), (b, t, hq, d)))
    lengths = torch.randint(1, n + 1, (b,), generator=gen, device="cuda")
    lengths[-1] = 0 if b > 1 else n
    read = torch.arange(n, device="cuda") < lengths[:, None]
    return q, k, v, dout, 3 * torch.randn((b, hq, t), generator=gen, device="cuda"), lengths, read


def _with_lse(q, k, v, dout, dlse, read, scale):
    """Gradients of sum(dout out) + sum(dlse lse) and their bounds: dS = P (dP - delta + dlse), the last term rounded with the others."""
    (dq, dk, dv), (bq, bk, bv) = ao.attention_gradients(q, k, v, dout, read, scale)
    group = q.shape[2] // k.shape[2]
    p = ao.attention(q, k, v, read, scale)[2]
    more = p * dlse.double()[..., None]
    k64 = torch.where(read[:, :, None, None], k.double(), 0.0).repeat_interleave(group, 2)
    u = ao.U[q.dtype] * 1.01
    off = more.abs() * (u + 2 * ao.score_error(q, k64, scale) + 4 * ao.F32)

    def by_query(x, keys):
        return torch.einsum("bhsn,bnhd->bshd", x, keys) * scale

    def by_key(x, queries):
        return torch.einsum("bhsn,bshd->bnhd", x, queries).unflatten(2, (-1, group)).sum(3) * scale

    mq, mk = by_query(more, k64), by_key(more, q.double())
    n, t = k.shape[1], q.shape[1] * group
    return ((dq + mq, dk + mk, dv),
            (bq + u * mq.abs() + by_query(off, k64.abs()) * (1 + n * ao.F32), bk + u * mk.abs() + by_key(off, q.double().abs()) * (1 + t * ao.F32), bv))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formula(pkg, shape, dtype):
    q, k, v, dout, dlse, lengths, read = _inputs(shape, dtype)
    out, lse = pkg.attention.cross_attention(q, k, v, lengths=lengths, return_lse=True)
    got = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, lengths=lengths, lse_grad=dlse)
    spread = torch.stack((dlse, dlse), -1)[..., 0]               # not contiguous
    again = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, lengths=lengths, lse_grad=spread)
    want, bounds = _with_lse(q, k, v, dout, dlse, read, 1 / math.sqrt(shape[-1]))
    for g, a, w, b in zip(got, again, want, bounds):
        assert torch.equal(g, a)
        ao.within(g, w, b)
    without = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, lengths=lengths)
    zero = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, lengths=lengths, lse_grad=torch.zeros_like(dlse))
    assert all(torch.equal(a, b) for a, b in zip(without, zero))


def test_against_differences(pkg):
    q, k, v, dout, dlse, lengths, read = _inputs((2, 19, 150, 4, 2, 32), torch.float16)
    scale = 0.25
    out, lse = pkg.attention.cross_attention(q, k, v, lengths=lengths, scale=scale, return_lse=True)
    grads = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, lengths=lengths, scale=scale, lse_grad=dlse)
    bounds = _with_lse(q, k, v, dout, dlse, read, scale)[1]
    at = [x.double() for x in (q, k, v)]

    def value(*x):
        o, l, _ = ao.attention(*x, read, scale)
        return (o * dout.double()).sum() + (l.masked_fill(l == -math.inf, 0.0) * dlse.double()).sum()

    for i, (g, b) in enumerate(zip(grads, bounds)):
        d = torch.randn_like(at[i])
        step = 1e-5
        up, down = [list(at) for _ in range(2)]
        up[i], down[i] = at[i] + step * d, at[i] - step * d
        slope = (value(*up) - value(*down)) / (2 * step)
        assert (slope - (g.double() * d).sum()).abs() <= (b * d.abs()).sum() + 1e-6


@pytest.mark.parametrize("used", ["both", "out", "lse"])
def test_through_autograd(pkg, used):
    q, k, v, dout, dlse, lengths, _ = _inputs((2, 40, 90, 4, 2, 64), torch.bfloat16)
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    out, lse = pkg.attention.cross_attention(*leaves, lengths=lengths, return_lse=True)
    loss = 0
    if used != "lse":
        loss = loss + (out * dout).sum(dtype=torch.float32)
    if used != "out":
        loss = loss + (lse.masked_fill(lse == -math.inf, 0.0) * dlse).sum()
    loss.backward()
    zero = torch.zeros_like(dout) if used == "lse" else dout
    want = pkg.attention.cross_attention_backward(zero, q, k, v, out.detach(), lse.detach(), lengths=lengths,
                                                  lse_grad=None if used == "out" else dlse.masked_fill(lse == -math.inf, 0.0))
    assert all(torch.equal(x.grad, w) for x, w in zip(leaves, want))


def test_refusals(pkg):
    q, k, v, dout, dlse, lengths, _ = _inputs((2, 5, 9, 2, 2, 64), torch.bfloat16)
    out, lse = pkg.attention.cross_attention(q, k, v, return_lse=True)
    for bad in (dlse.double(), dlse.cpu(), dlse[:, :1], dlse.half(), dlse.transpose(0, 1).contiguous()[:1], 1.0):
        with pytest.raises(ValueError, match="lse_grad"):
            pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, lse_grad=bad)
