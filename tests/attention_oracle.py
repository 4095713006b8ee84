"""Plain float64 forms of the attention operators, with bounds on what float32 sums and one rounding may change.

``U`` is half a unit in the last place of each type, relative: what one rounding may move.  Bounds are per element and hold
for any order of the sums.
"""
import math

import torch

U = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}   # 2^-24, 2^-11, 2^-8
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}   # half the least step
F32 = 2.0 ** -24


def within(got, want, bound):
    """Every element of `got` within `bound` of `want`, and finite where it is."""
    got = got.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    off = (got - want).abs()
    off = torch.where(torch.isfinite(want), off, torch.zeros_like(off))
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0, "off by %g where %g is allowed" % (off.flatten()[(off - bound).argmax()], bound.flatten()[(off - bound).argmax()])


def axis_of_pair(sections, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


def units(positions, frequencies, sections, interleaved):
    """cos and sin [..., 1, pairs] of the float32 products, in float64."""
    axes = torch.tensor(axis_of_pair(sections, interleaved), device=positions.device)
    p = positions.to(torch.float32)[axes].movedim(0, -1)
    angle = (p * frequencies).double().unsqueeze(-2)
    return angle.cos(), angle.sin()


def split(x, pairs, adjacent):
    if adjacent:
        return x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2], x[..., 2 * pairs:]
    return x[..., :pairs], x[..., pairs:2 * pairs], x[..., 2 * pairs:]


def join(a, b, rest, adjacent):
    y = torch.stack((a, b), -1).flatten(-2) if adjacent else torch.cat((a, b), -1)
    return torch.cat((y, rest), -1)


def rotary(x, positions, frequencies, sections, inverse=False, adjacent=False, interleaved=False):
    cos, sin = units(positions, frequencies, sections, interleaved)
    a, b, rest = split(x, cos.shape[-1], adjacent)
    if inverse:
        sin = -sin
    return join(a * cos - b * sin, b * cos + a * sin, rest, adjacent)


def pair_size(x, pairs, adjacent):
    """|a| + |b| of each element's pair, |x| of elements that pass through."""
    a, b, rest = split(x.abs(), pairs, adjacent)
    return join(a + b, a + b, rest, adjacent)


def rotary_bound(want, x, pairs, adjacent, dtype, more=0.0):
    """cos and sin are within 2 units, two products and a sum add 2 more; `more`: relative error of what is turned."""
    return U[dtype] * want.abs() * 1.01 + (8 * F32 + more) * pair_size(x, pairs, adjacent) + TINY[dtype]


def norm(x, w, eps):
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return n if w is None else n * w.double()


def norm_error(dim):
    """Relative error of x * r * w: the sum of squares (dim / 2 units after the root), its root, two products."""
    return (dim / 2 + 8) * F32


def attention(q, k, v, read, scale):
    """(out, lse, P) over the keys for which `read` [batch, keys] is true, everything in float64."""
    group = q.shape[2] // k.shape[2]
    k = torch.where(read[:, :, None, None], k.double(), 0.0).repeat_interleave(group, 2)
    v = torch.where(read[:, :, None, None], v.double(), 0.0).repeat_interleave(group, 2)
    s = torch.einsum("bshd,bnhd->bhsn", q.double(), k) * scale
    s = s.masked_fill(~read[:, None, None, :], -math.inf)
    lse = torch.logsumexp(s, -1) if s.shape[-1] else torch.full(s.shape[:-1], -math.inf, dtype=s.dtype, device=s.device)
    p = torch.where(read[:, None, None, :], (s - lse.masked_fill(lse == -math.inf, 0.0)[..., None]).exp(), 0.0)
    return torch.einsum("bhsn,bnhd->bshd", p, v), lse, p


def attention_gradients(q, k, v, dout, read, scale):
    """(dq, dk, dv) and their bounds, for products whose operands P and dS are rounded to the tensors' type."""
    dtype, group, dim = q.dtype, q.shape[2] // k.shape[2], q.shape[-1]
    out, lse, p = attention(q, k, v, read, scale)
    q64, do = q.double(), dout.double()
    k64 = torch.where(read[:, :, None, None], k.double(), 0.0).repeat_interleave(group, 2)
    v64 = torch.where(read[:, :, None, None], v.double(), 0.0).repeat_interleave(group, 2)
    delta = (do * out).sum(-1).transpose(1, 2)
    ds = p * (torch.einsum("bshd,bnhd->bhsn", do, v64) - delta[..., None])

    def shared(x):   # sum over the query heads of a key head
        return x.view(*x.shape[:2], -1, group, dim).sum(3)

    dq = torch.einsum("bhsn,bnhd->bshd", ds, k64) * scale
    dk = shared(torch.einsum("bhsn,bshd->bnhd", ds, q64)) * scale
    dv = shared(torch.einsum("bhsn,bshd->bnhd", p, do))
    e = score_error(q, k64, scale)
    # out comes in rounded: sum |dout| |out| u; dP in float32 sums of dim products
    off = ds.abs() * (U[dtype] * 1.01 + 2 * e) + p * (
        2 * dim * F32 * torch.einsum("bshd,bnhd->bhsn", do.abs(), v64.abs()) +
        (U[dtype] * 1.01 + dim * F32) * (do.abs() * out.abs()).sum(-1).transpose(1, 2)[..., None] +
        # what is off in out before its rounding is off in delta
        ((U[dtype] + 2 * e) * torch.einsum("bhsn,bnhd->bshd", p, v64.abs()) * do.abs()).sum(-1).transpose(1, 2)[..., None]
    ) + TINY[dtype]
    u, n, t = U[dtype] * 1.01, k.shape[1], q.shape[1] * group
    bq = u * dq.abs() + scale * torch.einsum("bhsn,bnhd->bshd", off, k64.abs()) * (1 + n * F32) + TINY[dtype]
    bk = u * dk.abs() + scale * shared(torch.einsum("bhsn,bshd->bnhd", off, q64.abs())) * (1 + t * F32) + TINY[dtype]
    offp = p * (u + 2 * e) + TINY[dtype]
    bv = u * dv.abs() + shared(torch.einsum("bhsn,bshd->bnhd", offp, do.abs())) * (1 + t * F32) + TINY[dtype]
    return (dq, dk, dv), (bq, bk, bv)


def score_error(q, k64, scale):
    """Largest absolute error of a score (a float32 sum of dim products, scaled), and of the exponential taken of it."""
    size = (q.double().norm(dim=-1).max() * k64.norm(dim=-1).max() * abs(scale)).item() if k64.numel() and q.numel() else 0.0
    return (q.shape[-1] + 8) * F32 * size + 2.0 ** -20


def attention_bound(q, k, v, out, p, read, scale):
    """P rounded to the tensors' type (its least steps where it is tiny, against a largest value of at least 1), sums in
    float32, the result rounded once."""
    dtype, group, n = q.dtype, q.shape[2] // k.shape[2], k.shape[1]
    k64 = torch.where(read[:, :, None, None], k.double(), 0.0).repeat_interleave(group, 2)
    v64 = torch.where(read[:, :, None, None], v.double(), 0.0).repeat_interleave(group, 2)
    a = torch.einsum("bhsn,bnhd->bshd", p, v64.abs())
    e = score_error(q, k64, scale)
    return U[dtype] * 1.01 * out.abs() + (U[dtype] * 1.01 + 2 * e + n * F32) * a + TINY[dtype] * (1 + v64.abs().sum(1, keepdim=True))
