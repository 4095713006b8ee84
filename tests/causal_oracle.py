"""Plain float64 forms of attention where every query has its own keys to read, with bounds for products whose operands are rounded to
the tensors' type (see attention_oracle)."""
import math

import torch

import attention_oracle as ao

U, F32 = ao.U, ao.F32
# what a weight may be off by where it is tiny: half the least step of its type, or, where that is less, 2^-126, below which the GPU's
# exponential (ex2.approx.ftz) gives 0
TINY = {t: max(x, 2.0 ** -126) for t, x in ao.TINY.items()}


def window_read(batch, tokens, window=None, sinks=0, lengths=None, device="cuda"):
    """[batch, tokens, tokens]: which keys each query reads."""
    i, j = torch.arange(tokens, device=device)[:, None], torch.arange(tokens, device=device)
    read = (j <= i) & ((i - j < (window or 1 << 40)) | (j < sinks))
    read = read.expand(batch, -1, -1)
    if lengths is not None:
        n = lengths.to(device).long()[:, None, None]
        read = read & (i < n) & (j < n)
    return read


def cached_read(tokens, table, pages, page_size, lengths, counts=None, tree=None, window=None, sinks=0):
    """[batch, tokens, places of the table], token by token from the definition."""
    batch, n = table.shape[0], table.shape[1] * page_size
    read = torch.zeros((batch, tokens, n), dtype=torch.bool)
    table, window = table.cpu().long(), window or 1 << 40
    for b in range(batch):
        held, fresh = max(0, int(lengths[b])), tokens if counts is None else min(max(0, int(counts[b])), tokens)
        row = None if tree is None else (tree[b] if tree.dim() == 3 else tree).cpu()
        for i in range(fresh):
            at = torch.arange(n)
            if row is None:
                place = held + i
                mine = (at <= place) & ((place - at < window) | (at < sinks))
            else:
                others = row[i, :fresh].clone()
                others[i] = False
                place = held + int(others.sum())
                mine = (at < held) & ((place - at < window) | (at < sinks))
                for j in range(fresh):
                    if row[i, j] and held + j < n:
                        mine[held + j] = True
            read[b, i] = mine & (at < held + fresh)
    there = (table >= 0) & (table < pages)
    return (read & there.repeat_interleave(page_size, 1)[:, None]).to(lengths.device)


def gathered(pool, table):
    """[batch, places, heads, dim]; zeros where there is no page."""
    there = (table >= 0) & (table < pool.shape[0])
    x = pool[torch.where(there, table, 0).long()] if len(pool) else pool.new_zeros((*table.shape, *pool.shape[1:]))
    return torch.where(there[:, :, None, None, None], x, torch.zeros_like(x)).flatten(1, 2)


def read_alone(x, read, group):
    """Keys or values in float64, zeros where no query of the sample reads, head by query head."""
    return torch.where(read.any(1)[:, :, None, None], x.double(), 0.0).repeat_interleave(group, 2)


def attention(q, k, v, read, scale):
    """(out, lse, P)"""
    group = q.shape[2] // k.shape[2]
    rows = read.any(2)
    q64 = torch.where(rows[:, :, None, None], q.double(), 0.0)
    k64, v64 = read_alone(k, read, group), read_alone(v, read, group)
    s = (torch.einsum("bshd,bnhd->bhsn", q64, k64) * scale).masked_fill(~read[:, None], -math.inf)
    lse = torch.logsumexp(s, -1) if s.shape[-1] else torch.full(s.shape[:-1], -math.inf, dtype=s.dtype, device=s.device)
    p = torch.where(read[:, None], (s - lse.masked_fill(lse == -math.inf, 0.0)[..., None]).exp(), 0.0)
    return torch.einsum("bhsn,bnhd->bshd", p, v64), lse, p


def score_error(q, k64, read, scale):
    rows = read.any(2)
    return ao.score_error(torch.where(rows[:, :, None, None], q.double(), 0.0), k64, scale)


def bound(q, k, v, out, p, read, scale):
    """P rounded to the tensors' type, sums in float32, the result rounded once (as attention_oracle.attention_bound)."""
    dtype, group, n = q.dtype, q.shape[2] // k.shape[2], k.shape[1]
    k64, v64 = read_alone(k, read, group), read_alone(v, read, group)
    a = torch.einsum("bhsn,bnhd->bshd", p, v64.abs())
    e = score_error(q, k64, read, scale)
    return U[dtype] * 1.01 * out.abs() + (U[dtype] * 1.01 + 2 * e + n * F32) * a + TINY[dtype] * (1 + v64.abs().sum(1, keepdim=True))


def lse_bound(q, k, read, lse, scale):
    """A sum of n float32 terms and the scores' own error; its logarithm, and the sum of the two, rounded."""
    e = score_error(q, read_alone(k, read, q.shape[2] // k.shape[2]), read, scale)
    return 2 * e + (k.shape[1] + 4) * F32 + 4 * F32 * lse.abs().nan_to_num(0, 0, 0)


def gradients(q, k, v, dout, read, scale, lse_grad=None):
    """(dq, dk, dv) and their bounds; rows that read nothing have none."""
    dtype, group, dim = q.dtype, q.shape[2] // k.shape[2], q.shape[-1]
    out, lse, p = attention(q, k, v, read, scale)
    rows = read.any(2)[:, :, None, None]
    q64, do = torch.where(rows, q.double(), 0.0), torch.where(rows, dout.double(), 0.0)
    k64, v64 = read_alone(k, read, group), read_alone(v, read, group)
    delta = (do * out).sum(-1).transpose(1, 2)
    if lse_grad is not None:
        delta = delta - torch.where(rows[:, :, :, 0].transpose(1, 2), lse_grad.double(), 0.0)
    ds = p * (torch.einsum("bshd,bnhd->bhsn", do, v64) - delta[..., None])

    def shared(x):   # sum over the query heads of a key head
        return x.view(*x.shape[:2], -1, group, dim).sum(3)

    dq = torch.einsum("bhsn,bnhd->bshd", ds, k64) * scale
    dk = shared(torch.einsum("bhsn,bshd->bnhd", ds, q64)) * scale
    dv = shared(torch.einsum("bhsn,bshd->bnhd", p, do))
    e = score_error(q, k64, read, scale)
    u = U[dtype] * 1.01
    # dS is rounded; P's error; dP in float32 sums of dim products; out comes in rounded, with what is off in it before
    off = ds.abs() * (u + 2 * e) + p * (
        2 * dim * F32 * torch.einsum("bshd,bnhd->bhsn", do.abs(), v64.abs()) + 2 * F32 * delta.abs()[..., None] +
        (u + dim * F32) * (do.abs() * out.abs()).sum(-1).transpose(1, 2)[..., None] +
        ((U[dtype] + 2 * e) * torch.einsum("bhsn,bnhd->bshd", p, v64.abs()) * do.abs()).sum(-1).transpose(1, 2)[..., None]
    ) + torch.where(read[:, None], TINY[dtype], 0.0)
    n, t = k.shape[1], q.shape[1] * group
    bq = u * dq.abs() + scale * torch.einsum("bhsn,bnhd->bshd", off, k64.abs()) * (1 + n * F32) + TINY[dtype]
    bk = u * dk.abs() + scale * shared(torch.einsum("bhsn,bshd->bnhd", off, q64.abs())) * (1 + t * F32) + TINY[dtype]
    offp = p * (u + 2 * e) + torch.where(read[:, None], TINY[dtype], 0.0)
    bv = u * dv.abs() + shared(torch.einsum("bhsn,bshd->bnhd", offp, do.abs())) * (1 + t * F32) + TINY[dtype]
    return (dq, dk, dv), (bq, bk, bv)
