"""Training's form and generation's together: a sequence through window_attention at once, and through append_rotary and cached_attention by
prompt, chunk, draft and single tokens."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402
import causal_oracle as co      # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(None, 0), (48, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_text_read_at_once_and_piece_by_piece(pkg, dtype, window, sinks):
    A = pkg.attention
    b, n, hq, hk, dim, page = 2, 301, 8, 2, 64, 16
    gen = torch.Generator(device="cuda")
    gen.manual_seed(0)
    x = torch.randn((b, n, hq + 2 * hk, dim), generator=gen, device="cuda").to(dtype)
    q, k, v = x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:]
    f = 10000.0 ** (-torch.arange(dim // 2, device="cuda") / (dim // 2))
    places = torch.arange(n, device="cuda").expand(1, b, -1)
    qr, kr = A.rotary(q, k, places, f, (dim // 2,))
    whole = A.window_attention(qr, kr, v, window=window, sinks=sinks)
    scale = float(torch.tensor(1 / math.sqrt(dim)))
    read = co.window_read(b, n, window, sinks)
    want, _, p = co.attention(qr, kr, v, read, scale)
    bound = co.bound(qr, kr, v, want, p, read, scale)
    ao.within(whole, want, bound)

    kp = torch.full((64, page, hk, dim), math.nan, dtype=dtype, device="cuda")
    vp = torch.full_like(kp, math.nan)
    table = torch.randperm(64, generator=gen, device="cuda")[:2 * 22].view(2, 22)   # room for the drafts too
    held = torch.zeros(b, dtype=torch.int64, device="cuda")
    got = torch.zeros_like(want)
    at = [0, 0]

    def step(tokens, counts):
        """The next counts[b] tokens of each sample, in a batch padded to `tokens`."""
        qs, ks, vs = (torch.full((b, tokens, h, dim), math.nan, dtype=dtype, device="cuda") for h in (hq, hk, hk))
        for i in range(b):
            c = counts[i]
            qs[i, :c], ks[i, :c], vs[i, :c] = q[i, at[i]:at[i] + c], k[i, at[i]:at[i] + c], v[i, at[i]:at[i] + c]
        new = torch.tensor(counts, device="cuda")
        turned = A.append_rotary(qs, ks, vs, None, f, (dim // 2,), kp, vp, table, held, counts=new)
        out = A.cached_attention(turned, kp, vp, table, held, counts=new, window=window, sinks=sinks)
        for i in range(b):
            got[i, at[i]:at[i] + counts[i]] = out[i, :counts[i]].double()
            assert not out[i, counts[i]:].any()
            at[i] += counts[i]
        held.add_(new)

    step(140, [140, 77])                 # prompts of two lengths
    for _ in range(3):
        step(1, [1, 1])                  # single tokens
    step(50, [9, 50])                    # a chunk
    while min(at) < n:                   # the rest, a few at a time
        step(20, [min(20, n - at[0]), min(13, n - at[1])])
    ao.within(got, want, bound)

    # a tree of drafts whose one branch is the text that follows: the branch's rows are the text's
    back = 11
    held.fill_(n - back)
    branch = [3 * i for i in range(back)]            # the text's tokens among the drafted ones
    drafted = 3 * back
    draft = torch.randn((b, drafted, hq + 2 * hk, dim), generator=gen, device="cuda").to(dtype)
    draft[:, branch] = x[:, n - back:]
    parent = [(branch[i - 1] if i else -1) for i in range(back)]
    parents = {t: parent[i] for i, t in enumerate(branch)}
    for t in range(drafted):                         # others hang on the branch, two to a token
        parents.setdefault(t, t - t % 3)
    tree = torch.zeros((drafted, drafted), dtype=torch.bool)
    for t in range(drafted):
        a = t
        while a >= 0:
            tree[t, a] = True
            a = parents[a]
    depth = tree.sum(1) - 1
    qs, ks, vs = draft[:, :, :hq], draft[:, :, hq:hq + hk], draft[:, :, hq + hk:]
    turned = A.append_rotary(qs, ks, vs, (n - back + depth.cuda()).expand(1, b, -1), f, (dim // 2,), kp, vp, table, held)
    if window is None or window > back:              # the window does not cut the branch itself
        out = A.cached_attention(turned, kp, vp, table, held, tree=tree.cuda(), window=window, sinks=sinks)
        ao.within(out[:, branch], want[:, n - back:], bound[:, n - back:])


def test_training_step_through_rotation_and_window(pkg):
    """Gradients of the joint projection through rotation and attention, against float64 autograd of the plain form."""
    A = pkg.attention
    b, n, hq, hk, dim = 2, 130, 4, 2, 64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    x = torch.randn((b, n, hq + 2 * hk, dim), generator=gen, device="cuda").to(torch.bfloat16).requires_grad_()
    f = 100.0 ** (-torch.arange(dim // 2, device="cuda") / (dim // 2))
    places = torch.arange(n, device="cuda").expand(1, b, -1)
    lengths = torch.tensor([n, 90], device="cuda")
    dout = torch.randn((b, n, hq, dim), generator=gen, device="cuda").to(torch.bfloat16)
    q, k = A.rotary(x[:, :, :hq], x[:, :, hq:hq + hk], places, f, (dim // 2,))
    A.window_attention(q, k, x[:, :, hq + hk:], window=40, sinks=2, lengths=lengths).backward(dout)

    read = co.window_read(b, n, 40, 2, lengths)
    scale = float(torch.tensor(1 / math.sqrt(dim)))
    q, k, v = q.detach(), k.detach(), x.detach()[:, :, hq + hk:]
    (dq, dk, dv), (bq, bk, bv) = co.gradients(q, k, v, dout, read, scale)
    back = [ao.rotary(g, places, f, (dim // 2,), inverse=True) for g in (dq, dk)]
    # what is off in a pair's gradients is off in both of its elements after the rotation; one more rounding
    off = [ao.pair_size(e, dim // 2, False) + ao.rotary_bound(w, g.abs() + e, dim // 2, False, torch.bfloat16)
           for e, w, g in zip((bq, bk), back, (dq, dk))]
    want, bound = torch.cat((*back, dv), 2), torch.cat((*off, bv), 2)
    ao.within(x.grad, want, bound)
