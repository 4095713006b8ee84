"""Branches of drafts longer than the window.  New tokens are read by the tree alone, so a caller takes far ancestors out of it (first
tokens that stay visible stay in); the window over the cache follows, and rows are those of window_attention."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402
import causal_oracle as co      # noqa: E402
from test_gpu_cached_attention import check   # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hq,hk,dim", [(torch.bfloat16, 8, 2, 128), (torch.float16, 1, 1, 64)])
@pytest.mark.parametrize("held,drafts,window,sinks", [(90, 20, 16, 0), (90, 15, 4, 4), (2, 40, 16, 4), (0, 30, 7, 3), (300, 150, 100, 130), (50, 9, 1, 1)])
def test_chains_beyond_the_window(pkg, dtype, hq, hk, dim, held, drafts, window, sinks):
    n, page = held + drafts, 16
    gen = torch.Generator(device="cuda")
    gen.manual_seed(held + drafts)
    q, k, v = (torch.randn((1, n, h, dim), generator=gen, device="cuda").to(dtype) for h in (hq, hk, hk))
    whole, lse = pkg.attention.window_attention(q, k, v, window=window, sinks=sinks, return_lse=True)
    pages = (n + page - 1) // page
    kp, vp = (torch.full((pages, page, hk, dim), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    kp.view(-1, hk, dim)[:n], vp.view(-1, hk, dim)[:n] = k[0], v[0]
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    i, j = torch.arange(drafts, device="cuda")[:, None], torch.arange(drafts, device="cuda")
    chain = j <= i
    near = chain & ((i - j < window) | (held + j < sinks))
    how = dict(window=window, sinks=sinks)
    # by the definition of the tree; and the text's own rows where far ancestors are taken out
    check(pkg, q[:, held:].contiguous(), kp, vp, table, torch.tensor([held], device="cuda"), tree=chain, **how)
    out, lse_drafts = check(pkg, q[:, held:].contiguous(), kp, vp, table, torch.tensor([held], device="cuda"), tree=near, **how)
    scale = float(torch.tensor(1 / math.sqrt(dim)))
    read = co.window_read(1, n, window, sinks)
    want, want_lse, p = co.attention(q, k, v, read, scale)
    bound = co.bound(q, k, v, want, p, read, scale)
    ao.within(whole, want, bound)
    ao.within(out, want[:, held:], bound[:, held:])
    ao.within(lse_drafts, want_lse[:, :, held:], co.lse_bound(q, k, read, want_lse, scale)[:, :, held:])
