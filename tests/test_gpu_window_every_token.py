"""Long sequences without a window, both passes: whole against float64, and longer ones by stretches of queries."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402
import causal_oracle as co      # noqa: E402
from test_gpu_window_attention import check, make   # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype,batch,tokens,hq,hk,dim", [(BF16, 1, 3000, 4, 1, 128), (F16, 2, 1537, 3, 3, 64), (BF16, 2, 2048, 7, 1, 72)])
@pytest.mark.parametrize("ragged", [False, True])
def test_whole(pkg, dtype, batch, tokens, hq, hk, dim, ragged):
    q, k, v, dout = make(dtype, batch, tokens, hq, hk, dim, seed=tokens, packed=True)
    lengths = torch.tensor([tokens - 700, tokens][:batch], device="cuda") if ragged else None
    check(pkg, q, k, v, dout, lengths)


def test_by_stretches(pkg):
    """8192 tokens: every row of the forward pass and of dq, and what the stretches add to every key."""
    A = pkg.attention
    n, hq, step = 8192, 4, 1024
    q, k, v, dout = make(BF16, 1, n, hq, 2, 128)
    out, lse = A.window_attention(q, k, v, return_lse=True)
    dq, dk, dv = A.window_attention_backward(dout, q, k, v, out, lse)
    scale = float(torch.tensor(1 / math.sqrt(128)))
    want, bound = [torch.zeros(k.shape, dtype=torch.float64, device="cuda") for _ in range(2)], [torch.zeros(k.shape, dtype=torch.float64, device="cuda") for _ in range(2)]
    for first in range(0, n, step):
        rows, keys = slice(first, first + step), first + step
        a = (q[:, rows], k[:, :keys], v[:, :keys])
        read = (torch.arange(keys, device="cuda") <= torch.arange(first, keys, device="cuda")[:, None])[None]
        o, l, p = co.attention(*a, read, scale)
        ao.within(out[:, rows], o, co.bound(*a, o, p, read, scale))
        ao.within(lse[:, :, rows], l, co.lse_bound(a[0], a[1], read, l, scale))
        grads, bounds = co.gradients(*a, dout[:, rows], read, scale)
        ao.within(dq[:, rows], grads[0], bounds[0])
        for i in range(2):
            want[i][:, :keys] += grads[1 + i]
            bound[i][:, :keys] += bounds[1 + i]
    ao.within(dk, want[0], bound[0])
    ao.within(dv, want[1], bound[1])
