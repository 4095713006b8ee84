"""A query that reads one key: lse is its score, so a gradient of lse is the gradient of the score, and nothing else is."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402
import causal_oracle as co      # noqa: E402
from test_gpu_window_attention import make   # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,window", [(1, None), (1, 5), (700, 1)])
def test_gradient_of_lse_alone(pkg, dtype, tokens, window):
    A = pkg.attention
    q, k, v, dout = make(dtype, 3, tokens, 8, 2, 128, seed=2)
    out, lse = A.window_attention(q, k, v, window=window, return_lse=True)
    plain = A.window_attention_backward(dout, q, k, v, out, lse, window=window)
    g = torch.randn((3, 8, tokens), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    dq, dk, dv = A.window_attention_backward(dout, q, k, v, out, lse, window=window, lse_grad=g)
    assert torch.equal(dv, plain[2])
    scale = float(torch.tensor(1 / math.sqrt(128)))
    ds = g.double().transpose(1, 2)[..., None]                             # [batch, tokens, heads, 1]
    q64, do, k64, v64 = q.double(), dout.double(), k.double().repeat_interleave(4, 2), v.double().repeat_interleave(4, 2)

    def shared(x):
        return x.view(3, tokens, 2, 4, 128).sum(3)

    # dS = P (dP - delta) is rounded to the type; delta is dP less the gradient of lse in float32, dP a float32 sum of 128 products that the
    # kernel for keys takes in another order; there P comes from the score and lse, each off as scores are (P is 1 but for that)
    e = ao.score_error(q, k64, scale)
    u = co.U[dtype] * 1.01
    off = ds.abs() * (u + 2 * e) + 4 * 128 * co.F32 * (do.abs() * v64.abs()).sum(-1, keepdim=True) + 4 * co.F32 * ds.abs() + co.TINY[dtype]
    want = scale * ds * k64
    ao.within(dq, want, u * want.abs() + scale * off * k64.abs() + co.TINY[dtype])
    want = shared(scale * ds * q64)
    ao.within(dk, want, u * want.abs() + scale * shared(off * q64.abs()) * (1 + 8 * co.F32) + co.TINY[dtype])
