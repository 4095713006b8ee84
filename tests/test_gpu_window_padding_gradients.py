"""Gradients behind a sequence's length are zeros whatever the sequence itself holds."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_window_attention import make   # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype,tokens,hq,hk,dim,window,sinks", [
    (torch.bfloat16, 40, 2, 1, 64, None, 0), (torch.float16, 260, 4, 2, 128, None, 0), (torch.bfloat16, 700, 8, 2, 128, 300, 4),
    (torch.float16, 900, 3, 3, 72, 500, 130)])
@pytest.mark.parametrize("of", ["q", "k", "v", "dout"])
def test_rows_behind_a_length(pkg, what, dtype, tokens, hq, hk, dim, window, sinks, of):
    q, k, v, dout = make(dtype, 3, tokens, hq, hk, dim)
    lengths = torch.tensor([tokens - 5, 0, tokens // 2 + 1], device="cuda")
    x = dict(q=q, k=k, v=v, dout=dout)
    for b in (0, 2):
        x[of][b, int(lengths[b]) - 2] = what
    how = dict(window=window, sinks=sinks, lengths=lengths)
    out, lse = pkg.attention.window_attention(q, k, v, return_lse=True, **how)
    grads = pkg.attention.window_attention_backward(dout, q, k, v, out, lse, **how)
    for b in range(3):
        n = int(lengths[b])
        assert not out[b, n:].any() and (lse[b, :, n:] == -math.inf).all()
        for name, g in zip(("dq", "dk", "dv"), grads):
            assert not g[b, n:].any(), name
