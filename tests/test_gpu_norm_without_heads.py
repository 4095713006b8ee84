"""The norm's backward pass where there are no heads: the weights' gradients are sums of nothing."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(0, 0), (0, None), (2, 0), (0, 2)])
def test_weight_gradients(pkg, heads, wdtype):
    dim = 64
    hq, hk = heads
    q = torch.randn(2, 3, hq, dim, device="cuda")
    k = None if hk is None else torch.randn(2, 3, hk, dim, device="cuda")
    w = torch.ones(dim, device="cuda", dtype=wdtype)
    wk = None if hk is None else w
    positions = torch.arange(6, device="cuda").view(1, 2, 3)
    frequencies = torch.ones(dim // 2, device="cuda")
    for _ in range(2):
        used = [torch.full((dim,), math.nan, device="cuda", dtype=wdtype) for _ in range(8)]   # what the allocator hands out next
        del used
        dq, dk, dwq, dwk = pkg.attention.qk_norm_rotary_backward(q, k, q, k, positions, frequencies, (dim // 2,), w, wk)
        assert dq.shape == q.shape and (k is None or dk.shape == k.shape)
        for dw, n in ((dwq, hq), (dwk, hk)):
            if n == 0:
                assert torch.equal(dw, torch.zeros_like(w))
            elif n:
                assert torch.isfinite(dw).all() and dw.any()
