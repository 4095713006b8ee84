"""Queries behind a sample's count have no effect and get zeros, infinities among them: one element of a query makes its scores infinite."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_cached_attention import check, make, random_tree   # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype,tokens,hq,hk,dim", [(BF16, 2, 8, 2, 128), (F16, 1, 16, 1, 64), (BF16, 4, 4, 1, 64), (F16, 16, 1, 1, 128), (BF16, 20, 8, 2, 128),
                                                    (F16, 150, 2, 1, 64)])
@pytest.mark.parametrize("lengths", [[1600, 333, 40], [9000, 17, 2000]])
@pytest.mark.parametrize("how", [dict(), dict(window=100, sinks=20)])
def test_padded_queries(pkg, what, dtype, tokens, hq, hk, dim, lengths, how):
    counts = torch.tensor([tokens // 2, 0, tokens], device="cuda")
    q, *rest = make(dtype, 3, tokens, hq, hk, dim, 16, lengths, counts=counts)
    for b in range(3):
        q[b, int(counts[b]):, :, 0] = what
    for tree in (None, random_tree(tokens, 4, 3)):
        out, lse = check(pkg, q, *rest, counts=counts, tree=tree, **how)
        for b in range(3):
            assert not out[b, int(counts[b]):].any() and (lse[b, :, int(counts[b]):] == -math.inf).all()
