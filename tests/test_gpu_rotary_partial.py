"""Heads of which a part is turned: the other elements stay as they are, bit by bit, whatever lies beside them."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# head_dim, pairs turned: vectors of 16 bytes, of 8, single elements; ends of the turned part inside a vector
PARTS = [(64, 16), (128, 48), (128, 8), (72, 12), (72, 8), (34, 5), (96, 13), (256, 4), (6, 1)]


def _inputs(dtype, dim, pairs):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(pairs)
    x = torch.randn((2, 5, 3, dim), generator=gen, device="cuda").to(dtype)
    positions = torch.randint(1, 4000, (1, 2, 5), generator=gen, device="cuda")
    frequencies = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=F32) / pairs)
    return x, positions, frequencies


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("dim,pairs", PARTS)
def test_elements_that_pass_through(pkg, dtype, adjacent, dim, pairs):
    x, positions, frequencies = _inputs(dtype, dim, pairs)
    turned = pkg.attention.rotary(x, None, positions, frequencies, (pairs,), adjacent=adjacent)[0][..., :2 * pairs]
    for at in range(2 * pairs, dim):
        for value in (math.inf, -math.inf, -0.0):
            y = x.clone()
            y[0, at % 5, at % 3, at] = value
            y[1, :, :, at] = value
            for inverse in (False, True):
                got = pkg.attention.rotary(y, y, positions, frequencies, (pairs,), adjacent=adjacent, inverse=inverse)
                for g in got:
                    assert torch.equal(g[..., 2 * pairs:], y[..., 2 * pairs:])
                    assert torch.equal(g[..., 2 * pairs:].signbit(), y[..., 2 * pairs:].signbit())
                if not inverse:
                    assert torch.equal(got[0][..., :2 * pairs], turned)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("dim,pairs", PARTS)
def test_norm_beside_an_infinity(pkg, dtype, adjacent, dim, pairs):
    """The norm of a head with an infinity leaves zeros but for that element; an infinite gradient reaches its own weight's alone."""
    x, positions, frequencies = _inputs(dtype, dim, pairs)
    w = torch.ones(dim, device="cuda")
    for at in (2 * pairs, (2 * pairs + dim) // 2, dim - 1):
        y = x.clone()
        y[1, 2, 1, at] = math.inf
        got = pkg.attention.qk_norm_rotary(y, None, positions, frequencies, (pairs,), w, adjacent=adjacent)[0][1, 2, 1]
        rest = torch.arange(dim, device="cuda") != at
        assert torch.isnan(got[at]) and not got[rest].any()
        dy = torch.ones_like(x)
        dy[1, 2, 1, at] = math.inf
        dw = pkg.attention.qk_norm_rotary_backward(dy, None, x, None, positions, frequencies, (pairs,), w, adjacent=adjacent)[2]
        assert torch.isfinite(dw[rest]).all() and torch.isinf(dw[at])
