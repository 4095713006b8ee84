"""Arguments of the attention operators that would do something else than they say."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def _inputs(dtype=torch.float32):
    q = torch.randn(1, 2, 2, 64, device="cuda").to(dtype)
    return q, torch.zeros(1, 1, 2, device="cuda"), torch.ones(32, device="cuda")


@pytest.mark.parametrize("sections", [(16.5,), ("32",), (1 << 40,), (None,), (32 + 0j,)])
def test_sections_that_are_no_whole_numbers(pkg, sections):
    q, positions, frequencies = _inputs()
    with pytest.raises(ValueError, match="sections"):
        pkg.attention.rotary(q, q, positions, frequencies, sections)
    with pytest.raises(ValueError, match="sections"):
        pkg.attention.qk_norm_rotary(q, q, positions, frequencies, sections)


@pytest.mark.parametrize("scale", ["0.1", (0.1,), 1j])
def test_scale_that_is_no_number(pkg, scale):
    q, _, _ = _inputs(torch.bfloat16)
    with pytest.raises(ValueError, match="scale"):
        pkg.attention.cross_attention(q, q, q, scale=scale)
