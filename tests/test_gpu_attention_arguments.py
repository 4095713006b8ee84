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


@pytest.mark.parametrize("which", ["positions", "frequencies", "eps", "scale"])
@pytest.mark.parametrize("leaf", [True, False])
def test_gradients_that_are_not_worked_out(pkg, which, leaf):
    """A tensor that requires a gradient and would get none is refused; without gradients it is an ordinary argument."""
    A = pkg.attention
    q, positions, frequencies = _inputs(torch.bfloat16)
    q.requires_grad_(leaf)                      # alone, and beside inputs whose gradients are worked out
    eps, scale = torch.tensor(1e-6), torch.tensor(0.1)
    dict(positions=positions, frequencies=frequencies, eps=eps, scale=scale)[which].requires_grad_()
    calls = [lambda: A.rotary(q, q, positions, frequencies, (32,)), lambda: A.rotary(q, None, positions, frequencies, (32,), inverse=True),
             lambda: A.qk_norm_rotary(q, q, positions, frequencies, (32,), None, None, eps)]
    if which == "eps":
        calls = calls[2:]
    if which == "scale":
        calls = [lambda: A.cross_attention(q, q, q, scale=scale), lambda: A.cross_attention(q, q, q, scale=scale, return_lse=True)]
    for call in calls:
        with pytest.raises(ValueError, match=which):
            call()
        with torch.no_grad():
            call()
