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


@pytest.mark.parametrize("requires", [False, True])
def test_forward_mode_is_refused(pkg, requires):
    """A tangent would be dropped and read as zero."""
    A = pkg.attention
    q, positions, frequencies = _inputs(torch.bfloat16)
    w = torch.ones(64, device="cuda")
    fw = torch.autograd.forward_ad

    def calls(dual, f, weight):
        return [lambda: A.rotary(dual, q, positions, f, (32,)), lambda: A.rotary(q, dual, positions, f, (32,), inverse=True),
                lambda: A.qk_norm_rotary(dual, None, positions, f, (32,), weight), lambda: A.qk_norm_rotary(q, None, positions, f, (32,), weight),
                lambda: A.cross_attention(dual, q, q), lambda: A.cross_attention(q, dual, q), lambda: A.cross_attention(q, q, dual)]

    with fw.dual_level():
        dual = fw.make_dual(q.detach().clone().requires_grad_(requires), torch.ones_like(q))
        for i, call in enumerate(calls(dual, frequencies, w)):
            if i != 3:
                with pytest.raises((ValueError, NotImplementedError) if requires else ValueError):
                    call()
        with pytest.raises(ValueError):
            A.rotary(q, q, positions, fw.make_dual(frequencies, torch.ones_like(frequencies)), (32,))
        with pytest.raises(ValueError):
            calls(q, frequencies, fw.make_dual(w, torch.ones_like(w)))[3]()
        for call in calls(q, frequencies, w):          # nothing carries a tangent
            call()


def test_arguments_that_change_between_the_passes(pkg):
    """The backward pass uses what the forward pass was given: sections in a list, numbers in tensors."""
    A = pkg.attention
    q, positions, _ = _inputs()
    positions = torch.stack((positions[0] + 3, positions[0] + 7))
    frequencies, w = torch.rand(32, device="cuda"), torch.ones(64, device="cuda")
    dy = torch.randn_like(q)

    def gradients(change):
        sections, eps, scale = [8, 24], torch.tensor(1e-2), torch.tensor(0.3)
        x, z, h = (t.detach().clone().requires_grad_() for t in (q, q, q.bfloat16()))
        y = A.rotary(x, None, positions, frequencies, sections)[0]
        n = A.qk_norm_rotary(z, None, positions, frequencies, sections, w, None, eps)[0]
        c = A.cross_attention(h, h, h, scale=scale)
        if change:
            sections[:] = [24, 8]
            eps.fill_(1.0)
            scale.fill_(2.0)
        torch.autograd.backward((y, n, c), (dy, dy, dy.bfloat16()))
        return x.grad, z.grad, h.grad

    assert all(torch.equal(a, b) for a, b in zip(gradients(True), gradients(False)))


def test_wrong_arguments_beside_gradients(pkg):
    """They are seen before anything is kept for the backward pass."""
    A = pkg.attention
    q, positions, frequencies = _inputs()
    q.requires_grad_()
    for call in (lambda: A.rotary(q, None, positions.cpu().numpy(), frequencies, (32,)), lambda: A.rotary(q, q.detach().cpu().numpy(), positions, frequencies, (32,)),
                 lambda: A.qk_norm_rotary(q, None, positions, [1.0] * 32, (32,)), lambda: A.qk_norm_rotary(q, None, positions, frequencies, (32,), 1.0),
                 lambda: A.cross_attention(q, q, q), lambda: A.cross_attention(q.bfloat16(), q.bfloat16(), q.bfloat16(), lengths=[1])):
        with pytest.raises(ValueError):
            call()
