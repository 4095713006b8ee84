"""A first backward kernel whose last CTA takes longer than the limit of any wait inside the second."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_keys_for_seconds(pkg):
    """One query row over 2^29 keys of 8 elements is about three seconds of one CTA, while the other kernel's have begun beside it."""
    keys, dim = 1 << 29, 8
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GB")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(0)
    few = torch.randn((1, 1 << 16, 1, dim), generator=gen, device="cuda").to(torch.bfloat16)
    k = few.repeat(1, keys >> 16, 1, 1)
    v = k.roll(1, 3)
    q, dout = (torch.randn((1, 1, 1, dim), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    out, lse = pkg.attention.cross_attention(q, k, v, return_lse=True)
    dq, dk, dv = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse)
    assert pkg._capi.attention_status(0, torch.cuda.current_stream().cuda_stream) == 0
    # the keys repeat, and so do their gradients, bit by bit
    for g in (dk, dv):
        first = g[:, :1 << 16]
        assert torch.isfinite(first).all() and first.any()
        for at in range(0, keys, 1 << 24):
            part = g[:, at:at + (1 << 24)].unflatten(1, (-1, 1 << 16))
            assert torch.equal(part, first[:, None].expand_as(part))
