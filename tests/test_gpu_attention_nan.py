"""Numbers that are none in what is read: they reach the rows that read them and no others, whichever way a call takes."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

# batch, tokens, keys, q heads, kv heads, head_dim: single tokens of one part, of some, of more than 32 parts; many queries
WAYS = [(1, 1, 50, 4, 2, 64), (1, 1, 1601, 32, 8, 128), (1, 1, 6404, 2, 1, 128), (2, 3, 700, 4, 4, 80),
        (1, 300, 385, 4, 2, 128), (2, 257, 130, 4, 2, 64)]


def _inputs(shape, dtype):
    b, t, n, hq, hk, d = shape
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    return [torch.randn(s, generator=gen, device="cuda").to(dtype) for s in ((b, t, hq, d), (b, n, hk, d), (b, n, hk, d))]


def _only(got, clean, rows):
    """Rows [batch, head, token] are not numbers, in the result and in lse; the others are what they were."""
    out, lse = got[0].transpose(1, 2), got[1]
    assert torch.isnan(out[rows]).all() and torch.isnan(lse[rows]).all()
    assert torch.equal(out[~rows], clean[0].transpose(1, 2)[~rows]) and torch.equal(lse[~rows], clean[1][~rows])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", WAYS)
def test_nan_in_a_query(pkg, shape, dtype):
    q, k, v = _inputs(shape, dtype)
    clean = pkg.attention.cross_attention(q, k, v, return_lse=True)
    q[-1, -1, 1, 3] = math.nan
    rows = torch.zeros(clean[1].shape, dtype=torch.bool, device="cuda")
    rows[-1, 1, -1] = True
    _only(pkg.attention.cross_attention(q, k, v, return_lse=True), clean, rows)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("key", [2, 19, 45])
@pytest.mark.parametrize("shape", WAYS)
def test_nan_in_a_key_that_is_read(pkg, shape, key, value):
    """A score that is not a number or is infinite leaves its rows without a number: exp(inf - inf)."""
    q, k, v = _inputs(shape, torch.bfloat16)
    q = q.abs()
    clean = pkg.attention.cross_attention(q, k, v, return_lse=True)
    k[0, key, 0, 5] = value
    rows = torch.zeros(clean[1].shape, dtype=torch.bool, device="cuda")
    rows[0, :shape[3] // shape[4]] = True
    _only(pkg.attention.cross_attention(q, k, v, return_lse=True), clean, rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("key", [0, 1, 16, 49, 64, 113, 127, 128, 352])
def test_nan_in_any_column_of_a_tile(pkg, key, dtype):
    """Of every eight pairs of keys the first is weighed in another way than the rest."""
    q, k, v = _inputs((1, 300, 385, 4, 2, 64), dtype)
    clean = pkg.attention.cross_attention(q, k, v, return_lse=True)
    k[0, key, 1, 0] = math.nan
    rows = torch.zeros(clean[1].shape, dtype=torch.bool, device="cuda")
    rows[0, 2:] = True
    _only(pkg.attention.cross_attention(q, k, v, return_lse=True), clean, rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", WAYS)
def test_gradients_beside_a_score_of_minus_infinity(pkg, shape, dtype):
    """A key whose scores are all -infinity is a key that is not read, for every gradient but the one that its infinity multiplies."""
    q, k, v = _inputs(shape, dtype)
    q[..., 0] = q[..., 0].abs() + 0.1
    dout = torch.randn_like(q)
    mask = torch.ones(k.shape[:2], dtype=torch.bool, device="cuda")
    mask[0, 19] = False

    def both(k, **how):
        out, lse = pkg.attention.cross_attention(q, k, v, return_lse=True, **how)
        return out, lse, *pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, **how)

    want = both(k, key_mask=mask)
    bad = k.clone()
    bad[0, 19, :, 0] = -math.inf
    out, lse, dq, dk, dv = both(bad)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert torch.equal(dq[..., 1:], want[2][..., 1:]) and torch.equal(dk, want[3]) and torch.equal(dv, want[4])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", WAYS)
def test_gradients_of_rows_without_weights(pkg, shape, dtype):
    """Scores that are all -infinity give zeros, lse of -infinity and no gradients to keys and values; neighbours keep theirs."""
    q, k, v = _inputs(shape, dtype)
    q[..., 0] = q[..., 0].abs() + 0.1
    dout = torch.randn_like(q)

    def both():
        out, lse = pkg.attention.cross_attention(q, k, v, return_lse=True)
        return out, lse, *pkg.attention.cross_attention_backward(dout, q, k, v, out, lse)

    clean = both()
    k[0, :, 0, 0] = -math.inf
    group = shape[3] // shape[4]
    out, lse, dq, dk, dv = both()
    assert not out[0, :, :group].any() and (lse[0, :group] == -math.inf).all()
    assert not dk[0, :, 0].any() and not dv[0, :, 0].any()
    assert not dq[0, :, :group, 1:].any()            # element 0 is 0 times the infinity in the keys
    for got, want in ((dq, clean[2]), (dk, clean[3]), (dv, clean[4])):
        heads = group if got is dq else 1
        assert torch.equal(got[:, :, heads:], want[:, :, heads:]) and torch.equal(got[1:], want[1:])


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("where", ["q", "dout"])
@pytest.mark.parametrize("kind", ["lengths", "mask"])
def test_keys_that_are_not_read_get_zeros(pkg, kind, where, value):
    """Also in a tile of which a part is read, and beside gradients that are not finite."""
    q, k, v = _inputs((2, 70, 300, 4, 2, 64), torch.float16)
    dout = torch.randn_like(q)
    {"q": q, "dout": dout}[where][:, 5, :, 3] = value
    read = torch.arange(300, device="cuda") < torch.tensor([100, 200], device="cuda")[:, None]
    args = dict(lengths=torch.tensor([100, 200], device="cuda"))
    if kind == "mask":
        read &= torch.arange(300, device="cuda") % 3 > 0
        args = dict(key_mask=read)
    out, lse = pkg.attention.cross_attention(q, k, v, return_lse=True, **args)
    dq, dk, dv = pkg.attention.cross_attention_backward(dout, q, k, v, out, lse, **args)
    assert not dk[~read].any() and not dv[~read].any()
    assert not torch.isfinite(dk[read]).all()
