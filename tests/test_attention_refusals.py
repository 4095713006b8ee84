"""What the attention operators refuse, at the C entry points (no GPU is touched before the checks) and in Python."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


def _call(pkg, name, desc):
    lib = pkg._capi.load()
    rc = getattr(lib, name)(0, None, ctypes.byref(desc))
    return rc, lib.mlxd_last_error().decode()


def _rotary(capi, **change):
    heads = capi.Heads(1 << 20, 4 * 3 * 64, 3 * 64, 64)
    d = capi.RotaryDesc(dtype=capi.BF16, batch=2, tokens=4, q_heads=3, k_heads=3, head_dim=64, q=heads, k=heads, q_out=heads,
                        k_out=heads, positions=1 << 20, positions_dtype=capi.I64, frequencies=1 << 20, n_axes=2,
                        weight_dtype=capi.F32, eps=1e-6, q_grad=heads, k_grad=heads)
    d.sections[0] = d.sections[1] = 16
    for k, v in change.items():
        if k == "sections":
            for i, x in enumerate(v):
                d.sections[i] = x
        else:
            setattr(d, k, v)
    return d


@pytest.mark.parametrize("entry", ["mlxd_rotary", "mlxd_qk_norm_rotary", "mlxd_qk_norm_rotary_backward"])
@pytest.mark.parametrize("change,text", [
    (dict(dtype=0), "float32, bfloat16 or float16"), (dict(dtype=99), "float32, bfloat16 or float16"),
    (dict(batch=-1), "negative size"), (dict(head_dim=63), "head_dim"), (dict(head_dim=258), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(n_axes=0), "axes"), (dict(n_axes=5), "axes"), (dict(sections=(16, 17)), "pairs"), (dict(sections=(0, 0)), "pairs"),
    (dict(sections=(-1, 4)), "negative section"), (dict(sections=(2 ** 31 - 1, 2 ** 31 - 1)), "pairs"),
    (dict(positions_dtype=0), "positions must be"), (dict(positions=None), "positions"), (dict(frequencies=None), "frequencies"),
])
def test_rotary_descriptors(pkg, entry, change, text):
    rc, why = _call(pkg, entry, _rotary(pkg._capi, **change))
    assert rc == pkg._capi.ERR_INVALID and text in why and entry[5:] in why


def test_norm_descriptors(pkg):
    capi = pkg._capi
    heads = capi.Heads(None, 0, 0, 0)
    for change, text in ((dict(weight_dtype=0), "weights must be"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                         (dict(q_out=heads), "q_out"), (dict(k=heads), "k and k_out")):
        rc, why = _call(pkg, "mlxd_qk_norm_rotary", _rotary(capi, **change))
        assert rc == capi.ERR_INVALID and text in why
    for change, text in ((dict(q_grad=heads), "q_grad"), (dict(q_weight=1 << 20), "come together"), (dict(k_weight_grad=1 << 20), "come together")):
        rc, why = _call(pkg, "mlxd_qk_norm_rotary_backward", _rotary(capi, **change))
        assert rc == capi.ERR_INVALID and text in why
    lib = capi.load()
    for entry in ("mlxd_rotary", "mlxd_qk_norm_rotary", "mlxd_qk_norm_rotary_backward"):
        assert getattr(lib, entry)(0, None, None) == capi.ERR_INVALID
    assert lib.mlxd_qk_norm_rotary_workspace(0, None, None) == capi.ERR_INVALID


def _cross(capi, **change):
    heads = capi.Heads(1 << 20, 64 * 64, 64, 64)
    d = capi.CrossDesc(dtype=capi.BF16, batch=2, q_tokens=4, kv_tokens=6, q_heads=4, kv_heads=2, head_dim=64, scale=0.125, q=heads,
                       k=heads, v=heads, out=heads, lse=1 << 20, dout=heads, dq=heads, dk=heads, dv=heads)
    for k, v in change.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("entry", ["mlxd_cross_attention", "mlxd_cross_attention_backward"])
@pytest.mark.parametrize("change,text", [
    (dict(dtype=1), "bfloat16 or float16"), (dict(dtype=-7), "bfloat16 or float16"), (dict(batch=-1), "negative size"),
    (dict(q_heads=3), "multiple of kv_heads"), (dict(kv_heads=0), "multiple of kv_heads"), (dict(head_dim=12), "head_dim"),
    (dict(head_dim=136), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(lengths=1 << 20, lengths_dtype=1), "lengths"),
    (dict(q_heads=1 << 24, kv_heads=1), "too many rows"),
])
def test_cross_descriptors(pkg, entry, change, text):
    rc, why = _call(pkg, entry, _cross(pkg._capi, **change))
    assert rc == pkg._capi.ERR_INVALID and text in why and entry[5:] in why


def test_cross_tensors(pkg):
    capi = pkg._capi
    for name in ("q", "k", "v", "out"):
        for heads, text in ((capi.Heads(None, 0, 0, 0), "is needed"), (capi.Heads((1 << 20) + 8, 4096, 64, 64), "16 bytes"),
                            (capi.Heads(1 << 20, 4096, 68, 64), "multiples of 8")):
            rc, why = _call(pkg, "mlxd_cross_attention", _cross(capi, **{name: heads}))
            assert rc == capi.ERR_INVALID and text in why and name in why
    rc, why = _call(pkg, "mlxd_cross_attention_backward", _cross(capi, lse=None))
    assert rc == capi.ERR_INVALID and "lse" in why
    rc, why = _call(pkg, "mlxd_cross_attention_backward", _cross(capi))
    assert rc == capi.ERR_INVALID and "workspace" in why
    lib = capi.load()
    for entry in ("mlxd_cross_attention", "mlxd_cross_attention_backward"):
        assert getattr(lib, entry)(0, None, None) == capi.ERR_INVALID
    assert lib.mlxd_cross_attention_workspace(0, None, 0, None) == capi.ERR_INVALID


def test_struct_sizes(pkg):
    capi = pkg._capi
    assert ctypes.sizeof(capi.Heads) == 32
    assert ctypes.sizeof(capi.RotaryDesc) == 24 + 4 * 32 + 8 + 8 + 24 + 8 + 4 + 16 + 12 + 16 + 8 + 2 * 32 + 32
    assert ctypes.sizeof(capi.CrossDesc) == 32 + 4 * 32 + 8 + 16 + 16 + 4 * 32 + 16


def test_host_tensors_are_refused(pkg):
    A = pkg.attention
    x, f = torch.zeros(1, 2, 2, 64), torch.ones(32)
    with pytest.raises(ValueError, match="no CPU path"):
        A.rotary(x, x, torch.zeros(1, 1, 2), f, (32,))
    with pytest.raises(ValueError, match="no CPU path"):
        A.cross_attention(x.half(), x.half(), x.half())
    with pytest.raises(ValueError, match="must be a torch tensor"):
        A.qk_norm_rotary(x.numpy(), None, torch.zeros(1, 1, 2), f, (32,))


@pytest.mark.gpu
def test_tensors_that_do_not_fit(pkg):
    A = pkg.attention
    x = torch.zeros(1, 2, 2, 64, device="cuda", dtype=torch.bfloat16)
    f, p = torch.ones(32, device="cuda"), torch.zeros(1, 1, 2, device="cuda")
    w = torch.ones(64, device="cuda")
    refused = [
        lambda: A.rotary(x.double(), x.double(), p, f, (32,)), lambda: A.rotary(x, x.float(), p, f, (32,)),
        lambda: A.rotary(x, x[..., :32], p, f, (32,)), lambda: A.rotary(x, x[:, :1], p, f, (32,)),
        lambda: A.rotary(x, x, p[0], f, (32,)), lambda: A.rotary(x, x, p[:, :, :1], f, (32,)), lambda: A.rotary(x, x, p, f, (16, 16)),
        lambda: A.rotary(x, x, p, f[:31], (32,)), lambda: A.rotary(x, x, p, f.double(), (32,)), lambda: A.rotary(x, x, p, f.cpu(), (32,)),
        lambda: A.rotary(x, x, p.double(), f, (32,)), lambda: A.rotary(x[0, 0], x[0, 0], p, f, (32,)),
        lambda: A.rotary(x, x, torch.zeros(5, 1, 2, device="cuda"), f, (8, 8, 8, 4, 4)),
        lambda: A.qk_norm_rotary(x, x, p, f, (32,), w[:32], w), lambda: A.qk_norm_rotary(x, x, p, f, (32,), w, w.half()),
        lambda: A.qk_norm_rotary(x, x, p, f, (32,), w.double(), None), lambda: A.qk_norm_rotary(x, x, p, f, (32,), w.cpu(), w.cpu()),
        lambda: A.qk_norm_rotary(x, x, p, f, (32,), w, w, -1.0),
        lambda: A.qk_norm_rotary_backward(x[:, :1], x, x, x, p, f, (32,)), lambda: A.qk_norm_rotary_backward(x, None, x, x, p, f, (32,)),
        lambda: A.cross_attention(x.float(), x.float(), x.float()), lambda: A.cross_attention(x, x.half(), x.half()),
        lambda: A.cross_attention(x, x, x[:, :1]), lambda: A.cross_attention(x, x[..., :32], x[..., :32]),
        lambda: A.cross_attention(x[0], x[0], x[0]), lambda: A.cross_attention(x[..., :60], x[..., :60], x[..., :60]),
        lambda: A.cross_attention(x, x, x, lengths=torch.zeros(2, device="cuda", dtype=torch.int32)),
        lambda: A.cross_attention(x, x, x, lengths=torch.zeros(1, device="cuda")),
        lambda: A.cross_attention(x, x, x, lengths=torch.zeros(1, dtype=torch.int32)),
        lambda: A.cross_attention(x, x, x, key_mask=torch.zeros(1, 2, device="cuda")),
        lambda: A.cross_attention(x, x, x, key_mask=torch.zeros(1, 3, device="cuda", dtype=torch.bool)),
        lambda: A.cross_attention(x, x, x, scale=float("inf")),
        lambda: A.cross_attention_backward(x, x, x, x, x, torch.zeros(1, 2, 3, device="cuda")),
        lambda: A.cross_attention_backward(x.half(), x, x, x, x, torch.zeros(1, 2, 2, device="cuda")),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was taken" % i)


@pytest.mark.parametrize("entry", ["mlxd_cross_attention", "mlxd_cross_attention_backward"])
@pytest.mark.parametrize("change,text", [(dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(kv_tokens=(1 << 30) + 1), "2^30"),
                                         (dict(batch=1 << 10, kv_tokens=1 << 30, q_heads=4, kv_heads=4), "too many keys")])
def test_cross_limits(pkg, entry, change, text):
    rc, why = _call(pkg, entry, _cross(pkg._capi, **change))
    assert rc == pkg._capi.ERR_INVALID and text in why


@pytest.mark.gpu
def test_self_check_word_is_clean(pkg):
    x = torch.randn(2, 200, 4, 64, device="cuda").to(torch.bfloat16)
    out, lse = pkg.attention.cross_attention(x, x, x, return_lse=True)
    pkg.attention.cross_attention_backward(x, x, x, x, out, lse)
    assert pkg._capi.attention_status(0, torch.cuda.current_stream().cuda_stream) == 0
    assert pkg._capi.load().mlxd_attention_status(0, None, None) == pkg._capi.ERR_INVALID


@pytest.mark.gpu
def test_keys_end_where_the_mask_does(pkg):
    """Under a mask whose last keys are not read the call gives what the shorter call gives."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    for tokens in (1, 300):
        q, k, v = (torch.randn(s, generator=gen, device="cuda").to(torch.float16)
                   for s in ((2, tokens, 4, 64), (2, 1500, 4, 64), (2, 1500, 4, 64)))
        for end in (0, 1, 127, 128, 129, 640, 641, 1499):
            mask = torch.zeros(2, 1500, dtype=torch.bool, device="cuda")
            mask[:, :end] = True
            got = pkg.attention.cross_attention(q, k, v, key_mask=mask)
            want = pkg.attention.cross_attention(q, k, v, lengths=torch.tensor([end, end], device="cuda"))
            assert torch.equal(got, want)
