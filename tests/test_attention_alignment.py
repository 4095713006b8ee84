"""Pointers that a kernel could not read by whole elements are refused at the C entry points, before a GPU is touched."""
import ctypes

import pytest


def _call(pkg, name, desc):
    lib = pkg._capi.load()
    rc = getattr(lib, name)(0, None, ctypes.byref(desc))
    return rc, lib.mlxd_last_error().decode()


AT = 1 << 20


def _rotary(capi, **change):
    heads = capi.Heads(AT, 4 * 3 * 64, 3 * 64, 64)
    d = capi.RotaryDesc(dtype=capi.BF16, batch=2, tokens=4, q_heads=3, k_heads=3, head_dim=64, q=heads, k=heads, q_out=heads,
                        k_out=heads, positions=AT, positions_dtype=capi.I64, frequencies=AT, n_axes=1, q_weight=AT, k_weight=AT,
                        weight_dtype=capi.F32, eps=1e-6, q_grad=heads, k_grad=heads, q_weight_grad=AT, k_weight_grad=AT, workspace=AT,
                        workspace_bytes=1 << 30)
    d.sections[0] = 32
    for k, v in change.items():
        setattr(d, k, v)
    return d


ENTRIES = ["mlxd_rotary", "mlxd_qk_norm_rotary", "mlxd_qk_norm_rotary_backward"]


@pytest.mark.parametrize("name", ["q", "k", "q_out", "k_out", "q_grad", "k_grad"])
@pytest.mark.parametrize("entry", ENTRIES)
def test_rotary_tensors(pkg, entry, name):
    capi = pkg._capi
    for dtype, off in ((capi.BF16, 1), (capi.F16, 3), (capi.F32, 2)):
        rc, why = _call(pkg, entry, _rotary(capi, dtype=dtype, **{name: capi.Heads(AT + off, 768, 192, 64)}))
        assert rc == capi.ERR_INVALID and "multiple of its element's size" in why


@pytest.mark.parametrize("entry", ENTRIES)
def test_rotary_vectors(pkg, entry):
    capi = pkg._capi
    changes = [dict(positions=AT + 4), dict(positions=AT + 2, positions_dtype=capi.I32), dict(frequencies=AT + 2)]
    if entry != "mlxd_rotary":
        changes += [dict(q_weight=AT + 2), dict(k_weight=AT + 1, weight_dtype=capi.F16)]
    if entry == "mlxd_qk_norm_rotary_backward":
        changes += [dict(q_weight_grad=AT + 2), dict(k_weight_grad=AT + 2), dict(workspace=AT + 4), dict(workspace=AT + 8)]
    for change in changes:
        rc, why = _call(pkg, entry, _rotary(capi, **change))
        assert rc == capi.ERR_INVALID and ("multiple of" in why or "16 bytes" in why), (change, why)


@pytest.mark.parametrize("entry", ["mlxd_cross_attention", "mlxd_cross_attention_backward"])
def test_cross(pkg, entry):
    capi = pkg._capi
    heads = capi.Heads(AT, 64 * 64, 64, 64)
    for change in (dict(lse=AT + 2), dict(lengths=AT + 4, lengths_dtype=capi.I64), dict(lengths=AT + 2, lengths_dtype=capi.I32),
                   dict(workspace=AT + 4), dict(workspace=AT + 8)):
        d = capi.CrossDesc(dtype=capi.BF16, batch=2, q_tokens=4, kv_tokens=6, q_heads=4, kv_heads=2, head_dim=64, scale=0.125, q=heads,
                           k=heads, v=heads, out=heads, lse=AT, dout=heads, dq=heads, dk=heads, dv=heads, workspace=AT,
                           workspace_bytes=1 << 30)
        for k, v in change.items():
            setattr(d, k, v)
        rc, why = _call(pkg, entry, d)
        assert rc == capi.ERR_INVALID and ("multiple of" in why or "16 bytes" in why), (change, why)


@pytest.mark.parametrize("entry", ENTRIES + ["mlxd_qk_norm_rotary_workspace"])
@pytest.mark.parametrize("name", ["q_heads", "k_heads"])
def test_more_heads_than_the_kernels_count(pkg, entry, name):
    """Numbers of heads near 2^31, whose sums and steps would not fit an int."""
    capi, lib = pkg._capi, pkg._capi.load()
    for heads in ((1 << 29) + 1, (1 << 31) - 1):
        d = _rotary(capi, **{name: heads})
        if entry.endswith("workspace"):
            size = ctypes.c_size_t()
            rc, why = getattr(lib, entry)(0, ctypes.byref(d), ctypes.byref(size)), lib.mlxd_last_error().decode()
        else:
            rc, why = _call(pkg, entry, d)
        assert rc == capi.ERR_INVALID and "2^29 heads" in why


def test_gradient_of_lse(pkg):
    capi, lib = pkg._capi, pkg._capi.load()
    heads = capi.Heads(AT, 64 * 64, 64, 64)
    d = capi.CrossDesc(dtype=capi.BF16, batch=2, q_tokens=4, kv_tokens=6, q_heads=4, kv_heads=2, head_dim=64, scale=0.125, q=heads,
                       k=heads, v=heads, out=heads, lse=AT, dout=heads, dq=heads, dk=heads, dv=heads, workspace=AT, workspace_bytes=1 << 30)
    rc = lib.mlxd_cross_attention_backward_lse(0, None, ctypes.byref(d), AT + 2)
    assert rc == capi.ERR_INVALID and "lse_grad" in lib.mlxd_last_error().decode()
