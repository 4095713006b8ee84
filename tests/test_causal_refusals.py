"""What cached and window attention and appends to a cache refuse at the C entry points (no GPU is touched before the checks)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
AT = 1 << 20


def _call(pkg, name, desc):
    lib = pkg._capi.load()
    rc = getattr(lib, name)(0, None, ctypes.byref(desc))
    return rc, lib.mlxd_last_error().decode()


def _change(d, change):
    for name, value in change.items():
        at = d
        *path, last = name.split("__")
        for x in path:
            at = getattr(at, x)
        if last == "sections":
            for i, x in enumerate(value):
                at.sections[i] = x
        else:
            setattr(at, last, value)
    return d


def _cache(capi):
    pages = capi.Pages(AT, 16 * 2 * 64, 2 * 64, 64)
    return capi.Cache(k=pages, v=pages, pages=9, page_size=16, page_table=AT, page_table_dtype=capi.I32, table_width=4, page_table_stride=4,
                      lengths=AT, counts=AT, lengths_dtype=capi.I64, counts_dtype=capi.I32)


def _append(capi, **change):
    heads = capi.Heads(AT, 64 * 64, 2 * 64, 64)
    d = capi.AppendDesc(r=capi.RotaryDesc(dtype=capi.BF16, batch=2, tokens=4, q_heads=4, k_heads=2, head_dim=64, q=heads, k=heads, q_out=heads,
                                          positions=AT, positions_dtype=capi.I64, frequencies=AT, n_axes=1), v=heads, cache=_cache(capi))
    d.r.sections[0] = 32
    return _change(d, change)


def _cached(capi, **change):
    heads = capi.Heads(AT, 64 * 64, 4 * 64, 64)
    d = capi.CachedDesc(dtype=capi.BF16, batch=2, tokens=4, q_heads=4, kv_heads=2, head_dim=64, scale=0.125, q=heads, out=heads, lse=AT,
                        cache=_cache(capi))
    return _change(d, change)


def _window(capi, **change):
    heads = capi.Heads(AT, 64 * 64, 4 * 64, 64)
    d = capi.WindowDesc(dtype=capi.BF16, batch=2, tokens=4, q_heads=4, kv_heads=2, head_dim=64, scale=0.125, q=heads, k=heads, v=heads,
                        out=heads, lse=AT, dout=heads, dq=heads, dk=heads, dv=heads, workspace=AT, workspace_bytes=1 << 20)
    return _change(d, change)


CACHE = [
    (dict(cache__pages=-1), "negative size"), (dict(cache__table_width=-2), "negative size"), (dict(cache__page_size=0), "page_size"),
    (dict(cache__page_size=4), "page_size"), (dict(cache__page_size=24), "page_size"), (dict(cache__page_size=-16), "page_size"),
    (dict(cache__table_width=1 << 27), "2^30 places"), (dict(cache__page_table_dtype=2), "page_table must be"),
    (dict(cache__lengths_dtype=0), "lengths must be"), (dict(cache__counts_dtype=1), "counts must be"), (dict(cache__lengths=None), "lengths are needed"),
    (dict(cache__page_table=None), "page_table is needed"), (dict(cache__page_table=AT + 2), "page_table does not start"),
    (dict(cache__lengths=AT + 4), "lengths does not start"), (dict(cache__counts=AT + 1), "counts does not start"),
]


@pytest.mark.parametrize("change,text", CACHE + [
    (dict(r__dtype=99), "float32, bfloat16 or float16"), (dict(r__batch=-1), "negative size"), (dict(r__head_dim=63), "head_dim"),
    (dict(r__n_axes=5), "axes"), (dict(r__sections=(33,)), "pairs"), (dict(r__positions_dtype=0), "positions must be"),
    (dict(r__frequencies=None), "frequencies"), (dict(r__k_heads=0), "keys and values"), (dict(r__inverse=1), "inverse"),
    (dict(r__q_out__data=None), "q and q_out"), (dict(r__k__data=None), "k and v"), (dict(v__data=None), "k and v"),
    (dict(cache__k__data=None), "pages are needed"), (dict(cache__v__data=None), "pages are needed"),
    (dict(v__data=AT + 1), "multiple of its element"), (dict(cache__v__data=AT + 1), "multiple of its element"),
    (dict(r__positions=AT + 4), "positions"), (dict(r__tokens=1 << 30, r__batch=1), "2^30 tokens"),
])
def test_append_descriptors(pkg, change, text):
    rc, why = _call(pkg, "mlxd_append_rotary", _append(pkg._capi, **change))
    assert rc == pkg._capi.ERR_INVALID and text in why and "append_rotary" in why


SIZES = [
    (dict(dtype=1), "bfloat16 or float16"), (dict(batch=-1), "negative size"), (dict(tokens=-4), "negative size"),
    (dict(q_heads=3), "multiple of kv_heads"), (dict(kv_heads=0), "multiple of kv_heads"), (dict(head_dim=12), "head_dim"),
    (dict(head_dim=136), "head_dim"), (dict(tokens=1 << 30), "2^30 tokens"), (dict(q_heads=1 << 24, kv_heads=1), "too many rows"),
    (dict(window=-1), "window and sinks"), (dict(sinks=-1), "window and sinks"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(lse=AT + 2), "lse does not start"), (dict(workspace=AT + 8), "workspace must start"),
]


@pytest.mark.parametrize("change,text", SIZES + CACHE + [
    (dict(q__data=None), "q is needed"), (dict(out__data=AT + 8), "out must start"), (dict(q__stride_token=68), "q must start"),
    (dict(cache__k__data=None), "k_pages is needed"), (dict(cache__v__data=AT + 8), "v_pages must start"),
    (dict(cache__v__stride_row=132), "v_pages must start"), (dict(cache__k__stride_page=2052), "k_pages must start"),
    (dict(tree=AT, tokens=1 << 17), "tree of more"),
])
def test_cached_descriptors(pkg, change, text):
    rc, why = _call(pkg, "mlxd_cached_attention", _cached(pkg._capi, **change))
    assert rc == pkg._capi.ERR_INVALID and text in why and "cached_attention" in why


@pytest.mark.parametrize("entry", ["mlxd_window_attention", "mlxd_window_attention_backward"])
@pytest.mark.parametrize("change,text", SIZES + [
    (dict(lengths=AT, lengths_dtype=1), "lengths must be"), (dict(lengths=AT + 4, lengths_dtype=4), "lengths"),
    (dict(q__data=None), "q is needed"), (dict(k__data=AT + 8), "k must start"), (dict(v__stride_head=4), "v must start"),
])
def test_window_descriptors(pkg, entry, change, text):
    capi = pkg._capi
    if change.get("lengths_dtype") == 4:
        change = dict(change, lengths_dtype=capi.I64)
    rc, why = _call(pkg, entry, _window(capi, **change))
    assert rc == capi.ERR_INVALID and text in why and entry[5:] in why


@pytest.mark.parametrize("change,text", [
    (dict(dout__data=None), "dout is needed"), (dict(dk__data=AT + 4), "dk must start"), (dict(lse=None), "lse is needed"),
    (dict(lse_grad=AT + 1), "lse_grad"), (dict(workspace=None), "workspace too small"), (dict(workspace_bytes=3), "workspace too small"),
])
def test_window_backward_descriptors(pkg, change, text):
    rc, why = _call(pkg, "mlxd_window_attention_backward", _window(pkg._capi, **change))
    assert rc == pkg._capi.ERR_INVALID and text in why


def test_null_descriptors_and_sizes(pkg):
    capi, lib = pkg._capi, pkg._capi.load()
    for entry in ("mlxd_append_rotary", "mlxd_cached_attention", "mlxd_window_attention", "mlxd_window_attention_backward"):
        assert getattr(lib, entry)(0, None, None) == capi.ERR_INVALID
    assert lib.mlxd_cached_attention_workspace(0, None, None) == capi.ERR_INVALID
    assert lib.mlxd_window_attention_workspace(0, None, 1, None) == capi.ERR_INVALID
    assert lib.mlxd_cached_attention_workspace(0, ctypes.byref(_cached(capi)), None) == capi.ERR_INVALID
    bytes_ = ctypes.c_size_t()
    assert lib.mlxd_window_attention_workspace(0, ctypes.byref(_window(capi)), 1, ctypes.byref(bytes_)) == capi.OK
    assert bytes_.value >= 2 * 4 * 4 * 4
    assert ctypes.sizeof(capi.Cache) == 2 * 32 + 8 + 8 + 8 + 8 + 16 + 8
    assert ctypes.sizeof(capi.AppendDesc) == ctypes.sizeof(capi.RotaryDesc) + 32 + ctypes.sizeof(capi.Cache)
    assert ctypes.sizeof(capi.CachedDesc) == 40 + 64 + 8 + ctypes.sizeof(capi.Cache) + 24 + 16
    assert ctypes.sizeof(capi.WindowDesc) == 40 + 4 * 32 + 8 + 8 + 8 + 4 * 32 + 8 + 16


def test_host_tensors_are_refused(pkg):
    A = pkg.attention
    x, f, n = torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16), torch.ones(32), torch.zeros(1, dtype=torch.int32)
    pool, table = torch.zeros(2, 8, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU path"):
        A.append_rotary(x, x, x, None, f, (32,), pool, pool, table, n)
    with pytest.raises(ValueError, match="no CPU path"):
        A.cached_attention(x, pool, pool, table, n)
    with pytest.raises(ValueError, match="no CPU path"):
        A.window_attention(x, x, x)
    with pytest.raises(ValueError, match="no CPU path"):
        A.window_attention_backward(x, x, x, x, x, torch.zeros(1, 2, 2))
