"""How much room the backward pass of window attention asks for with many first tokens that stay visible (no GPU is touched)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


def workspace(pkg, batch, tokens, hq, hk, dim, window, sinks):
    capi = pkg._capi
    d = capi.WindowDesc(dtype=capi.BF16, batch=batch, tokens=tokens, q_heads=hq, kv_heads=hk, head_dim=dim, scale=1, window=window, sinks=sinks)
    n = ctypes.c_size_t()
    assert capi.load().mlxd_window_attention_workspace(0, ctypes.byref(d), 1, ctypes.byref(n)) == capi.OK
    return n.value


@pytest.mark.parametrize("batch,tokens,hq,hk,window,sinks", [
    (4, 131072, 32, 32, 16, 8192), (1, 32768, 32, 8, 512, 16384), (1, 1 << 20, 8, 1, 16, 1 << 19), (64, 16384, 32, 32, 100, 4),
    (1, 131072, 8, 1, 16, 1 << 30), (16, 8192, 32, 8, 128, 4)])
def test_room_for_parts_is_bounded(pkg, batch, tokens, hq, hk, window, sinks):
    """Beside 8 bytes a row: 1024 tiles of float32 dk and dv."""
    rows = 8 * batch * hq * tokens
    assert rows <= workspace(pkg, batch, tokens, hq, hk, 128, window, sinks) <= rows + 16 + 1024 * 2 * 128 * 128 * 4


@pytest.mark.parametrize("tokens,hq,hk,window,sinks,parts", [(16384, 32, 8, 2048, 4, 7), (16384, 2, 1, 700, 3, 16), (4096, 8, 8, 512, 0, 1)])
def test_few_first_tokens_are_split(pkg, tokens, hq, hk, window, sinks, parts):
    more = workspace(pkg, 1, tokens, hq, hk, 128, window, sinks) - 8 * hq * tokens
    assert more == (0 if parts == 1 else parts * hk * 2 * 128 * 128 * 4)
