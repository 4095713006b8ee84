"""Gradients of first tokens that stay visible, whose queries are split among CTAs and whose parts are added: all keys against float64."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402
import causal_oracle as co      # noqa: E402
from test_gpu_window_attention import check, make   # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def splits(pkg, batch, tokens, hq, hk, dim, window, sinks):
    """Whether the call asks for room for parts, beside what it keeps of each row."""
    capi = pkg._capi
    d = capi.WindowDesc(dtype=capi.BF16, batch=batch, tokens=tokens, q_heads=hq, kv_heads=hk, head_dim=dim, scale=1, window=window, sinks=sinks)
    n = ctypes.c_size_t()
    assert capi.load().mlxd_window_attention_workspace(0, ctypes.byref(d), 1, ctypes.byref(n)) == capi.OK
    return n.value > 8 * batch * hq * tokens + 16


@pytest.mark.parametrize("dtype,batch,tokens,hq,hk,dim,window,sinks", [
    (BF16, 1, 2100, 8, 1, 64, 16, 3), (F16, 1, 2100, 4, 1, 128, 16, 130), (BF16, 2, 1111, 8, 1, 128, 1, 1), (F16, 2, 1600, 16, 2, 72, 60, 257),
    (BF16, 1, 4300, 2, 1, 64, 100, 4), (F16, 1, 400, 130, 1, 32, 5, 2)])
@pytest.mark.parametrize("how", ["plain", "packed", "lengths"])
def test_against_float64(pkg, dtype, batch, tokens, hq, hk, dim, window, sinks, how):
    assert splits(pkg, batch, tokens, hq, hk, dim, window, sinks)
    q, k, v, dout = make(dtype, batch, tokens, hq, hk, dim, seed=tokens, packed=how == "packed")
    for short in ([0, sinks, 300] if how == "lengths" else [None]):
        lengths = None
        if short is not None:   # parts behind a sequence's end have no rows
            lengths = torch.tensor([short, tokens - 1][:batch], device="cuda")
            for b in range(batch):
                for x in (q, k, v, dout):
                    x[b, int(lengths[b]):] = math.nan
            if short:           # the rows that the last lengths have cut off
                for x, y in zip((q, k, v, dout), make(dtype, batch, tokens, hq, hk, dim, seed=tokens)):
                    for b in range(batch):
                        x[b, :int(lengths[b])] = y[b, :int(lengths[b])]
        check(pkg, q, k, v, dout, lengths, window, sinks)


def test_a_long_sequence(pkg):
    """16384 tokens in sixteen parts: what stretches of queries add to the first keys, and the bounds, add up."""
    A = pkg.attention
    n, window, sinks, step = 16384, 700, 3, 2048
    assert splits(pkg, 1, n, 2, 1, 128, window, sinks)
    q, k, v, dout = make(BF16, 1, n, 2, 1, 128)
    out, lse = A.window_attention(q, k, v, window=window, sinks=sinks, return_lse=True)
    got = A.window_attention_backward(dout, q, k, v, out, lse, window=window, sinks=sinks)[1:]
    scale = float(torch.tensor(1 / math.sqrt(128)))
    want, bound = [0, 0], [0, 0]
    for first in range(0, n, step):
        rows = torch.arange(first, first + step, device="cuda")
        keys = torch.cat((torch.arange(min(sinks, max(0, first - window + 1)), device="cuda"), torch.arange(max(0, first - window + 1), first + step, device="cuda")))
        read = ((keys <= rows[:, None]) & ((rows[:, None] - keys < window) | (keys < sinks)))[None]
        grads, bounds = co.gradients(q[:, rows], k[:, keys], v[:, keys], dout[:, rows], read, scale)
        for i in range(2):
            want[i], bound[i] = want[i] + grads[1 + i][:, :sinks], bound[i] + bounds[1 + i][:, :sinks]
    for i in range(2):
        ao.within(got[i][:, :sinks], want[i], bound[i])
