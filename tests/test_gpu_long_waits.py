"""The limit of a wait is one of standstill: a warp whose turn comes seconds later, because its CTA has that much to do, does not give up.  In
a kernel of its own (wait_pace.cu), and in a call of window attention whose one tile of a short sequence is each CTA's last."""
import json
import math
import os
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402
import causal_oracle as co      # noqa: E402

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


def test_waits_behind_progress(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("needs nvcc")
    out = str(tmp_path / "wait_pace")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", os.path.join(HERE, "wait_pace.cu"), "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    seen = json.loads(r.stdout)
    assert seen["came"] == [1, 0, 0, 0]                  # with progress until it comes; as if it were next; after progress has ended
    behind, plain, stopped, _ = seen["seconds"]
    assert 4 <= behind < 5 and 1 < plain < 4 and 1 + 1 < stopped < 10 and stopped > plain + 0.5


def test_a_short_sequence_beside_a_long_one(pkg):
    """Two samples in one padded batch, the long one with seconds of work: jobs run from the last tokens to the first, so the short
    one's end is what every CTA comes to last."""
    n, short, heads, dim = 425984, 100, 128, 8
    gen = torch.Generator(device="cuda")
    gen.manual_seed(0)
    q, k, v = (torch.randn((2, n, h, dim), generator=gen, device="cuda").to(torch.bfloat16) for h in (heads, 1, 1))
    k[1, short:] = math.nan
    v[1, short:] = math.nan
    lengths = torch.tensor([n, short], device="cuda")
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    out, lse = pkg.attention.window_attention(q, k, v, lengths=lengths, return_lse=True)
    end.record()
    assert pkg._capi.attention_status(0, torch.cuda.current_stream().cuda_stream) == 0
    assert begin.elapsed_time(end) > 2200, begin.elapsed_time(end)   # longer than the limit of a wait that stands still
    assert not out[1, short:].any() and (lse[1, :, short:] == -math.inf).all() and torch.isfinite(out).all()
    scale = float(torch.tensor(1 / math.sqrt(dim)))
    for b, rows in ((1, range(short)), (0, [0, 129, 5000, 100000, n - 1])):
        rows = torch.tensor(rows, device="cuda")
        keys = int(rows[-1]) + 1
        a = (q[b:b + 1, rows], k[b:b + 1, :keys], v[b:b + 1, :keys])
        read = (torch.arange(keys, device="cuda") <= rows[:, None])[None]
        want, want_lse, p = co.attention(*a, read, scale)
        ao.within(out[b:b + 1, rows], want, co.bound(*a, want, p, read, scale))
        ao.within(lse[b:b + 1, :, rows], want_lse, co.lse_bound(a[0], a[1], read, want_lse, scale))
