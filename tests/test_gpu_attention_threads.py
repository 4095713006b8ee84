"""Calls from threads that have not used CUDA before, as autograd's own threads have not: memory comes from torch's cache, so that the
call's own first step is the thread's first."""
import threading

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def _in_a_thread(call):
    got = []

    def run():
        try:
            got.append(call())
        except Exception as e:   # noqa: BLE001 - handed to the test
            got.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


@pytest.mark.parametrize("tokens", [1, 300])
def test_cross_attention(pkg, tokens):
    A = pkg.attention
    q, k, v = (torch.randn(2, n, 4, 64, device="cuda").to(torch.bfloat16) for n in (tokens, 700, 700))
    want = A.cross_attention(q, k, v, return_lse=True)
    grads = A.cross_attention_backward(q, q, k, v, *want)
    for _ in range(2):
        torch.cuda.synchronize()
        out = _in_a_thread(lambda: A.cross_attention(q, k, v))
        assert torch.equal(out, want[0])
        del out
        got = _in_a_thread(lambda: A.cross_attention_backward(q, q, k, v, *want))
        assert all(torch.equal(a, b) for a, b in zip(got, grads))
        del got


def test_rotary(pkg):
    A = pkg.attention
    q = torch.randn(2, 9, 4, 64, device="cuda")
    positions, f, w = torch.zeros(1, 2, 9, device="cuda"), torch.ones(32, device="cuda"), torch.ones(64, device="cuda")
    calls = [lambda: A.rotary(q, q, positions, f, (32,)), lambda: A.qk_norm_rotary(q, q, positions, f, (32,), w, w),
             lambda: A.qk_norm_rotary_backward(q, q, q, q, positions, f, (32,), w, w)]
    for call in calls:
        want = call()
        got = call()
        del got
        assert all(torch.equal(a, b) for a, b in zip(_in_a_thread(call), want))


AUTOGRAD = """
import torch
from __graft_entry__ import load_package
A = load_package().attention
q, k = (torch.randn(2, n, 4, 64, device="cuda").to(torch.bfloat16).requires_grad_() for n in (300, 700))
with torch.no_grad():
    out, lse = A.cross_attention(q, k, k, return_lse=True)
    for _ in range(2):
        spare = [torch.empty_like(x) for x in (q, k, k, k) for _ in range(4)] + [torch.empty(1 << 16, device="cuda") for _ in range(4)]
        del spare
        grads = A.cross_attention_backward(out, q, k, k, out, lse)
torch.autograd.backward(A.cross_attention(q, k, k), out)
assert torch.equal(q.grad, grads[0])
"""


def test_autograd_in_a_fresh_process():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", AUTOGRAD], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
