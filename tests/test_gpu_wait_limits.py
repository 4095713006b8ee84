"""What a kernel of cross attention does when a wait runs out: a flag that nothing sets, in a kernel of its own (wait_limits.cu)."""
import json
import os
import shutil
import subprocess

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def seen(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("needs nvcc")
    out = str(tmp_path_factory.mktemp("wait_limits") / "wait_limits")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", os.path.join(HERE, "wait_limits.cu"),
                    "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    return json.loads(r.stdout)


def test_every_warp_gives_up(seen):
    assert seen["gave_up"] == [1, 1, 1, 1] and seen["failed"] == 1


def test_the_limit_is_about_two_seconds(seen):
    assert 1 < seen["seconds"] < 10, seen["seconds"]


def test_products_have_ended(seen):
    assert seen["ended"] == 1


def test_its_rows_are_not_numbers(seen):
    assert seen["spoiled"] == 128 * 24 and seen["wrong"] == 0
