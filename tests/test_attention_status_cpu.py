"""The self-check word of cross attention: no failure is lost to a reader, whichever stream it asks about."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "mlx-data_b200", "csrc")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not shutil.which("g++") or not os.path.exists(os.path.join(CUDA, "include", "cuda_runtime.h")):
        pytest.skip("needs g++ and CUDA's headers")
    out = str(tmp_path_factory.mktemp("attention_status") / "attention_status")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I" + os.path.join(CUDA, "include"), "-I" + CSRC,
                    os.path.join(HERE, "attention_status.cpp"), "-o", out], check=True)
    return out


@pytest.mark.parametrize("scenario", ["two_askers", "failure_while_asking"])
def test_scenario(program, scenario):
    r = subprocess.run([program, scenario], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, (r.returncode, r.stdout + r.stderr)
