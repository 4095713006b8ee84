"""The loader builds where torch is not installed: the attention module is left out, everything else is made."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mlx-data_b200")


def _plan(*args):
    """What make would run."""
    if not shutil.which("make"):
        pytest.skip("needs make")
    r = subprocess.run(["make", "-n", "-B", "-C", PKG, *args], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    return r.stdout, r.stderr


def test_without_torch(tmp_path):
    """A Python whose finder knows no torch stands in for a machine without it."""
    python = tmp_path / "python"
    python.write_text("#!/bin/sh\nexec env PYTHONPATH=%s %s \"$@\"\n" % (tmp_path, shutil.which("python3")))
    python.chmod(0o755)
    (tmp_path / "sitecustomize.py").write_text(
        "import importlib.util as u\n"
        "real = u.find_spec\n"
        "u.find_spec = lambda name, *more: None if name == 'torch' else real(name, *more)\n")
    out, err = _plan("PYTHON=%s" % python)
    assert "attention.cpp" not in out and "Traceback" not in err
    assert "bindings.cpp" in out and "rotary.cu" in out and "-o %s/_c" % PKG in out


def test_with_torch():
    pytest.importorskip("torch")
    out, _ = _plan()
    assert "attention.cpp" in out and "bindings.cpp" in out


def test_the_operators_say_what_is_missing(pkg, monkeypatch):
    """A package built without the module names it when an operator is used."""
    pytest.importorskip("torch")
    import importlib
    real = importlib.import_module

    def missing(name, package=None):
        if name == "._attention":
            raise ModuleNotFoundError("No module named 'mlx_data_b200._attention'", name="mlx_data_b200._attention")
        return real(name, package)

    monkeypatch.setattr(importlib, "import_module", missing)
    monkeypatch.setattr(pkg.attention, "_ops", pkg.attention._Operators())
    with pytest.raises(ImportError, match="built without torch"):
        pkg.attention.rotary(None, None, None, None, ())
