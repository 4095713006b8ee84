"""The example that runs the loader and the attention operators together."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_caption_step(pkg):
    spec = importlib.util.spec_from_file_location("caption_step", os.path.join(ROOT, "examples", "caption_step.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.main()
    assert 0 < int(got["mask"].sum()) < got["mask"].numel()          # ragged images: some patches are padding
    assert got["out"].shape == (4, 48, example.HEADS * example.DIM) and torch.isfinite(got["out"].float()).all()
    assert all(g is not None and torch.isfinite(g.float()).all() and g.float().norm() > 0 for g in got["grads"].values())
    # the last token alone, through the way of single tokens, is the last row of the whole text: two bfloat16 roundings apart
    a, b = got["step"][:, 0].double(), got["out"][:, -1].double()
    size = got["v"].double().abs().amax()
    assert (a - b).abs().max() <= 4 * 2.0 ** -8 * size
