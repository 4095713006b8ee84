"""The caption example's sizes of resized images are the pipeline's: a patch more or less would mask what is image, or read padding."""
import importlib.util
import os

import pytest

pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("caption_step", os.path.join(ROOT, "examples", "caption_step.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_sizes(example, oracle):
    for h in range(200, 460, 3):
        for w in range(200, 460):
            assert example.resized(h, w, 224) == tuple(oracle.smallest_side_dims(h, w, 224)), (h, w)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_patches_of_every_image_are_read(example, pkg, seed):
    """The smaller side of every image is the size that was asked for, whole patches, none of them masked."""
    import torch
    pixels, grid = example.image_batch(pkg, 6, 224, seed)
    assert torch.equal(grid.min(1).values, torch.full((6,), 224 // example.PATCH, device="cuda"))
    _, _, mask = example.patches(pixels, grid)
    assert torch.equal(mask.sum(1), grid.prod(1))
