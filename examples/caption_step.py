"""Captions of images of different sizes: from the loader's padded batch to the gradients of a decoder's attention.

The pipeline resizes ragged images, pads them to the largest of a batch and leaves the batch in GPU memory.  Its patches become
the states that text reads: the image's own queries and keys are normalised and turned by row and column
(``attention.qk_norm_rotary``), the text's by their place in the text (``attention.rotary``), and the text reads the patches that
are image and not padding (``attention.cross_attention`` with a mask of keys).  Runs a forward and a backward pass, and one step
of generation.  ``python examples/caption_step.py`` on a GPU.
"""
import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from __graft_entry__ import load_package  # noqa: E402

PATCH, HEADS, KV_HEADS, DIM = 16, 8, 2, 64


def resized(h, w, size):
    """Height and width that ``image_resize_smallest_side`` gives an image: both scaled in float64, halves rounded up."""
    scale = size / min(h, w)
    return math.floor(scale * h + 0.5), math.floor(scale * w + 0.5)


def image_batch(dx, n, size=224, seed=0):
    """``n`` images of different sizes as one padded float32 batch in GPU memory, and the rows and columns of patches of each."""
    rng = np.random.default_rng(seed)
    samples = []
    for _ in range(n):
        h, w = (int(x) for x in rng.integers(size, 2 * size, 2))
        samples.append({"image": rng.integers(0, 256, (h, w, 3), dtype=np.uint8)})
    dx.core.set_device_output(True)
    try:
        stream = dx.buffer_from_vector(samples).to_stream().image_resize_smallest_side("image", size).batch(n).key_cast("image")
        pixels = torch.as_tensor(next(iter(stream))["image"], device="cuda")
    finally:
        dx.core.set_device_output(False)
    sizes = [resized(*s["image"].shape[:2], size) for s in samples]
    assert pixels.shape[1:3] == tuple(max(x) for x in zip(*sizes))   # the largest of the batch, to which the others are padded
    return pixels, torch.tensor([(h // PATCH, w // PATCH) for h, w in sizes], device="cuda")


def patches(pixels, grid):
    """[n, rows * columns, 3 * PATCH^2] of the padded batch, positions (row, column), and which patches are image."""
    n, h, w, c = pixels.shape
    rows, cols = h // PATCH, w // PATCH
    x = pixels[:, :rows * PATCH, :cols * PATCH].reshape(n, rows, PATCH, cols, PATCH, c).permute(0, 1, 3, 2, 4, 5)
    at = torch.arange(rows * cols, device="cuda")
    positions = torch.stack((at // cols, at % cols))[:, None].expand(2, n, -1)
    mask = (at // cols < grid[:, :1]) & (at % cols < grid[:, 1:])
    return x.reshape(n, rows * cols, -1).to(torch.bfloat16), positions, mask


class Decoder(torch.nn.Module):
    """One layer: text reads an image's patches."""

    def __init__(self, dx):
        super().__init__()
        kw = dict(bias=False, device="cuda", dtype=torch.bfloat16)
        self.A = dx.attention
        self.queries = torch.nn.Linear(HEADS * DIM, HEADS * DIM, **kw)
        self.states = torch.nn.Linear(3 * PATCH * PATCH, 2 * KV_HEADS * DIM, **kw)
        self.k_weight = torch.nn.Parameter(torch.ones(DIM, device="cuda"))
        half = torch.arange(DIM // 2, device="cuda", dtype=torch.float32)
        self.register_buffer("frequencies", 10000.0 ** (-half / (DIM // 2)))

    def image(self, x, positions):
        k, v = self.states(x).unflatten(-1, (2, KV_HEADS, DIM)).unbind(2)
        # rows and columns take half of the pairs each; queries of the image itself are not needed here
        k, _ = self.A.qk_norm_rotary(k, None, positions, self.frequencies, (DIM // 4, DIM // 4), self.k_weight)
        return k, v

    def forward(self, text, start, k, v, mask):
        n, t, _ = text.shape
        q = self.queries(text).unflatten(-1, (HEADS, DIM))
        places = torch.arange(start, start + t, device="cuda")[None, None].expand(1, n, t)
        q, _ = self.A.rotary(q, None, places, self.frequencies, (DIM // 2,))
        return self.A.cross_attention(q, k, v, key_mask=mask).flatten(2)


def main(n=4, tokens=48):
    dx = load_package()
    torch.manual_seed(0)
    x, positions, mask = patches(*image_batch(dx, n))
    layer = Decoder(dx)
    text = torch.randn(n, tokens, HEADS * DIM, device="cuda").to(torch.bfloat16)
    k, v = layer.image(x, positions)
    out = layer(text, 0, k, v, mask)
    loss = out.float().square().mean()
    loss.backward()
    with torch.no_grad():   # one step of generation reads the same states
        step = layer(text[:, -1:], tokens - 1, k, v, mask)
    return dict(loss=loss.item(), out=out.detach(), step=step, mask=mask, k=k.detach(), v=v.detach(),
                grads={name: p.grad for name, p in layer.named_parameters()})


if __name__ == "__main__":
    got = main()
    print("loss %.5f, %d of %d patches are image" % (got["loss"], int(got["mask"].sum()), got["mask"].numel()))
    for name, g in got["grads"].items():
        print("%-16s gradient norm %.3e" % (name, g.float().norm().item()))
