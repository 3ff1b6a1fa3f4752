"""A transformer stage over voxels: classes of hidden voxels from the others.

Scenes are rooms on a voxel grid (riemannengine_amd.scenes); every voxel has a
class, given by where it lies, and some are hidden. The model:

  RiemannEmbedding   class -> features (the hidden ones have a class of their
                     own) + a linear map of the coordinates
  AttentionBlock x n layer norm, attention inside each scene, layer norm, MLP
  RiemannLayerNorm   and a linear layer to the classes' logits

With --local the blocks see where a voxel lies themselves: queries and keys are
normed by head and turned by the coordinates, attention stays inside a window of
each scene's rows (which are sorted along a line through the scene, with its
first rows in everyone's sight), and the feed-forward part is gated.

    python examples/voxel_transformer.py [--steps 50] [--dtype bf16] [--local]
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import riemannengine as rie  # noqa: E402
from riemannengine_amd import scenes  # noqa: E402

CLASSES = 8


# AttentionBlock's options with --local, for heads of 32: 5 pairs for each axis
LOCAL = {"window": 128, "sinks": 4, "rotary": [5, 5, 5], "head_norm": True, "gated": True}


def batch(rng, n_scenes, voxels, in_order=False):
    """Coordinates [n, 4] (batch first) and classes [n]: parts of rooms of
    different sizes, the class by the octant of a coarse cell. in_order: each
    scene's rows by coarse cells, so that near rows are near voxels."""
    coords = []
    for b in range(n_scenes):
        c = scenes.indoor_scene(rng, voxel=0.2)
        c = c[rng.permutation(len(c))[:int(voxels * rng.uniform(0.5, 1.0))]]
        if in_order:
            c = c[np.lexsort((c // 4).T)]
        coords.append(np.concatenate([np.full((len(c), 1), b), c], 1))
    coords = np.concatenate(coords).astype(np.int32)
    cell = (coords[:, 1:] // 4) % 2
    return torch.from_numpy(coords), torch.from_numpy(
        (cell[:, 0] * 4 + cell[:, 1] * 2 + cell[:, 2]).astype(np.int64))


class Stage:
    """Plain layers: the framework's are C++ modules, held side by side with
    torch's own."""

    def __init__(self, channels, heads, kv_heads, blocks, dtype, device, options):
        nn = rie.nn
        self.embedding = nn.RiemannEmbedding(CLASSES + 1, channels, scale=channels ** 0.5)
        self.blocks = [nn.AttentionBlock(channels, heads, kv_heads, **options)
                       for _ in range(blocks)]
        self.norm = nn.RiemannLayerNorm(channels)
        for m in (self.embedding, *self.blocks, self.norm):
            m.to(device)
        for m in (self.embedding, *self.blocks):
            m.to(dtype)  # the norms' parameters stay fp32
        self.where = torch.nn.Linear(3, channels).to(device)
        self.head = torch.nn.Linear(channels, CLASSES).to(device)

    def parameters(self):
        for m in (self.embedding, *self.blocks, self.norm, self.where, self.head):
            yield from m.parameters()

    def __call__(self, ids, base, coords):
        x = self.embedding(ids, base)
        place = self.where(torch.remainder(coords[:, 1:].float(), 8.0) / 8.0)
        x = rie.SparseTensor(x.F + place.to(x.F.dtype), x.coordinate_map_key,
                             x.coordinate_manager)
        for block in self.blocks:
            x = block(x)
        return self.head(self.norm(x).F.float())


def train(steps=50, n_scenes=3, voxels=1500, channels=128, heads=4, kv_heads=2, blocks=2,
          dtype=torch.bfloat16, seed=0, log=print, local=False):
    """The losses of `steps` training steps."""
    device = torch.device("cuda:0")
    torch.manual_seed(seed)
    rng = np.random.default_rng(seed)
    model = Stage(channels, heads, kv_heads, blocks, dtype, device, LOCAL if local else {})
    optimizer = torch.optim.Adam(model.parameters(), lr=1e-3)
    losses = []
    for step in range(steps):
        coords, ids = (t.to(device) for t in batch(rng, n_scenes, voxels, local))
        hidden = torch.rand(len(ids), device=device) < 0.3
        base = rie.SparseTensor(torch.zeros(len(ids), 1, device=device), coords)
        logits = model(torch.where(hidden, CLASSES, ids), base, coords)
        loss = torch.nn.functional.cross_entropy(logits[hidden], ids[hidden])
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
        if step % 10 == 0 or step == steps - 1:
            log(f"step {step}: {len(ids)} voxels, loss {losses[-1]:.3f}")
    return losses


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=50)
    parser.add_argument("--dtype", choices=["f32", "bf16"], default="bf16")
    parser.add_argument("--local", action="store_true")
    args = parser.parse_args()
    train(args.steps, dtype={"f32": torch.float32, "bf16": torch.bfloat16}[args.dtype],
          local=args.local)
