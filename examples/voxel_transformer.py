"""A transformer block over voxel scans: training steps, then the same causal
attention served token by token against a cache.

    python examples/voxel_transformer.py
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent
                       / 'mlx-lattice_amd'))

import mlx_lattice_amd.nn as lnn  # noqa: E402
import mlx_lattice_amd.ops as ops  # noqa: E402


def scan(rows: int, generator: torch.Generator) -> torch.Tensor:
    """Distinct voxels of a cube of 64, in scan order."""
    places = torch.randperm(64 ** 3, generator=generator)[:rows].sort().values
    return torch.stack([places // 4096, places // 64 % 64, places % 64],
                       1).to(torch.int32)


def train(steps: int = 20, channels: int = 64) -> list[float]:
    """Fits a block to a field over two scans; the losses of the steps."""
    generator = torch.Generator().manual_seed(0)
    coords = [scan(n, generator).cuda() for n in (3000, 2001)]
    feats = [torch.randn((len(c), channels), generator=generator).cuda()
             for c in coords]
    x = ops.sparse_collate(coords, feats)
    target = torch.sin(x.coords[:, 1:].float().sum(1, keepdim=True) / 9)
    block = lnn.VoxelTransformerBlock(channels, 4, kv_heads=2, left=96,
                                      right=96, sinks=2, p=0.1, seed=7,
                                      device='cuda')
    for parameter in block.parameters():
        parameter.requires_grad_()
    optimizer = torch.optim.Adam(block.parameters(), lr=1e-3)
    offsets = ops.batch_offsets(x)
    losses = []
    for _ in range(steps):
        optimizer.zero_grad()
        out = block(x, offsets=offsets)
        loss = ((out.feats[:, :1] - target) ** 2).mean()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


@torch.no_grad()
def serve(rows: int = 300, heads: int = 8, kv_heads: int = 2, dim: int = 32
          ) -> float:
    """Feeds two scans row by row to a causal attention with a cache, a row of
    each at a time; the largest difference from the scans' single pass."""
    generator = torch.Generator().manual_seed(1)
    coords = torch.stack([scan(rows, generator) for _ in range(2)]).cuda()
    packed = torch.randn((2, rows, heads + 2 * kv_heads, dim),
                         generator=generator).cuda().to(torch.bfloat16)
    dims = (12, 10, 10)
    frequencies = ops.rotary_frequencies(dims, device='cuda')
    window = {'left': 64, 'right': 0, 'sinks': 4}

    def turn(part, positions):
        return ops.rotary_positions(part[:, :heads + kv_heads], positions,
                                    frequencies, dims=dims)

    offsets = torch.tensor([0, rows, 2 * rows], dtype=torch.int32,
                           device='cuda')
    flat = packed.view(2 * rows, -1, dim)
    turned = turn(flat, coords.view(-1, 3))
    whole = ops.window_attention(
        turned[:, :heads], turned[:, heads:], flat[:, heads + kv_heads:],
        offsets=offsets, **window).view(2, rows, heads, dim)

    keys, values = (torch.zeros((2, rows, kv_heads, dim), device='cuda',
                                dtype=torch.bfloat16) for _ in range(2))
    token = torch.arange(3, dtype=torch.int32, device='cuda')
    lengths = torch.zeros(2, dtype=torch.int32, device='cuda')
    worst = torch.zeros((), device='cuda')
    for at in range(rows):
        turned = turn(packed[:, at], coords[:, at])
        keys[:, at] = turned[:, heads:]
        values[:, at] = packed[:, at, heads + kv_heads:]
        lengths += 1
        out = ops.window_attention(
            turned[:, :heads], keys.view(2 * rows, kv_heads, dim),
            values.view(2 * rows, kv_heads, dim), offsets=token,
            key_offsets=offsets, key_lengths=lengths, **window)
        worst = torch.maximum(worst, (out - whole[:, at]).abs().max())
    return float(worst)


if __name__ == '__main__':
    losses = train()
    print(f'training loss {losses[0]:.3f} -> {losses[-1]:.3f}')
    print(f'token by token, largest difference {serve():.3g}')
