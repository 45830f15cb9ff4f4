"""Modules of a transformer block over the rows of voxel scans (no reference
counterpart): layer norm, counter-based dropout, windowed attention with rotary
positions by voxel coordinates, and the block they make with pointwise convs.

Rows of a scan are adjacent and in scan order, as a sorted cloud or
``sparse_collate`` of sorted clouds lays them; the window is one of rows in
that order."""

from __future__ import annotations

import torch
from torch import nn

from mlx_lattice_amd.core import QuantizedCache, SparseTensor
from mlx_lattice_amd.nn.conv import SubmConv3d
from mlx_lattice_amd.ops import (
    batch_offsets,
    cache_attention,
    dropout,
    layer_norm,
    residual_norm,
    rotary_frequencies,
    rotary_positions,
    window_attention,
    write_cache,
)

__all__ = ['Dropout', 'LayerNorm', 'VoxelTransformerBlock', 'WindowAttention']


class LayerNorm(nn.Module):
    """Layer norm of feature rows delegating to :func:`layer_norm`."""

    def __init__(self, channels: int, *, eps: float = 1e-5, bias: bool = True,
                 device=None, dtype: torch.dtype = torch.float32) -> None:
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(
            torch.ones(channels, device=device, dtype=dtype),
            requires_grad=False)
        self.bias = nn.Parameter(
            torch.zeros(channels, device=device, dtype=dtype),
            requires_grad=False) if bias else None

    def forward(self, x: SparseTensor) -> SparseTensor:
        return layer_norm(x, self.weight, self.bias, eps=self.eps)


def _draw() -> int:
    """A number of torch's CPU generator."""
    return int(torch.randint(2 ** 62, (), device='cpu'))


class Dropout(nn.Module):
    """Dropout delegating to :func:`dropout`, with a residual.

    ``seed`` is the layer's own, by default drawn from torch's CPU generator,
    as initial weights are (ranks that build their layers from the same state
    and train on different rows give seeds of their own); ``calls`` counts the
    layer's training passes and is the generator's offset, so that each pass
    has a mask of its own and a run repeats from the two numbers.  Both are in
    ``state_dict``: a resumed run goes on with the masks.  A seed that was
    given stays when a state is loaded.

    A pass that checkpointing makes again in the backward pass has the mask of
    the first: it is known by a number drawn from torch's CPU generator, whose
    state checkpointing restores.  Where the first cannot be told (the state
    was not kept, several passes began with the same, or it lies more than
    4096 passes back), a pass inside a backward pass is an error.
    """

    def __init__(self, p: float, *, seed: int | None = None) -> None:
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError('p must be between 0 and 1.')
        self.p = p
        self._drawn_seed = seed is None
        # Without dropout nothing is drawn, and a network's weights are those
        # of its seed.
        self.seed = _draw() if seed is None and p > 0.0 else seed
        self.calls = 0
        # The offsets of the last passes by the number drawn; None: of several.
        self._offsets: dict[int, int | None] = {}

    def forward(self, x: SparseTensor, *,
                residual: SparseTensor | None = None) -> SparseTensor:
        if not self.training or self.p == 0.0:
            if residual is None:
                return x
            if not x.same_coords(residual):
                raise ValueError('sparse tensor coordinates must match.')
            return x.replace(feats=x.feats + residual.feats)
        offset = self._offset()
        if self.seed is None:  # p was zero before
            # Leaves the generator as a pass made again will find it.
            state = torch.get_rng_state()
            self.seed = _draw()
            torch.set_rng_state(state)
        return dropout(x, self.p, seed=self.seed, offset=offset,
                       residual=residual)

    def get_extra_state(self) -> torch.Tensor:
        seed = 0 if self.seed is None else self.seed
        # 64 bits of a seed are in use; a tensor holds them as signed.
        seed = (int(seed) + 2 ** 63) % 2 ** 64 - 2 ** 63
        return torch.tensor([self.calls, seed, self.seed is not None],
                            device='cpu')

    def set_extra_state(self, state: torch.Tensor) -> None:
        self.calls, seed, known = state.tolist()
        if self._drawn_seed and known:
            self.seed = seed

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict,
                              missing_keys, unexpected_keys, error_msgs):
        super()._load_from_state_dict(
            state_dict, prefix, local_metadata, strict, missing_keys,
            unexpected_keys, error_msgs)
        # A state from before the layer had one leaves its masks as they are.
        key = prefix + '_extra_state'
        if key in missing_keys:
            missing_keys.remove(key)

    def _offset(self) -> int:
        drawn = _draw()
        if torch._C._current_graph_task_id() != -1:
            offset = self._offsets.get(drawn)
            if offset is None:
                raise RuntimeError(
                    'a dropout pass inside a backward pass must repeat an '
                    "earlier one, known by the state of torch's CPU "
                    'generator: checkpoint with preserve_rng_state, and give '
                    'each pass a state of its own.')
            return offset
        offset = self.calls
        self.calls += 1
        same = self._offsets.get(drawn, offset) == offset
        self._offsets[drawn] = offset if same else None
        if len(self._offsets) > 4096:
            del self._offsets[next(iter(self._offsets))]
        return offset


class WindowAttention(nn.Module):
    """Attention of each row over the rows ``left`` before to ``right`` after
    it in its scan, and the scan's first ``sinks`` rows.

    One pointwise conv makes the queries, keys and values; the heads of the
    first two are turned by the voxel's x, y and z, a third of a head's
    channels each.
    """

    def __init__(self, channels: int, heads: int, *,
                 kv_heads: int | None = None, left: int | None = 128,
                 right: int | None = 128, sinks: int = 0,
                 rotary_base: float = 10000.0, bias: bool = True, device=None,
                 dtype: torch.dtype = torch.float32) -> None:
        super().__init__()
        self.heads = heads
        self.kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or channels % heads or (channels // heads) % 2:
            raise ValueError('channels must be an even number for each head.')
        if self.kv_heads < 1 or heads % self.kv_heads:
            raise ValueError(
                'the number of heads must be a multiple of the number of key '
                'heads.')
        self.dim = channels // heads
        self.left, self.right, self.sinks = left, right, sinks
        third = self.dim // 6 * 2
        self.dims = (self.dim - 2 * third, third, third)
        # Not a buffer: its float64 is kept when the module changes dtype.
        self._frequencies = rotary_frequencies(self.dims, rotary_base,
                                               device=device)
        self.project = SubmConv3d(
            channels, (heads + 2 * self.kv_heads) * self.dim, kernel_size=1,
            bias=bias, device=device, dtype=dtype)
        self.out = SubmConv3d(channels, channels, kernel_size=1, bias=bias,
                              device=device, dtype=dtype)

    def make_cache(self, batches: int, capacity: int, *,
                   dtype: torch.dtype = torch.float8_e4m3fn
                   ) -> QuantizedCache:
        """An empty 8-bit cache for ``batches`` scans of up to ``capacity``
        rows, on the layer's device."""
        return QuantizedCache.empty(batches, capacity, self.kv_heads, self.dim,
                                    dtype=dtype,
                                    device=self.project.weight.device)

    def forward(self, x: SparseTensor, *,
                offsets: torch.Tensor | None = None,
                cache: QuantizedCache | None = None,
                lengths: torch.Tensor | None = None) -> SparseTensor:
        """``offsets``: the scans' row offsets, which the layers of a level
        can share; ``batch_offsets(x)`` by default, which for a tensor without
        ``batch_counts``, as strided convs give it, waits for the device.

        With a ``cache`` the rows of ``x`` are new rows of streamed scans: they
        are appended to it and see what it holds, ``lengths`` ``(B,)`` counting
        the rows of each scan with the new ones (int32, on the device)."""
        if (cache is None) != (lengths is None):
            raise ValueError('cache and lengths go together.')
        if offsets is None:
            offsets = batch_offsets(x)
        packed = self.project(x).feats.view(x.capacity, -1, self.dim)
        turned = packed[:, :self.heads + self.kv_heads]
        turned = rotary_positions(turned, x.coords[:, 1:],
                                  self._on(x.device), dims=self.dims)
        queries, keys = turned[:, :self.heads], turned[:, self.heads:]
        values = packed[:, self.heads + self.kv_heads:]
        window = {'left': self.left, 'right': self.right, 'sinks': self.sinks,
                  'offsets': offsets}
        if cache is None:
            rows = window_attention(queries, keys, values, **window)
        else:
            write_cache(cache, keys, values, offsets=offsets, lengths=lengths)
            rows = cache_attention(queries, cache, lengths=lengths, **window)
        return self.out(x.replace(feats=rows.view(x.capacity, -1)))

    def _on(self, device: torch.device) -> torch.Tensor:
        if self._frequencies.device != device:
            self._frequencies = self._frequencies.to(device)
        return self._frequencies


class VoxelTransformerBlock(nn.Module):
    """Pre-norm block: ``x + dropout(attention(norm(x)))``, then the same with
    a ReLU layer of ``hidden`` channels (4 times the channels by default).

    ``seed`` gives the two dropouts the seeds ``2 * seed`` and ``2 * seed +
    1``; by default each draws its own.  With ``layer_scale`` each part is
    multiplied by a gate a channel, which starts at that value.
    """

    def __init__(self, channels: int, heads: int, *, hidden: int | None = None,
                 p: float = 0.0, seed: int | None = None,
                 layer_scale: float | None = None, device=None,
                 dtype: torch.dtype = torch.float32, **attention) -> None:
        super().__init__()
        hidden = 4 * channels if hidden is None else hidden
        made = {'device': device, 'dtype': dtype}
        self.norm1 = LayerNorm(channels, **made)
        self.attention = WindowAttention(channels, heads, **attention, **made)
        self.drop1 = Dropout(p, seed=None if seed is None else 2 * seed)
        self.norm2 = LayerNorm(channels, **made)
        self.expand = SubmConv3d(channels, hidden, kernel_size=1, **made)
        self.contract = SubmConv3d(hidden, channels, kernel_size=1, **made)
        self.drop2 = Dropout(p, seed=None if seed is None else 2 * seed + 1)
        self.gate1, self.gate2 = (
            None if layer_scale is None else nn.Parameter(
                torch.full((channels,), float(layer_scale), device=device,
                           dtype=dtype), requires_grad=False)
            for _ in range(2))

    def forward(self, x: SparseTensor, *,
                offsets: torch.Tensor | None = None,
                cache: QuantizedCache | None = None,
                lengths: torch.Tensor | None = None) -> SparseTensor:
        """``cache`` and ``lengths``: as :class:`WindowAttention` takes them."""
        mixed = self.attention(self.norm1(x), offsets=offsets, cache=cache,
                               lengths=lengths)
        if self.gate1 is None:
            x = self.drop1(mixed, residual=x)
            inner = self.expand(self.norm2(x), activation='relu')
            return self.drop2(self.contract(inner), residual=x)
        x, normed = residual_norm(
            self.drop1(mixed), x, self.norm2.weight, self.norm2.bias,
            gate=self.gate1, eps=self.norm2.eps)
        inner = self.expand(normed, activation='relu')
        inner = self.drop2(self.contract(inner))
        return x.replace(feats=torch.addcmul(x.feats, inner.feats, self.gate2))
