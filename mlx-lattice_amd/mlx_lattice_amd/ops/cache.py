"""An 8-bit cache of attention keys and values: writing rows, reading them
back, and attention over it (no reference counterpart)."""

from __future__ import annotations

import torch

from mlx_lattice_amd._native import ext
from mlx_lattice_amd.core import QuantizedCache

__all__ = ['cache_attention', 'read_cache', 'write_cache']

_ALL = 2 ** 31 - 1


def write_cache(cache: QuantizedCache, k: torch.Tensor, v: torch.Tensor, *,
                offsets: torch.Tensor, lengths: torch.Tensor) -> None:
    """Append rows to ``cache``, in place.

    ``k`` and ``v`` have shape ``(rows, kv_heads, dim)`` (float32, float16 or
    bfloat16; each may be a slice of packed rows).  Sequence ``s`` gets the
    rows ``offsets[s] : offsets[s + 1]`` as the last of its ``lengths[s]``
    tokens: ``lengths`` counts the new ones, as :func:`cache_attention` takes
    it.  Both are int32 on the device and are not read back; offsets must not
    decrease, and are clamped to the rows there are.  Tokens past the cache's
    capacity are not written; tokens past the length keep their bytes.

    A block that gets new tokens takes the least exponent, at least -126, that
    leaves their largest finite magnitude at most the largest code (448 or
    127), or its earlier tokens' exponent if that is larger; earlier codes are
    divided by the power of two between.  Quotients are rounded half to even.
    Infinities and NaN become NaN in ``float8_e4m3fn``; ``int8`` has neither:
    they become the largest code and 0.  Without gradient.
    """
    ext.cache_write(cache.parts, cache.dim, k, v, offsets, lengths)


def read_cache(cache: QuantizedCache, *, lengths: torch.Tensor,
               dtype: torch.dtype = torch.float32
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that ``cache`` stands for, ``(B, capacity, kv_heads,
    dim)`` each, rounded once to ``dtype`` (float32, float16 or bfloat16);
    zeros at and past ``lengths`` ``(B,)``.

    Flattened to rows they are what :func:`window_attention` takes, with
    ``key_offsets = arange(B + 1) * capacity`` and ``key_lengths = lengths``.
    """
    return ext.cache_read(cache.parts, cache.dim, lengths, dtype)


def cache_attention(q: torch.Tensor, cache: QuantizedCache, *,
                    offsets: torch.Tensor, lengths: torch.Tensor,
                    left: int | None = None, right: int | None = None,
                    sinks: int = 0, scale: float | None = None
                    ) -> torch.Tensor:
    """:func:`window_attention` over an 8-bit cache, ``(queries, heads, dim)``.

    ``q`` has shape ``(queries, heads, dim)``, ``heads`` a multiple of the
    cache's key heads (float32, float16 or bfloat16; it may be a slice of
    packed rows); ``scale`` is ``dim ** -0.5`` by default.  Sequence ``s``
    holds the query rows ``offsets[s] : offsets[s + 1]`` and the first
    ``lengths[s]`` tokens of the cache, with the queries at their end: query
    ``i`` of ``n`` has position ``p = i + lengths[s] - n``.  It sees token
    ``j`` where ``j <= p + right`` and either ``j >= p - left`` or ``j <
    sinks``; ``None`` is no bound, ``right=0`` is causal.  Both tensors are
    int32 on the device and are not read back; offsets must not decrease, and
    are clamped to the rows there are.

    A query that sees nothing gives zeros, as do rows in no sequence; what a
    query does not see never reaches it.  Products of queries and codes are
    summed before the blocks' powers of two go in, and overflow float32 from
    queries of ``2 ** 112`` on.  Without gradient.
    """
    left, right = (_ALL if b is None else int(b) for b in (left, right))
    if scale is None:
        scale = cache.dim ** -0.5
    return ext.cache_attention(q, cache.parts, cache.dim, offsets, lengths,
                               left, right, int(sinks), float(scale))
