"""Sizes of attention over an 8-bit cache that reach kernels which only large
calls take, and the kernel that the library chooses for sizes (test
infrastructure)."""

from __future__ import annotations

import ctypes

import torch
from test_cache_host import Attention, Cache, _library

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
# Waves with rows of their own, in two tiles; and waves that share rows in two
# tiles, with the tokens split over blocks of threads.
MANY = (0, 2)
TWO_TILES = (1, 2)

# (queries and lengths of the sequences, heads, key heads, channels, left, right,
# first tokens)
MANY_SIZES = [
    ((1100, 1000), (1300, 1000), 32, 8, 128, None, 0, 0),
    # Windows that begin behind the first tokens, with and without a gap, and
    # sequences of no rows and of one.
    ((900, 0, 1, 1300), (2000, 50, 700, 1300), 64, 8, 104, 200, 0, 5),
    ((2100,), (2100,), 32, 8, 97, 40, 7, 70),
    # Queries before the first token; one block of tokens, and two.
    ((2500, 33), (40, 64), 32, 8, 128, None, 0, 0),
    ((30,) * 90, tuple(30 + s % 35 for s in range(90)), 64, 8, 112, None, None,
     0),
    # One head to a key head, and all heads to one.
    ((2100, 2300), (2200, 2300), 16, 16, 120, 600, 0, 33),
    ((1500, 800), (1600, 900), 32, 1, 128, 0, 300, 1)]
SPLIT_SIZES = [
    ((512,), (8192,), 8, 2, 128, None, 0, 0),
    ((500, 3, 130), (8000, 8190, 5000), 8, 2, 100, None, 0, 0),
    ((1100,), (8192,), 8, 2, 64, 5000, 0, 3),
    ((700, 800), (7000, 8000), 8, 2, 32, 6000, 9, 40)]


def capacity(lengths):
    return (max(lengths) + 31) // 32 * 32


def layout(dtype, code, batches, capacity, queries, heads, kv_heads, dim, left,
           right, sinks):
    """(share, tiles, splits) of a call."""
    lib = _library()
    piece = 4 if dtype == torch.float32 else 8
    dim = (dim + piece - 1) // piece * piece
    cache = Cache(code=int(code == torch.int8), sequences=batches,
                  kv_heads=kv_heads, blocks=capacity // 32, dim=dim, keys=4096,
                  values=4096, key_exponents=4096, value_exponents=4096)
    most = 2 ** 31 - 1
    args = Attention(dtype=_TYPES[dtype], queries=queries, heads=heads,
                     left=most if left is None else left,
                     right=most if right is None else right, sinks=sinks,
                     scale=1.0, q=4096, q_row_stride=heads * dim,
                     q_head_stride=dim, offsets=4096, lengths=4096)
    out = [ctypes.c_int() for _ in range(3)]
    assert lib.lattice_hip_cache_attention_layout(
        ctypes.byref(cache), ctypes.byref(args),
        *map(ctypes.byref, out)) == 0, lib.lattice_hip_last_error()
    return tuple(v.value for v in out)


def layout_of(dtype, code, counts, lengths, heads, kv_heads, dim, left, right,
              sinks, rows=None):
    return layout(dtype, code, len(counts), capacity(lengths),
                  sum(counts) if rows is None else rows, heads, kv_heads, dim,
                  left, right, sinks)
