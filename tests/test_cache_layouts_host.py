"""Which kernel attention over an 8-bit cache takes, by the library's own rule:
the sizes that the GPU tests of the large kernels use are theirs."""

from __future__ import annotations

import ctypes

import pytest
import torch
from cache_layouts import (
    MANY,
    MANY_SIZES,
    SPLIT_SIZES,
    TWO_TILES,
    layout,
    layout_of,
)
from test_cache_host import _attention, _cache, _library

CODES = (torch.float8_e4m3fn, torch.int8)
HALVES = (torch.float16, torch.bfloat16)


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('sizes', MANY_SIZES)
def test_waves_with_rows_of_their_own(sizes, dtype, code):
    assert layout_of(dtype, code, *sizes) == (*MANY, 1)


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', (torch.float32, *HALVES))
@pytest.mark.parametrize('sizes', SPLIT_SIZES)
def test_two_tiles_with_split_tokens(sizes, dtype, code):
    share, tiles, splits = layout_of(dtype, code, *sizes)
    assert (share, tiles) == TWO_TILES and splits > 1


def test_small_calls_share_one_tile():
    for dtype in (torch.float32, *HALVES):
        for dim in (32, 64, 96, 128):
            assert layout(dtype, torch.int8, 4, 512, 4, 8, 2, dim, None, 0,
                          0) == (1, 1, 1)
            assert layout(dtype, torch.int8, 1, 1 << 15, 1, 8, 2, dim, None, 0,
                          0)[:2] == (1, 1)


def test_refusals():
    lib = _library()
    out = ctypes.byref(ctypes.c_int())
    cache, args = _cache(), _attention()
    for results in ((None, out, out), (out, None, out), (out, out, None)):
        assert lib.lattice_hip_cache_attention_layout(
            ctypes.byref(cache), ctypes.byref(args), *results) == 1
        assert b'non-null' in lib.lattice_hip_last_error()
    assert lib.lattice_hip_cache_attention_layout(
        ctypes.byref(cache), ctypes.byref(_attention(heads=3)), out, out,
        out) == 1
    assert b'multiple' in lib.lattice_hip_last_error()
