"""Attention over an 8-bit cache in the kernels that only large calls take,
against float64: waves with rows of their own, which share a block of tokens in
LDS, and several tiles whose tokens are split over blocks."""

from __future__ import annotations

import math

import pytest
import torch
from cache_layouts import (
    MANY,
    MANY_SIZES,
    SPLIT_SIZES,
    TWO_TILES,
    capacity,
    layout_of,
)
from cache_reference import random_cache
from test_gpu_cache_attention import (
    _check,
    _ints,
    _offsets,
    _ops,
    _queries,
    _reference,
)
from transformer_reference import assert_within

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)
HALVES = DTYPES[1:]
CODES = (torch.float8_e4m3fn, torch.int8)
SPOILT = 0x7f  # NaN in e4m3, the largest code in int8


def _run(gen, sizes, dtype, code, rows=None, first=0, scale=None, spoil=None,
         **how):
    """The call over random rows and codes, some spoilt, against float64."""
    counts, lengths, heads, kv_heads, dim, left, right, sinks = sizes
    cache = random_cache(gen, code, len(counts), capacity(lengths), kv_heads,
                         dim, **how)
    q = _queries(gen, dtype, sum(counts) if rows is None else rows, heads, dim)
    if spoil is not None:
        spoil(cache)
    return q, cache, _check(q, cache, counts, lengths, left, right, sinks,
                            scale, first=first, device='cuda')


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('sizes', MANY_SIZES)
def test_many_queries(sizes, dtype, code):
    assert layout_of(dtype, code, *sizes) == (*MANY, 1)
    _run(torch.Generator(device='cuda').manual_seed(1), sizes, dtype, code)


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('sizes', SPLIT_SIZES)
def test_several_tiles_with_split_tokens(sizes, dtype, code):
    assert layout_of(dtype, code, *sizes)[:2] == TWO_TILES
    _run(torch.Generator(device='cuda').manual_seed(2), sizes, dtype, code)


@pytest.mark.parametrize('dtype', HALVES)
def test_rows_in_no_sequence_are_zero(dtype):
    sizes = ((1100, 1000), (1300, 1000), 32, 8, 128, None, 0, 0)
    rows = 300 + 2100 + 77
    assert layout_of(dtype, CODES[0], *sizes, rows=rows) == (*MANY, 1)
    _, _, got = _run(torch.Generator(device='cuda').manual_seed(3), sizes,
                     dtype, CODES[0], rows, first=300)
    assert not got[:300].any() and not got[2400:].any()


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('sizes', MANY_SIZES[:3])
def test_blocks_of_unequal_exponents(sizes, dtype, code):
    """Values of blocks from 2^-126 to 2^8 of one another."""

    def spoil(cache):
        e = cache.value_exponents
        e.copy_(torch.randint(-60, 0, e.shape, generator=gen, device='cuda'))
        e[:, :, ::5] = 0
        e[:, :, 3::7] = -126

    gen = torch.Generator(device='cuda').manual_seed(4)
    assert layout_of(dtype, code, *sizes)[:2] == MANY
    _, _, got = _run(gen, sizes, dtype, code, spoil=spoil)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype, sizes, kind', [
    *((dtype, ((1100, 1000), (1300, 1000), 32, 8, 128, 60, 0, 4), MANY)
      for dtype in HALVES),
    *((dtype, ((600, 500), (8100, 6000), 8, 2, 96, 5000, 0, 4), TWO_TILES)
      for dtype in DTYPES)])
def test_what_is_not_seen_never_arrives(dtype, sizes, kind, code):
    """NaN and the largest codes and exponents behind the end and ahead of
    every window; then in tokens that some queries see."""
    counts, lengths, left = sizes[0], sizes[1], sizes[5]
    assert layout_of(dtype, code, *sizes)[:2] == kind

    def spoil(cache):
        place = torch.arange(cache.capacity, device='cuda').view(-1, 32)
        for s, length in enumerate(lengths):
            cache.keys.view(torch.uint8)[s, :, length:] = SPOILT
            values = cache.values.view(torch.uint8)[s].movedim(3, 2)
            values[:, place >= length] = SPOILT
            cache.key_exponents[s, :, (length + 31) // 32:] = 127
            cache.value_exponents[s, :, (length + 31) // 32:] = 127
            early = max(4, length - counts[s] - left)
            cache.keys.view(torch.uint8)[s, :, 4:early] = SPOILT
            values[:, (place >= 4) & (place < early)] = SPOILT

    gen = torch.Generator(device='cuda').manual_seed(5)
    q, cache, got = _run(gen, sizes, dtype, code, spoil=spoil)
    assert torch.isfinite(got).all()
    if code != torch.float8_e4m3fn:
        return
    at = lengths[0] - counts[0] // 2
    cache.values.view(torch.uint8)[0, 1, at // 32, 9, at % 32] = SPOILT
    cache.keys.view(torch.uint8)[1, 0, lengths[1] - 30, 5] = SPOILT
    got = _check(q, cache, counts, lengths, left, 0, 4, device='cuda')
    assert torch.isnan(got).any() and not torch.isnan(got).all()


@pytest.mark.parametrize('value', (math.inf, -math.inf, math.nan))
@pytest.mark.parametrize('dtype', HALVES)
def test_non_finite_queries_stay_in_their_rows(dtype, value):
    sizes = ((1100, 1000), (1300, 1000), 32, 8, 128, None, 0, 0)
    assert layout_of(dtype, CODES[1], *sizes)[:2] == MANY
    gen = torch.Generator(device='cuda').manual_seed(6)
    q, cache, clean = _run(gen, sizes, dtype, CODES[1])
    q = q.clone()
    rows = ((0, 0), (611, 9), (1099, 31), (2099, 17))
    for row, head in rows:
        q[row, head, 5] = value
    got = _ops().cache_attention(q, cache, offsets=_offsets(sizes[0]),
                                 lengths=_ints(*sizes[1]), right=0)
    for row, head in rows:
        assert torch.isnan(got[row, head]).all()
        got[row, head] = clean[row, head]
    assert torch.equal(got, clean)


@pytest.mark.parametrize('dtype', HALVES)
def test_scales_and_lengths_past_the_capacity(dtype):
    sizes = ((1100, 1000), (1300, 1000), 32, 8, 128, 300, 0, 4)
    counts, lengths = sizes[:2]
    gen = torch.Generator(device='cuda').manual_seed(7)
    q, cache, first = _run(gen, sizes, dtype, CODES[0], scale=0.0)
    args = {'offsets': _offsets(counts), 'left': 300, 'right': 0, 'sinks': 4}

    def call(q, lengths, scale):
        return _ops().cache_attention(q, cache, lengths=_ints(*lengths),
                                      scale=scale, **args)

    assert torch.equal(call(q, lengths, 0.0), first)
    assert torch.equal(call(q, lengths, -0.2), call(-q, lengths, 0.2))
    # Far past the capacity every query sees the first tokens alone.
    far = call(q, (10 ** 9, lengths[1]), 0.1)
    assert_within(far[:1100], *_reference(q[:1100], cache, (1100,), (4,), None,
                                          None, 0, 0.1, device='cuda'))
    want, bound = _reference(q, cache, counts, lengths, 300, 0, 4, 0.1,
                             device='cuda')
    assert_within(far[1100:], want[1100:], bound[1100:])


@pytest.mark.parametrize('dtype', HALVES)
def test_offsets_that_decrease_stay_inside(dtype):
    """Results are unspecified; nothing outside the tensors is written."""
    gen = torch.Generator(device='cuda').manual_seed(8)
    rows = 2100
    sizes = ((rows, 0, 0), (64, 30, 50), 32, 8, 128, None, 0, 0)
    assert layout_of(dtype, CODES[1], *sizes)[:2] == MANY
    cache = random_cache(gen, CODES[1], 3, 64, 8, 128)
    q = _queries(gen, dtype, rows, 32, 128)
    for offsets in ((rows, 5, rows // 2, 0), (7, rows, 3, rows),
                    (rows, rows - 1, 1, 0)):
        _ops().cache_attention(q, cache, offsets=_ints(*offsets),
                               lengths=_ints(64, 30, 50))
    torch.cuda.synchronize()


@pytest.mark.parametrize('dtype, sizes', [
    (torch.float16, MANY_SIZES[1]), (torch.bfloat16, MANY_SIZES[0]),
    (torch.float32, SPLIT_SIZES[1]), (torch.bfloat16, SPLIT_SIZES[0])])
def test_same_result_each_time_and_replayed(dtype, sizes):
    counts, lengths, left, right, sinks = *sizes[:2], *sizes[5:]
    gen = torch.Generator(device='cuda').manual_seed(9)
    q, cache, first = _run(gen, sizes, dtype, CODES[0])
    q = q.clone()
    args = {'offsets': _offsets(counts), 'lengths': _ints(*lengths),
            'left': left, 'right': right, 'sinks': sinks}
    for _ in range(3):
        assert torch.equal(first, _ops().cache_attention(q, cache, **args))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _ops().cache_attention(q, cache, **args)
    for _ in range(3):
        q.copy_(torch.randn(q.shape, generator=gen, device='cuda'))
        want = _ops().cache_attention(q, cache, **args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want)
