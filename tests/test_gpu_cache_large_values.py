"""An 8-bit cache at the end of float32's range: attention over values whose
sums leave it and whose averages do not, and rows behind the largest
exponents."""

from __future__ import annotations

import math

import pytest
import torch
from cache_reference import (
    appended,
    codes_of,
    decoded,
    random_cache,
    same_values,
)
from transformer_reference import assert_within, attention_f64

pytestmark = pytest.mark.gpu
CODES = (torch.float8_e4m3fn, torch.int8)
# What the largest codes below stand for: 240 * 2 ** 120 and 127 * 2 ** 121.
MOST = {torch.float8_e4m3fn: (240, 120), torch.int8: (127, 121)}


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _large(gen, code, batches, capacity, heads, dim):
    """Values of one sign a channel, of whose largest two have no sum."""
    cache = random_cache(gen, code, batches, capacity, heads, dim)
    most, exponent = MOST[code]
    signs = torch.where(torch.arange(cache.values.shape[3],
                                     device='cuda') % 3 == 0, -1.0, 1.0)
    cache.values.copy_((cache.values.float().abs() * 2).clamp(
        most // 2, most) * signs[:, None])
    cache.values.movedim(3, -1)[..., dim:] = 0
    cache.value_exponents.fill_(exponent)
    return cache


def _check(q, cache, counts, lengths, left=None, sinks=0):
    import mlx_lattice_amd.ops as ops

    offsets = [0]
    for n in counts:
        offsets.append(offsets[-1] + n)
    got = ops.cache_attention(q, cache, offsets=_ints(*offsets),
                              lengths=_ints(*lengths), left=left, right=0,
                              sinks=sinks)
    flat = [t.reshape(-1, *t.shape[2:]) for t in decoded(cache)]
    spans = [(offsets[s], n, s * cache.capacity, lengths[s])
             for s, n in enumerate(counts)]
    want, bound = attention_f64(q, *flat, spans, left, 0, sinks,
                                q.shape[-1] ** -0.5, device='cuda')[0]
    assert torch.isfinite(want.to(q.dtype)).all()
    assert_within(got, want, bound)


# One token, of which waves or whole blocks of them share the tokens, queries
# in one tile and in several, and rows enough for waves of their own.
@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', (torch.float32, torch.bfloat16))
@pytest.mark.parametrize('counts, lengths, heads, kv_heads, dim, left', [
    ((1,), (2,), 1, 1, 32, None), ((1, 1), (50, 700), 4, 2, 64, None),
    ((1,), (9000,), 4, 1, 128, None), ((3, 40), (30, 3000), 2, 1, 96, 2000),
    ((600,), (900,), 64, 4, 64, None), ((2100, 2300), (2100, 2500), 16, 8, 128,
                                        300)])
def test_averages_of_large_values(counts, lengths, heads, kv_heads, dim, left,
                                  dtype, code):
    gen = torch.Generator(device='cuda').manual_seed(1)
    capacity = (max(lengths) + 31) // 32 * 32
    cache = _large(gen, code, len(counts), capacity, kv_heads, dim)
    q = torch.randn((sum(counts), heads, dim), generator=gen, device='cuda')
    for scale in (0.0, 0.2):  # equal shares, and unequal ones
        _check((q * scale).to(dtype), cache, counts, lengths, left)


@pytest.mark.parametrize('dtype', (torch.float32, torch.bfloat16))
@pytest.mark.parametrize('counts, lengths', (
    ((1,), (300,)), ((1,), (9000,)), ((40,), (300,)), ((3000,), (3100,))))
def test_beside_tokens_that_are_not_seen(counts, lengths, dtype):
    """NaN ahead of the windows, in blocks that they reach into: rows are made
    again from what they see."""
    gen = torch.Generator(device='cuda').manual_seed(2)
    capacity = (max(lengths) + 31) // 32 * 32
    cache = _large(gen, torch.float8_e4m3fn, 1, capacity, 2, 128)
    left = lengths[0] - 40 if counts[0] == 1 else 100
    spoilt = torch.arange(capacity, device='cuda').view(-1, 32) < (
        lengths[0] - counts[0] - left)
    spoilt[:, :2] = False  # the first tokens stay
    if spoilt[1:].any():
        spoilt[1:, :2] = spoilt[1:, 2:4]
    values = cache.values.view(torch.uint8).movedim(4, 3)
    values[:, :, spoilt] = 0x7f
    q = torch.randn((counts[0], 32, 128), generator=gen, device='cuda')
    _check((q * 0.2).to(dtype), cache, counts, lengths, left, sinks=2)


@pytest.mark.parametrize('dtype', (torch.float32, torch.bfloat16))
def test_many_equal_shares(dtype):
    """12,000 values of 3.4e34 each."""
    from mlx_lattice_amd import QuantizedCache

    cache = QuantizedCache.empty(1, 12000, 1, 32, device='cuda')
    cache.values.copy_(torch.full(cache.values.shape, 416.0))
    cache.value_exponents.fill_(106)  # 416 * 2 ** 106 is 3.4e34
    _check(torch.zeros((1, 1, 32), dtype=dtype, device='cuda'), cache, (1,),
           (12000,))


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', (torch.float32, torch.bfloat16))
@pytest.mark.parametrize('dim', (32, 33))
@pytest.mark.parametrize('exponent', (125, 126, 127))
def test_rows_behind_the_largest_exponents(exponent, dim, dtype, code):
    """Exponents that no row asks for but a cache may hold: the new rows'
    codes are what is left of them."""
    import mlx_lattice_amd.ops as ops

    gen = torch.Generator(device='cuda').manual_seed(3)
    cache = random_cache(gen, code, 2, 64, 2, dim)
    cache.key_exponents.fill_(exponent)
    cache.value_exponents.fill_(exponent)
    size = torch.finfo(torch.bfloat16).max
    # Some on the border between two codes.
    rows = torch.rand((8, 4, dim), generator=gen, device='cuda') * 2 - 1
    rows *= size
    rows[1] = 2.0 ** exponent
    rows[2] = -1.5 * 2.0 ** min(exponent, 126)
    rows[3] = 2.0 ** 100
    rows[5, :, ::3], rows[5, :, 1::3] = math.inf, -math.inf
    rows[6, :, ::7] = math.nan
    rows = rows.to(dtype)
    k, v = rows[:, :2], rows[:, 2:]
    want = [codes_of(cache)[0], codes_of(cache)[1],
            cache.key_exponents.cpu().clone(),
            cache.value_exponents.cpu().clone()]
    for s, (at, before) in enumerate(((slice(0, 4), 7), (slice(4, 8), 40))):
        for which, part in enumerate((k, v)):
            for head in range(2):
                want[which][s, head], want[2 + which][s, head] = appended(
                    want[which][s, head], want[2 + which][s, head],
                    part[at, head].cpu().double(), code, before, before + 4,
                    64)
    assert (want[2] == exponent).all()
    ops.write_cache(cache, k, v, offsets=_ints(0, 4, 8),
                    lengths=_ints(11, 44))
    for got, ref in zip((*codes_of(cache), cache.key_exponents.cpu(),
                         cache.value_exponents.cpu()), want):
        assert same_values(got, ref)
