"""Attention over an 8-bit cache against float64 over what the cache stands
for."""

from __future__ import annotations

import math

import pytest
import torch
from cache_reference import decoded, random_cache
from transformer_reference import assert_within, attention_f64

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)
CODES = (torch.float8_e4m3fn, torch.int8)


def _ops():
    import mlx_lattice_amd.ops as ops

    return ops


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _offsets(counts, start=0):
    out = [start]
    for n in counts:
        out.append(out[-1] + n)
    return _ints(*out)


def _reference(q, cache, counts, lengths, left, right, sinks, scale,
               first=0, device='cpu'):
    keys, values = decoded(cache)
    spans, at = [], first
    for s, (count, length) in enumerate(zip(counts, lengths)):
        spans.append((at, count, s * cache.capacity, length))
        at += count
    flat = [t.reshape(-1, *t.shape[2:]) for t in (keys, values)]
    return attention_f64(q, *flat, spans, left, right, sinks, scale,
                         device=device)[0]


def _check(q, cache, counts, lengths, left=None, right=0, sinks=0, scale=None,
           offsets=None, first=0, device='cpu'):
    got = _ops().cache_attention(
        q, cache, offsets=_offsets(counts, first) if offsets is None
        else offsets, lengths=_ints(*lengths), left=left, right=right,
        sinks=sinks, scale=scale)
    assert got.shape == q.shape and got.dtype == q.dtype
    want, bound = _reference(
        q, cache, counts, lengths, left, right, sinks,
        q.shape[-1] ** -0.5 if scale is None else scale, first, device)
    assert_within(got, want, bound)
    return got


def _queries(gen, dtype, rows, heads, dim, scale=1.0):
    q = torch.randn((rows, heads + 3, dim), generator=gen, device='cuda')
    return (q * scale).to(dtype)[:, :heads]


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize(
    'counts, lengths, capacity, heads, kv_heads, dim, left, right, sinks', [
        ((1,), (1,), 32, 1, 1, 32, None, 0, 0),
        ((1,), (33,), 64, 4, 2, 64, None, 0, 0),
        ((1, 1), (500, 31), 512, 8, 2, 128, None, 0, 0),
        ((1, 1, 1), (400, 7, 333), 416, 4, 4, 96, 100, 0, 4),
        ((1,) * 4, (2000, 1999, 1500, 64), 2016, 8, 1, 64, 512, 0, 4),
        ((5, 0, 17), (40, 9, 100), 128, 6, 2, 80, None, 0, 0),
        ((64,), (64,), 64, 2, 2, 32, None, None, 0),
        ((33, 70), (200, 70), 224, 4, 2, 128, 50, 10, 3),
        ((200,), (1111,), 1120, 8, 2, 64, 300, 0, 40),
        ((90, 1), (90, 700), 704, 3, 1, 16, 0, 0, 1),
        ((31,), (900,), 928, 2, 2, 24, 64, 31, 0),
        ((3,), (3,), 32, 20, 1, 32, 1, 1, 0)])
def test_tokens_and_chunks(counts, lengths, capacity, heads, kv_heads, dim,
                           left, right, sinks, dtype, code):
    gen = torch.Generator(device='cuda').manual_seed(1)
    cache = random_cache(gen, code, len(counts), capacity, kv_heads, dim)
    q = _queries(gen, dtype, sum(counts), heads, dim)
    _check(q, cache, counts, lengths, left, right, sinks)


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', (1, 2, 7, 30, 33, 36, 100, 127))
def test_any_number_of_channels(dim, dtype, code):
    gen = torch.Generator(device='cuda').manual_seed(2)
    cache = random_cache(gen, code, 2, 160, 1, dim)
    q = _queries(gen, dtype, 42, 2, dim)
    _check(q, cache, (40, 2), (150, 160), 60, 0, 5)


# Rows enough for waves of their own, and chunks against long caches.
@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize(
    'counts, lengths, heads, kv_heads, dim, left, right, sinks', [
        ((3000, 2501), (3500, 2501), 16, 8, 64, 200, 0, 5),
        ((1500, 0, 700, 1, 2411), (1500, 9, 900, 3000, 2411), 8, 8, 32, 90, 9,
         3),
        ((2100, 1900), (2500, 1900), 12, 12, 80, 130, 0, 37),
        ((2200, 33, 1500), (2300, 3000, 1501), 12, 4, 128, None, 0, 0),
        ((2500,), (3100,), 16, 16, 96, 300, 20, 0)])
def test_many_rows(counts, lengths, heads, kv_heads, dim, left, right, sinks,
                   dtype, code):
    gen = torch.Generator(device='cuda').manual_seed(3)
    cache = random_cache(gen, code, len(counts), 3520, kv_heads, dim)
    q = _queries(gen, dtype, sum(counts), heads, dim)
    _check(q, cache, counts, lengths, left, right, sinks, device='cuda')


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('counts, lengths, heads, kv_heads, dim', [
    ((1,), (20000,), 4, 1, 128), ((1, 2), (9000, 4), 8, 2, 64),
    ((16,), (7001,), 2, 1, 96), ((1, 1), (5000, 8191), 1, 1, 32)])
def test_split_tokens(counts, lengths, heads, kv_heads, dim, dtype, code):
    gen = torch.Generator(device='cuda').manual_seed(4)
    cache = random_cache(gen, code, len(counts), 20000, kv_heads, dim)
    q = _queries(gen, dtype, sum(counts), heads, dim)
    _check(q, cache, counts, lengths, device='cuda')


@pytest.mark.parametrize('dtype', DTYPES)
def test_many_short_sequences(dtype):
    gen = torch.Generator(device='cuda').manual_seed(5)
    counts = [s % 4 for s in range(600)]
    lengths = [c + s % 30 for s, c in enumerate(counts)]
    cache = random_cache(gen, torch.int8, 600, 64, 1, 32)
    _check(_queries(gen, dtype, sum(counts), 2, 32), cache, counts, lengths, 7,
           1, 2, device='cuda')


# On either side of what one read of the offsets finds, written and attended.
@pytest.mark.parametrize('first', (0, 5))
@pytest.mark.parametrize('batches', (1, 60, 61, 62, 63, 64, 65, 130))
def test_numbers_of_sequences(batches, first):
    gen = torch.Generator(device='cuda').manual_seed(17)
    counts = [(3 * s + 1) % 5 for s in range(batches)]
    lengths = [c + s % 50 for s, c in enumerate(counts)]
    cache = random_cache(gen, torch.int8, batches, 64, 1, 32)
    rows = first + sum(counts) + 4
    q = _queries(gen, torch.float16, rows, 2, 32)
    k, v = (torch.randn((rows, 1, 32), generator=gen, device='cuda')
            for _ in range(2))
    before = decoded(cache)
    at = _offsets(counts, first)
    _ops().write_cache(cache, k, v, offsets=at, lengths=_ints(*lengths))
    for got, then, new in zip(decoded(cache), before, (k, v)):
        place = first
        for s, (count, length) in enumerate(zip(counts, lengths)):
            # Magnitudes are below 7.9 = 127 2^-4: half a step is 2^-5.
            wanted = new[place:place + count, 0].cpu().double()
            place += count
            start = length - count
            now, was = got[s, :length, 0], then[s, :start, 0]
            assert ((now[start:] - wanted).abs() <= 2.0 ** -5).all()
            assert ((now[:start] - was).abs() <= 2.0 ** -5).all()
    got = _check(q, cache, counts, lengths, 20, 1, 2, first=first,
                 device='cuda')
    assert not got[:first].any() and not got[-4:].any()


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('heads, count', ((4, 1), (4, 9), (64, 70)))
def test_blocks_of_unequal_exponents(heads, count, dtype, code):
    """Values of blocks from 2^-60 to 2^8 of one another, whose large ones may
    have next to no share: no share leaves the type's range."""
    gen = torch.Generator(device='cuda').manual_seed(6)
    cache = random_cache(gen, code, 1, 1024, 4, 64, -9, -6)
    cache.value_exponents.copy_(torch.randint(
        -60, 0, cache.value_exponents.shape, generator=gen, device='cuda'))
    cache.value_exponents[:, :, ::5] = 0
    # The keys of blocks of large values lie against the queries.
    q = _queries(gen, dtype, count, heads, 64).abs() + 0.5
    keys = cache.keys.float().abs() + 1
    keys[:, :, 160 * 5:] *= 1
    keys.view(1, 4, 32, 32, 64)[:, :, ::5] *= -1
    cache.keys.copy_(keys.clamp(-127, 127))
    cache.value_exponents[:, :, 20:] = -126
    got = _check(q, cache, (count,), (1000,))
    assert torch.isfinite(got).all()


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('counts, lengths', (((1, 1), (300, 77)),
                                             ((40, 70), (300, 200)),
                                             ((1500, 1500), (1600, 1500))))
def test_what_is_not_seen_never_arrives(counts, lengths, dtype, code):
    """NaN and the largest codes and exponents in tokens that no query, or
    only some queries, see."""
    gen = torch.Generator(device='cuda').manual_seed(7)
    cache = random_cache(gen, code, 2, 1600, 2, 64)
    q = _queries(gen, dtype, sum(counts), 4 if counts[0] < 100 else 20, 64)
    spoilt = 0x7f
    for s, length in enumerate(lengths):
        # Behind the end, and before every window.
        cache.keys.view(torch.uint8)[s, :, length:] = spoilt
        values = cache.values.view(torch.uint8)[s].movedim(3, 2)
        place = torch.arange(1600, device='cuda').view(50, 32)
        values[:, place >= length] = spoilt
        cache.key_exponents[s, :, (length + 31) // 32:] = 127
        cache.value_exponents[s, :, (length + 31) // 32:] = 127
        early = max(0, min(20, length - counts[s] - 60))
        cache.keys.view(torch.uint8)[s, :, 4:early] = spoilt
        values[:, (place >= 4) & (place < early)] = spoilt
    got = _check(q, cache, counts, lengths, 40, 0, 4,
                 device='cuda' if counts[0] > 100 else 'cpu')
    assert torch.isfinite(got).all()
    # One value that the later rows see.
    if code != torch.float8_e4m3fn:
        return
    at = lengths[0] - 30
    cache.values.view(torch.uint8)[0, 1, at // 32, 9, at % 32] = spoilt
    got = _check(q, cache, counts, lengths, 40, 0, 4,
                 device='cuda' if counts[0] > 100 else 'cpu')
    assert torch.isnan(got).any() and not torch.isnan(got).all()
    cache.keys.view(torch.uint8)[1, 0, lengths[1] - 3, 5] = spoilt
    _check(q, cache, counts, lengths, 40, 0, 4,
           device='cuda' if counts[0] > 100 else 'cpu')


@pytest.mark.parametrize('value', (math.inf, -math.inf, math.nan))
@pytest.mark.parametrize('dtype', DTYPES)
def test_non_finite_queries_stay_in_their_rows(dtype, value):
    gen = torch.Generator(device='cuda').manual_seed(8)
    cache = random_cache(gen, torch.int8, 1, 320, 2, 64)
    q = _queries(gen, dtype, 30, 4, 64).clone()
    clean = _ops().cache_attention(q, cache, offsets=_ints(0, 30),
                                   lengths=_ints(300), right=0)
    q[11, 2, 5] = value
    got = _ops().cache_attention(q, cache, offsets=_ints(0, 30),
                                 lengths=_ints(300), right=0)
    assert torch.isnan(got[11, 2]).all()
    got[11, 2] = clean[11, 2]
    assert torch.equal(got, clean)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('left, right, sinks', (
    (None, 0, 0), (3, 0, 2), (None, None, 0), (None, 5, 0)))
def test_queries_before_the_tokens_see_nothing(left, right, sinks, dtype):
    """More queries than the length counts: the first have positions below
    zero; and no tokens at all."""
    gen = torch.Generator(device='cuda').manual_seed(9)
    cache = random_cache(gen, torch.int8, 3, 64, 1, 32)
    q = _queries(gen, dtype, 70, 2, 32)
    _check(q, cache, (50, 10, 10), (20, 0, 64), left, right, sinks)


@pytest.mark.parametrize('dtype', DTYPES)
def test_rows_in_no_sequence_are_zero(dtype):
    gen = torch.Generator(device='cuda').manual_seed(10)
    cache = random_cache(gen, torch.int8, 2, 64, 2, 32)
    q = _queries(gen, dtype, 500, 4, 32)
    got = _check(q, cache, (10, 20), (40, 60), first=200)
    assert not got[:200].any() and not got[230:].any()


def test_lengths_past_the_capacity():
    """Positions are those of the length; the tokens are those there are."""
    gen = torch.Generator(device='cuda').manual_seed(11)
    cache = random_cache(gen, torch.int8, 2, 64, 1, 32)
    q = _queries(gen, torch.float32, 20, 2, 32)
    at = _offsets((10, 10))
    got = _ops().cache_attention(q, cache, offsets=at, lengths=_ints(70, 2000),
                                 left=20, right=0)
    keys, values = decoded(cache)
    for i in range(10):
        p = 60 + i
        seen = slice(max(0, p - 20), min(64, p + 1))
        for head in range(2):
            scores = keys[0, seen, 0] @ q[i, head].cpu().double() / 32 ** 0.5
            want = torch.softmax(scores, 0) @ values[0, seen, 0]
            assert (got[i, head].cpu().double() - want).abs().max() < 1e-5
    assert not got[10:].any()
    # Without a bound every token is seen, however far the length.
    for lengths in ((2000, 2 ** 29), (2 ** 31 - 1, 2 ** 31 - 1)):
        for right in (0, None):
            far = _ops().cache_attention(q, cache, offsets=at, right=right,
                                         lengths=_ints(*lengths))
            for i in range(20):
                scores = keys[i // 10, :, 0] @ q[i, 0].cpu().double()
                want = torch.softmax(scores / 32 ** 0.5,
                                     0) @ values[i // 10, :, 0]
                assert (far[i, 0].cpu().double() - want).abs().max() < 1e-5
    most = _ops().cache_attention(q, cache, offsets=at, left=5, sinks=3,
                                  lengths=_ints(2 ** 31 - 1, -7), right=0)
    sinks = _check(q[:1], cache, (1, 0), (64, 0), 0, 0, 3)
    assert torch.isfinite(most).all() and not most[10:].any()
    assert sinks.shape == (1, 2, 32)


def test_offsets_out_of_range_are_clamped():
    gen = torch.Generator(device='cuda').manual_seed(12)
    cache = random_cache(gen, torch.int8, 2, 64, 1, 32)
    q = _queries(gen, torch.float16, 50, 2, 32)
    _check(q, cache, (20, 30), (40, 50), offsets=_ints(-5, 20, 99))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', (90, 6000))
def test_offsets_that_decrease_stay_inside(rows, dtype):
    """Results are unspecified; nothing outside the tensors is written."""
    gen = torch.Generator(device='cuda').manual_seed(13)
    cache = random_cache(gen, torch.int8, 3, 64, 8, 32)
    q = _queries(gen, dtype, rows, 16, 32)
    for offsets in ((rows, 5, rows // 2, 0), (7, rows, 3, rows),
                    (rows, rows - 1, 1, 0)):
        _ops().cache_attention(q, cache, offsets=_ints(*offsets),
                               lengths=_ints(64, 30, 50))
    torch.cuda.synchronize()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('scale', (-0.3, 0.0, -0.0, 1e-30, 4.0))
def test_scales(scale, dtype):
    gen = torch.Generator(device='cuda').manual_seed(14)
    cache = random_cache(gen, torch.float8_e4m3fn, 2, 160, 2, 64)
    q = _queries(gen, dtype, 21, 4, 64)
    if scale >= 0:
        _check(q, cache, (20, 1), (160, 50), 60, 0, 3, scale)
    else:  # as the negated queries
        at = _offsets((20, 1))
        args = {'offsets': at, 'lengths': _ints(160, 50), 'left': 60,
                'right': 0, 'sinks': 3}
        assert torch.equal(
            _ops().cache_attention(q, cache, scale=scale, **args),
            _ops().cache_attention(-q, cache, scale=-scale, **args))
        _check(-q, cache, (20, 1), (160, 50), 60, 0, 3, -scale)


@pytest.mark.parametrize('dtype', (torch.float32, torch.bfloat16))
@pytest.mark.parametrize('heads, rows', ((4, 3), (64, 600)))
def test_keys_next_to_nothing_under_large_queries(heads, rows, dtype):
    """The factor of the scores, 0.05 log2(e) 2^-126, is below the normal
    numbers; the scores are some 0.005."""
    gen = torch.Generator(device='cuda').manual_seed(16)
    cache = random_cache(gen, torch.int8, 1, 704, 2, 128)
    cache.key_exponents.fill_(-126)
    q = _queries(gen, dtype, rows, heads, 128, 2.0 ** 114)
    got = _ops().cache_attention(q, cache, offsets=_ints(0, rows),
                                 lengths=_ints(700), right=0, scale=0.05)
    want, bound = _reference(q, cache, (rows,), (700,), None, 0, 0, 0.05,
                             device='cuda')
    # The factor is over 2^-130 and a multiple of 2^-149: off by at most 2^-20
    # of it.  That much of the scores (below 1) goes into the shares, on either
    # side of the quotient.
    values = decoded(cache)[1].abs().max()
    assert_within(got, want, bound.cpu() + values * 2 * 2.0 ** -20)


def test_long_tail_under_one_large_score():
    """A token with 2^13 times the share of each of 16,000 others, whose
    values the result is made of, in half precision."""
    from mlx_lattice_amd import QuantizedCache

    cache = QuantizedCache.empty(1, 16384, 1, 32, dtype=torch.int8,
                                 device='cuda')
    cache.keys[0, 0, 0, 0] = 64  # the score of the first token: 13 log 2
    cache.key_exponents.zero_()
    cache.values[:, :, :, 1] = 1
    cache.values[0, 0, 0, 1, 0] = 0
    q = torch.zeros((1, 1, 32), device='cuda', dtype=torch.float16)
    q[0, 0, 0] = 1
    scale = 13 * math.log(2) / 64
    got = _ops().cache_attention(q, cache, offsets=_ints(0, 1),
                                 lengths=_ints(16000), scale=scale)
    want = 15999 / (15999 + 2.0 ** 13)
    # One rounding of the result and one of equal shares, which are powers of
    # two here; float32 sums.
    assert abs(float(got[0, 0, 1]) - want) <= 2.0 ** -11 * want + 1e-6


def test_strides_and_alignment():
    gen = torch.Generator(device='cuda').manual_seed(15)
    cache = random_cache(gen, torch.int8, 1, 96, 2, 32)
    x = torch.randn((80, 9, 40), generator=gen, device='cuda').half()
    for q in (x[::2, :4, 3:35], x[:40, ::2, 8:40][:, :4],
              x[:40, :1, :32].expand(40, 4, 32),
              x[:40, :4, :32].movedim(2, 0).contiguous().movedim(0, 2),
              x[:40, :, :36].transpose(1, 2)[:, :32, :4].transpose(1, 2)):
        _check(q, cache, (40,), (90,))


@pytest.mark.parametrize('dtype', DTYPES)
def test_same_result_each_time(dtype):
    gen = torch.Generator(device='cuda').manual_seed(16)
    cache = random_cache(gen, torch.float8_e4m3fn, 2, 4096, 2, 64)
    q = _queries(gen, dtype, 2, 8, 64)
    args = {'offsets': _ints(0, 1, 2), 'lengths': _ints(4000, 3777)}
    first = _ops().cache_attention(q, cache, **args)
    for _ in range(3):
        assert torch.equal(first, _ops().cache_attention(q, cache, **args))


def test_tokens_past_32_bits():
    from mlx_lattice_amd import QuantizedCache

    gen = torch.Generator(device='cuda').manual_seed(17)
    capacity = (1 << 25) + 64  # of 128 channels: 4 GiB a part and a bit
    cache = QuantizedCache.empty(1, capacity, 1, 128, dtype=torch.int8,
                                 device='cuda')
    small = random_cache(gen, torch.int8, 1, 96, 1, 128)
    cache.keys[:, :, -96:] = small.keys
    cache.values[:, :, -3:] = small.values
    cache.key_exponents[:, :, -3:] = small.key_exponents
    cache.value_exponents[:, :, -3:] = small.value_exponents
    for count in (1, 20):
        q = _queries(gen, torch.float16, count, 2, 128)
        got = [_ops().cache_attention(
            q, c, offsets=_ints(0, count), lengths=_ints(length), left=50,
            right=0) for c, length in ((cache, capacity - 5), (small, 91))]
        # The window lies in the same blocks.
        assert torch.equal(*got)


def test_nothing_to_attend_to():
    from mlx_lattice_amd import QuantizedCache

    for batches, capacity, rows in ((0, 64, 5), (2, 0, 5), (2, 64, 0),
                                    (0, 0, 0)):
        cache = QuantizedCache.empty(batches, capacity, 2, 32, device='cuda')
        q = torch.ones((rows, 4, 32), device='cuda')
        at = torch.linspace(0, rows, batches + 1, device='cuda').int()
        out = _ops().cache_attention(
            q, cache, offsets=at, lengths=torch.zeros(
                batches, dtype=torch.int32, device='cuda'))
        assert out.shape == q.shape and not out.any()


def test_refusals():
    from mlx_lattice_amd import QuantizedCache

    ops = _ops()
    cache = QuantizedCache.empty(2, 64, 2, 32, device='cuda')
    q = torch.zeros((4, 4, 32), device='cuda')
    at, lengths = _ints(0, 2, 4), _ints(2, 2)

    def refused(message, error=ValueError, cache=cache, q=q, offsets=at,
                lengths=lengths, **more):
        with pytest.raises(error, match=message):
            ops.cache_attention(q, cache, offsets=offsets, lengths=lengths,
                                **more)

    refused('shape', q=q[:, :, :31])
    refused('shape', q=q[0])
    refused('multiple', q=q[:, :3])
    refused('multiple', q=q[:, :0])
    refused('float32, float16 or bfloat16', q=q.double())
    refused('HIP device tensor', q=q.cpu())
    refused('HIP device tensor', cache=QuantizedCache.empty(2, 64, 2, 32))
    refused('B \\+ 1', offsets=at[:2])
    refused('lengths must have shape', lengths=lengths.long())
    refused('non-negative', left=-1)
    refused('non-negative', sinks=-1)
    refused('no gradient', RuntimeError, q=q.clone().requires_grad_())
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        refused('forward-mode', RuntimeError, q=dual)
