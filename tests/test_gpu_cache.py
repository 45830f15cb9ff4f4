"""Writing rows into an 8-bit cache and reading it back, against a plain form:
codes and exponents are equal, what is not written keeps its bytes."""

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


def _state(cache):
    return [codes_of(cache)[0], codes_of(cache)[1],
            cache.key_exponents.cpu().clone(),
            cache.value_exponents.cpu().clone()]


def _bytes(cache):
    return [p.view(torch.uint8).clone() for p in cache.parts]


def _expected(cache, state, k, v, first, counts, totals):
    """``state`` with the rows from ``first`` on appended."""
    want = [t.clone() for t in state]
    at = first
    for s, (count, total) in enumerate(zip(counts, totals)):
        for which, rows in enumerate((k, v)):
            for head in range(cache.kv_heads):
                if not count:
                    continue
                codes, exponents = appended(
                    state[which][s, head], state[2 + which][s, head],
                    rows[at:at + count, head].detach().cpu().double(),
                    cache.dtype, total - count, total, cache.capacity)
                want[which][s, head] = codes
                want[2 + which][s, head] = exponents
        at += count
    return want


def _check(cache, k, v, counts, totals, offsets=None, first=0):
    state, before = _state(cache), _bytes(cache)
    _ops().write_cache(cache, k, v, lengths=_ints(*totals),
                       offsets=_offsets(counts, first)
                       if offsets is None else offsets)
    want = _expected(cache, state, k, v, first, counts, totals)
    for got, ref in zip(_state(cache), want):
        assert same_values(got, ref)
    # Tokens of blocks that were not written, and those behind the last.
    for which, (then, now) in enumerate(zip(before[:2], _bytes(cache)[:2])):
        if which == 1:
            then, now = (t.movedim(4, 3).reshape(before[0].shape)
                         for t in (then, now))
        for s, (count, total) in enumerate(zip(counts, totals)):
            start = max(0, total - count) // 32 * 32 if count else total
            end = min(max(total, 0), cache.capacity)
            assert torch.equal(then[s, :, :start], now[s, :, :start])
            assert torch.equal(then[s, :, end:], now[s, :, end:])


def _rows(gen, dtype, rows, heads, dim, scale=1.0):
    """Slices of packed rows, tokens of unequal size."""
    kv = torch.randn((rows, 2 * heads + 1, dim), generator=gen, device='cuda')
    size = torch.exp2(torch.randint(-3, 4, (rows, 1, 1), generator=gen,
                                    device='cuda').float())
    kv = (kv * size * scale).to(dtype)
    return kv[:, :heads], kv[:, heads:2 * heads]


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('counts, totals, heads, dim', [
    ((1,), (1,), 1, 32), ((1,), (32,), 2, 64), ((1,), (33,), 1, 128),
    ((2,), (33,), 1, 16), ((31,), (31,), 1, 96), ((32,), (32,), 3, 128),
    ((33,), (34,), 2, 80), ((0, 3, 64), (5, 33, 65), 2, 128),
    ((100, 1, 0, 7), (127, 128, 0, 7), 1, 24), ((1, 1, 1), (96, 65, 1), 4, 96),
    ((128,), (128,), 2, 32)])
def test_blocks(counts, totals, heads, dim, dtype, code):
    gen = torch.Generator(device='cuda').manual_seed(1)
    cache = random_cache(gen, code, len(counts), 128, heads, dim)
    k, v = _rows(gen, dtype, sum(counts), heads, dim)
    _check(cache, k, v, counts, totals)


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', (1, 2, 7, 30, 33, 100, 127))
def test_any_number_of_channels(dim, dtype, code):
    gen = torch.Generator(device='cuda').manual_seed(2)
    cache = random_cache(gen, code, 2, 96, 2, dim)
    k, v = _rows(gen, dtype, 50, 2, dim)
    _check(cache, k, v, (40, 10), (60, 70))


# New tokens far larger and far smaller than the block's earlier ones: codes
# move by 2 to 60 powers of two, or not at all.
@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('scale', (1e-12, 0.05, 1.0, 30.0, 1e4, 1e18))
def test_earlier_codes_are_moved(scale, code):
    gen = torch.Generator(device='cuda').manual_seed(3)
    cache = random_cache(gen, code, 3, 64, 2, 80)
    k, v = _rows(gen, torch.float32, 6, 2, 80, scale)
    _check(cache, k, v, (1, 3, 2), (17, 34, 33))


@pytest.mark.parametrize('code', CODES)
def test_token_by_token(code):
    gen = torch.Generator(device='cuda').manual_seed(4)
    cache = random_cache(gen, code, 2, 96, 2, 48)
    for step in range(70):
        k, v = _rows(gen, torch.bfloat16, 2, 2, 48, 2.0 ** (step % 9))
        _check(cache, k, v, (1, 1), (step + 1, step + 5))


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
def test_written_at_once_or_block_by_block(dtype, code):
    """Whole blocks are the same however many come at once."""
    from mlx_lattice_amd import QuantizedCache

    gen = torch.Generator(device='cuda').manual_seed(5)
    k, v = _rows(gen, dtype, 96, 2, 64)
    caches = [QuantizedCache.empty(1, 96, 2, 64, dtype=code, device='cuda')
              for _ in range(2)]
    _ops().write_cache(caches[0], k, v, offsets=_ints(0, 96),
                       lengths=_ints(96))
    for at in range(0, 96, 32):
        _ops().write_cache(caches[1], k[at:at + 32], v[at:at + 32],
                           offsets=_ints(0, 32), lengths=_ints(at + 32))
    for a, b in zip(*(c.parts for c in caches)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
def test_every_border_between_codes(dtype, code):
    """Values on and next to the borders of rounding, of both signs."""
    gen = torch.Generator(device='cuda').manual_seed(6)
    most = 448.0 if code == torch.float8_e4m3fn else 127.0
    steps = torch.arange(0, 32 * 64, device='cuda').float() / (32 * 64) * most
    k = steps.view(32, 1, 64).to(dtype)
    k[0, 0, 0] = most
    v = torch.where(torch.rand(k.shape, generator=gen, device='cuda') < 0.5,
                    k, -k)
    cache = random_cache(gen, code, 1, 32, 1, 64)
    _check(cache, k, v, (32,), (32,))


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('value', (math.inf, -math.inf, math.nan))
def test_infinities_and_nan(value, code):
    gen = torch.Generator(device='cuda').manual_seed(7)
    cache = random_cache(gen, code, 2, 64, 2, 40)
    k, v = (t.clone() for t in _rows(gen, torch.float16, 20, 2, 40))
    k[3, 0, 5] = value
    v[12, 1, 39] = value
    _check(cache, k, v, (9, 11), (30, 40))
    # Earlier codes of them are moved, too.
    k, v = _rows(gen, torch.float16, 2, 2, 40, 200.0)
    _check(cache, k, v, (1, 1), (31, 41))


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', (32, 33))
def test_infinities_under_far_exponents(dim, dtype, code):
    """Rows that hold nothing finite, whose exponent is the least, and rows
    behind earlier tokens beyond their type's range."""
    gen = torch.Generator(device='cuda').manual_seed(17)
    cache = random_cache(gen, code, 3, 64, 1, dim)
    cache.key_exponents[1] = 110
    cache.value_exponents[1] = -126
    k, v = (t.clone() for t in _rows(gen, dtype, 9, 1, dim))
    k[:3], v[:3] = math.inf, -math.inf
    for rows in (k, v):
        rows[4, 0, 3], rows[5, 0, dim - 1] = -math.inf, math.nan
        rows[8] = math.nan
    _check(cache, k, v, (3, 3, 3), (3, 40, 34))


@pytest.mark.parametrize('code', CODES)
def test_zeros_and_values_at_the_ends_of_float32(code):
    gen = torch.Generator(device='cuda').manual_seed(8)
    cache = random_cache(gen, code, 4, 32, 1, 32)
    k = torch.zeros((8, 1, 32), device='cuda')
    v = k.clone()
    k[2:4, 0, :5] = 1e-42  # subnormal
    k[4:6] = torch.finfo(torch.float32).max
    v[4:6, 0, ::2] = -2.0 ** -126
    v[6:8, 0, 7] = 2.0 ** -119
    _check(cache, k, v, (2, 2, 2, 2), (2, 9, 5, 2))


@pytest.mark.parametrize('code', CODES)
def test_tokens_outside_the_capacity_are_not_written(code):
    gen = torch.Generator(device='cuda').manual_seed(9)
    cache = random_cache(gen, code, 4, 64, 2, 32)
    k, v = _rows(gen, torch.float16, 150, 2, 32)
    # Past the end, across it, more rows than the length counts, a length
    # that is no length.
    _check(cache, k, v, (10, 70, 60, 10), (2000, 90, 40, -3))
    _check(cache, k, v, (1, 1, 1, 1), (65, 64, 2 ** 31 - 1, 0))


def test_rows_in_no_sequence_and_offsets_out_of_range():
    gen = torch.Generator(device='cuda').manual_seed(10)
    cache = random_cache(gen, torch.int8, 2, 64, 1, 32)
    k, v = _rows(gen, torch.float16, 50, 1, 32)
    _check(cache, k, v, (10, 12), (10, 20), first=7)
    # Clamped to the rows there are.
    _check(cache, k, v, (20, 30), (40, 50), offsets=_ints(-5, 20, 99))


@pytest.mark.parametrize('code', CODES)
def test_offsets_that_decrease_stay_inside(code):
    """What is written is unspecified; nothing outside the cache is."""
    from mlx_lattice_amd import QuantizedCache

    gen = torch.Generator(device='cuda').manual_seed(11)
    whole = random_cache(gen, code, 6, 64, 2, 32)
    inner = QuantizedCache(*(p[2:4] for p in whole.parts), 32)
    k, v = _rows(gen, torch.float16, 100, 2, 32)
    then = _bytes(whole)
    for offsets in ((90, 5, 60), (100, 50, 0), (40, 39, 41)):
        _ops().write_cache(inner, k, v, offsets=_ints(*offsets),
                           lengths=_ints(50, 60))
    for a, b in zip(then, _bytes(whole)):
        assert torch.equal(a[:2], b[:2]) and torch.equal(a[4:], b[4:])


def test_strides():
    """Rows and heads of any stride, heads that share one row, channels that
    are not adjacent."""
    gen = torch.Generator(device='cuda').manual_seed(12)
    cache = random_cache(gen, torch.int8, 1, 64, 4, 32)
    x = torch.randn((64, 9, 40), generator=gen, device='cuda').half()
    for k, v in ((x[::2, :4, 3:35], x[::2, 4:8, 8:40]),
                 (x[:32, :1, :32].expand(32, 4, 32), x[1:33, 1::2, :32]),
                 (x[:32, :4].transpose(1, 2)[:, :32].transpose(1, 2),
                  x[:32].movedim(2, 1)[:, :32].movedim(1, 2)[:, :4])):
        _check(cache, k, v, (32,), (40,))
    k = torch.randn((32, 32, 4), generator=gen, device='cuda').transpose(1, 2)
    _check(cache, k, k * 2, (32,), (50,))


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('batches, capacity, heads, dim', [
    (1, 32, 1, 32), (3, 96, 2, 80), (2, 160, 3, 128), (2, 64, 1, 7),
    (1, 64, 5, 33), (70, 32, 1, 16)])
def test_read(batches, capacity, heads, dim, dtype, code):
    gen = torch.Generator(device='cuda').manual_seed(13)
    cache = random_cache(gen, code, batches, capacity, heads, dim)
    totals = [(7 * s + capacity - 9) % (capacity + 40) for s in range(batches)]
    got = _ops().read_cache(cache, lengths=_ints(*totals), dtype=dtype)
    filled = (torch.arange(capacity)[None] < torch.tensor(totals)[:, None])
    for rows, want in zip(got, decoded(cache)):
        assert rows.shape == (batches, capacity, heads, dim)
        assert rows.dtype == dtype
        want = torch.where(filled[..., None, None], want, 0.0)
        # Codes have at most 7 bits: exact in every type.
        assert torch.equal(rows.cpu().double(), want)


def test_read_of_nan_and_far_exponents():
    gen = torch.Generator(device='cuda').manual_seed(14)
    cache = random_cache(gen, torch.float8_e4m3fn, 1, 64, 1, 32, -120, 100)
    cache.keys.view(torch.uint8)[0, 0, 5, 3] = 0x7f
    cache.values.view(torch.uint8)[0, 0, 1, 7, 9] = 0xff
    cache.keys.view(torch.uint8)[0, 0, 60, 3] = 0x7f
    k, v = _ops().read_cache(cache, lengths=_ints(60))
    want_k, want_v = decoded(cache)
    want_k[:, 60:] = want_v[:, 60:] = 0.0
    assert same_values(k.cpu().double(), want_k.float().double())
    assert same_values(v.cpu().double(), want_v.float().double())
    assert torch.isnan(k).sum() == 1 and torch.isnan(v).sum() == 1


def test_nothing_to_write_or_read():
    from mlx_lattice_amd import QuantizedCache

    empty = torch.zeros((0, 2, 32), device='cuda')
    for batches, capacity in ((0, 64), (2, 0), (2, 64)):
        cache = QuantizedCache.empty(batches, capacity, 2, 32, device='cuda')
        lengths = torch.zeros(batches, dtype=torch.int32, device='cuda')
        _ops().write_cache(cache, empty, empty, lengths=lengths,
                           offsets=_ints(*[0] * (batches + 1)))
        k, _ = _ops().read_cache(cache, lengths=lengths)
        assert k.shape == (batches, cache.capacity, 2, 32) and not k.any()


def test_many_sequences():
    gen = torch.Generator(device='cuda').manual_seed(15)
    counts = [s % 4 for s in range(500)]
    totals = [c + s % 60 for s, c in enumerate(counts)]
    cache = random_cache(gen, torch.int8, 500, 64, 1, 16)
    k, v = _rows(gen, torch.bfloat16, sum(counts), 1, 16)
    _check(cache, k, v, counts, totals)


def test_cache_past_32_bits():
    """Tokens whose bytes lie past 2^32, written and read back."""
    from mlx_lattice_amd import QuantizedCache

    gen = torch.Generator(device='cuda').manual_seed(16)
    capacity = (1 << 25) + 64  # of 128 channels: 4 GiB a part and a bit
    cache = QuantizedCache.empty(1, capacity, 1, 128, dtype=torch.int8,
                                 device='cuda')
    k, v = _rows(gen, torch.float16, 40, 1, 128)
    total = capacity - 3
    _ops().write_cache(cache, k, v, offsets=_ints(0, 40), lengths=_ints(total))
    tail = QuantizedCache(
        cache.keys[:, :, -96:].contiguous(),
        cache.values[:, :, -3:].contiguous(),
        cache.key_exponents[:, :, -3:].contiguous(),
        cache.value_exponents[:, :, -3:].contiguous(), 128)
    small = QuantizedCache.empty(1, 96, 1, 128, dtype=torch.int8,
                                 device='cuda')
    _ops().write_cache(small, k, v, offsets=_ints(0, 40), lengths=_ints(93))
    for a, b in zip(tail.parts, small.parts):
        assert torch.equal(a, b)
    assert not cache.keys[:, :, :-96].any()
    del tail, small
    torch.cuda.empty_cache()
    keys, _ = _ops().read_cache(cache, lengths=_ints(total),
                                dtype=torch.float16)
    exponents = cache.key_exponents[0, 0, -3:].cpu().double()
    want = (cache.keys[0, 0, -96:].cpu().double()
            * torch.exp2(exponents).repeat_interleave(32)[:, None])
    want[-3:] = 0
    assert torch.equal(keys[0, -96:, 0].cpu().double(), want)


def test_other_stream_and_version():
    from mlx_lattice_amd import QuantizedCache

    gen = torch.Generator(device='cuda').manual_seed(17)
    k, v = _rows(gen, torch.float16, 60, 2, 64)
    caches = [QuantizedCache.empty(1, 64, 2, 64, device='cuda')
              for _ in range(2)]
    versions = [p._version for p in caches[0].parts]
    args = {'offsets': _ints(0, 60), 'lengths': _ints(60)}
    _ops().write_cache(caches[0], k, v, **args)
    assert all(p._version > n for p, n in zip(caches[0].parts, versions))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _ops().write_cache(caches[1], k, v, **args)
        rows = _ops().read_cache(caches[1], lengths=args['lengths'])
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(*(c.parts for c in caches)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for a, b in zip(rows, _ops().read_cache(caches[0],
                                            lengths=args['lengths'])):
        assert torch.equal(a, b)


def test_refusals():
    from mlx_lattice_amd import QuantizedCache

    ops = _ops()
    cache = QuantizedCache.empty(2, 64, 2, 32, device='cuda')
    k = torch.zeros((4, 2, 32), device='cuda')
    at, lengths = _ints(0, 2, 4), _ints(2, 2)

    def refused(message, error=ValueError, cache=cache, k=k, v=k, offsets=at,
                lengths=lengths):
        with pytest.raises(error, match=message):
            ops.write_cache(cache, k, v, offsets=offsets, lengths=lengths)

    refused('shape', k=k[:, :1])
    refused('shape', v=k[:, :, :31])
    refused('shape', k=k[:3])
    refused('float32, float16 and bfloat16|float32, float16 or bfloat16',
            k=k.double(), v=k.double())
    refused('share a dtype', v=k.half())
    refused('HIP device tensor', v=k.cpu())
    refused('B \\+ 1', offsets=at[:2])
    refused('B \\+ 1', offsets=at.long())
    refused('lengths must have shape', lengths=_ints(2))
    refused('contiguous', offsets=_ints(0, 0, 2, 2, 4, 4)[::2])
    refused('no gradient', RuntimeError, k=k.clone().requires_grad_())
    with torch.no_grad():
        ops.write_cache(cache, k.clone().requires_grad_(), k, offsets=at,
                        lengths=lengths)
    with pytest.raises(ValueError, match='lengths must have shape'):
        ops.read_cache(cache, lengths=at)
    with pytest.raises(ValueError, match='float32, float16 or bfloat16'):
        ops.read_cache(cache, lengths=lengths, dtype=torch.float64)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(k, torch.ones_like(k))
        refused('forward-mode', RuntimeError, k=dual)
