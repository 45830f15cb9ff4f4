"""A plain float64 form of the 8-bit cache (test infrastructure): what its codes
stand for, and appending rows block by block."""

from __future__ import annotations

import math

import torch

BLOCK = 32
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def codes_of(cache):
    """Code values of keys and values, (B, heads, tokens, width), on the CPU."""
    keys = cache.keys.cpu().double()
    values = cache.values.cpu().double().movedim(4, 3)
    return keys, values.reshape(keys.shape)


def decoded(cache):
    """The keys and values that the cache stands for, (B, tokens, heads,
    dim)."""
    out = []
    for codes, exponents in zip(codes_of(cache), (cache.key_exponents,
                                                  cache.value_exponents)):
        scale = torch.exp2(exponents.cpu().double()).repeat_interleave(
            BLOCK, 2)[..., None]
        out.append((codes * scale)[..., :cache.dim].transpose(1, 2))
    return out


def rounded(x, dtype):
    """Half to even, to the type's codes."""
    if dtype == torch.int8:
        x = torch.where(torch.isnan(x), 0.0, x)
        return x.round().clamp(-127, 127)
    size = x.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    out = (x / step).round() * step
    return torch.where(torch.isfinite(x), out, math.nan)


def exponent_of(rows, dtype):
    sizes = rows.abs()
    most = float(torch.where(torch.isfinite(sizes), sizes, 0.0).max())
    e = -126
    while most > MOST[dtype] * 2.0 ** e:
        e += 1
    return e


def appended(codes, exponents, rows, dtype, before, total, capacity):
    """One sequence and head: the new code values (tokens, width) and block
    exponents after ``rows`` (float64) became tokens ``before`` to ``total``."""
    codes, exponents = codes.clone(), exponents.clone()
    dim = rows.shape[1]
    new = range(max(before, 0), min(total, capacity))
    for block in sorted({t // BLOCK for t in new}):
        lo = block * BLOCK
        mine = [t for t in new if t // BLOCK == block]
        fresh = rows[mine[0] - before:mine[-1] + 1 - before]
        e = exponent_of(fresh, dtype)
        if mine[0] > lo:
            old = max(int(exponents[block]), -126)
            e = max(e, old)
            if e != old:
                codes[lo:mine[0]] = rounded(
                    codes[lo:mine[0]] * 2.0 ** (old - e), dtype)
        codes[mine[0]:mine[-1] + 1, dim:] = 0
        codes[mine[0]:mine[-1] + 1, :dim] = rounded(fresh * 2.0 ** -e, dtype)
        exponents[block] = e
    return codes, exponents


def random_cache(gen, dtype, batches, capacity, heads, dim, low=-9, high=-4,
                 scale=0.3):
    """A cache full of codes of normal values, on the GPU."""
    from mlx_lattice_amd import QuantizedCache

    cache = QuantizedCache.empty(batches, capacity, heads, dim, dtype=dtype,
                                 device='cuda')
    for part, along in ((cache.keys, -1), (cache.values, -2)):
        x = torch.randn(part.shape, generator=gen, device='cuda')
        x = (x * (MOST[dtype] * scale)).clamp(-MOST[dtype], MOST[dtype])
        x = x.round() if dtype == torch.int8 else x
        x.movedim(along, -1)[..., dim:] = 0
        part.copy_(x.to(dtype))
    for e in (cache.key_exponents, cache.value_exponents):
        e.copy_(torch.randint(low, high, e.shape, generator=gen,
                              device='cuda'))
    return cache


def same_values(got, want):
    return bool(((got == want) | (torch.isnan(got) & torch.isnan(want))).all())
