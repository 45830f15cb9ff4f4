"""The transformer operators where their kernels go round again, or scale what
they hold: sizes past the blocks of a launch's cap, small cotangents, large
scores.  Against float64."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch
from transformer_reference import (
    UNIT,
    assert_within,
    attention_f64,
    layer_norm_f64,
    philox_words,
    rotary_f64,
)

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _ops():
    import mlx_lattice_amd.ops as ops

    return ops


def _normal(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device='cuda').to(dtype)


# Rows past 1024 blocks with sums of the weight, past 192 and 256 partials,
# past 4096 blocks (narrow and wide rows), and a second turn of the wide rows'
# column sums.
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows, channels', [
    (70001, 64), (140003, 64), (20011, 30), (5003, 2056), (500, 3000),
    (9001, 512)])
def test_layer_norm_of_many_rows(rows, channels, dtype):
    gen = torch.Generator(device='cuda').manual_seed(31)
    x = (_normal(gen, torch.float32, rows, channels) * 1.5
         + _normal(gen, torch.float32, 1, channels)).to(dtype)
    weight, bias = (_normal(gen, dtype, channels) for _ in range(2))
    dy = _normal(gen, dtype, rows, channels)
    active = rows - 3
    kwargs = {'active_rows': torch.tensor([active], dtype=torch.int32,
                                          device='cuda')}
    refs = layer_norm_f64(x, weight, bias, 1e-5, dy, active)
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    y = _ops().layer_norm(*leaves, **kwargs)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    for name, value, (ref, bound) in zip(('y', 'dx', 'dw', 'db'), got, refs):
        assert_within(value, ref, bound, name)
    # The rows' gradient alone, in a launch without sums.
    y = _ops().layer_norm(x, weight.detach(), bias.detach(), **kwargs)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], got[1])


# Blocks that stay for several tables, with several groups of rows each; pieces
# that fill a wave and that do not; and a lane a channel.
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('heads, dim, dims', [
    (4, 32, (12, 10, 10)), (3, 24, (8, 8, 4)), (2, 128, (44, 42, 42)),
    (5, 10, (4, 2, 2)), (1, 64, (64,))])
def test_rotary_of_many_rows(heads, dim, dims, dtype):
    gen = torch.Generator(device='cuda').manual_seed(32)
    rows = 60001
    x = _normal(gen, dtype, rows, heads + 1, dim)[:, 1:]
    positions = torch.randint(-300, 300, (rows, len(dims)), generator=gen,
                              device='cuda', dtype=torch.int32)
    frequencies = _ops().rotary_frequencies(dims, device='cuda')
    got = _ops().rotary_positions(x, positions, frequencies, dims=dims)
    assert_within(got, *rotary_f64(x, positions, frequencies, dims, False))


@pytest.mark.parametrize('dtype', DTYPES)
def test_dropout_of_many_values(dtype):
    """Past 65,536 blocks: the last values, of a second turn."""
    count = 2 ** 16 * 256 * (16 // dtype.itemsize) + 4096
    x = torch.ones(count, dtype=dtype, device='cuda')
    y = _ops().dropout(x, 0.5, seed=9, offset=4)
    share = float((y != 0).float().mean())
    # Five standard deviations.
    assert abs(share - 0.5) < 2.5 / math.sqrt(count)
    first = count - 4096
    words = _words_from(first // 4, 1024, 9, 4)
    assert (philox_words(8, 9, 4) == _words_from(0, 2, 9, 4)).all()
    kept = torch.from_numpy((words >= 2 ** 31).astype('uint8')).cuda().bool()
    assert torch.equal(y[first:] != 0, kept)


def _words_from(number, counters, seed, offset):
    """philox_words from counter ``number`` on."""
    low = 0xFFFFFFFF
    out = []
    for n in range(number, number + counters):
        c = [n & low, n >> 32, offset & low, offset >> 32 & low]
        k = [seed & low, seed >> 32 & low]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1],
                 a & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        out += c
    return np.array(out, dtype=np.uint64)


@pytest.mark.parametrize('rows, heads, left, right, sinks', [
    (400, 2, 300, 40, 3), (9000, 4, 150, 0, 4)])
def test_small_cotangents_in_half_precision(rows, heads, left, right, sinks):
    """Cotangents of 1e-5, whose slopes lie below half precision's smallest
    number: the gradients are off by the rounding of shares and slopes to
    eleven bits and by their own, not by that of numbers this small."""
    gen = torch.Generator(device='cuda').manual_seed(34)
    q, k, v, dy = (_normal(gen, torch.float16, rows, heads, 32)
                   for _ in range(4))
    dy = (dy.float() * 1e-5).half()
    leaves = [t.requires_grad_() for t in (q, k, v)]
    at = torch.tensor([0, rows], dtype=torch.int32, device='cuda')
    out = _ops().window_attention(*leaves, offsets=at, left=left, right=right,
                                  sinks=sinks)
    got = torch.autograd.grad(out, leaves, dy)
    # Linear in the cotangent: the bound of one of size one, scaled back, in
    # which half precision's smallest steps are smaller by as much.
    scale = 2.0 ** 17
    want = attention_f64(q, k, v, [(0, rows, 0, rows)], left, right, sinks,
                         32 ** -0.5, dy.double() * scale, 'cuda')[1:]
    for name, value, (ref, bound) in zip(('dq', 'dk', 'dv'), got, want):
        assert_within(value, ref / scale, bound / scale + 2.0 ** -25, name)


@pytest.mark.parametrize('dtype', DTYPES)
def test_large_scores_keep_the_shares(dtype):
    """Scores of hundreds: shares are off by their rounding and by that of a
    score in float32, whatever the scores' size."""
    gen = torch.Generator(device='cuda').manual_seed(35)
    rows, dim = 300, 64
    q, k, v, dy = (_normal(gen, dtype, rows, 1, dim) for _ in range(4))
    q, k = q * 4, k * 4
    leaves = [t.requires_grad_() for t in (q, k, v)]
    at = torch.tensor([0, rows], dtype=torch.int32, device='cuda')
    out = _ops().window_attention(*leaves, offsets=at, left=90, right=0)
    got = [out, *torch.autograd.grad(out, leaves, dy)]
    with torch.no_grad():
        q64, k64, v64, d64 = (t[:, 0].double() for t in (q, k, v, dy))
        i = torch.arange(rows, device='cuda')
        seen = (i[None] <= i[:, None]) & (i[None] >= i[:, None] - 90)
        scale = dim ** -0.5
        scores = (q64 @ k64.T * scale).masked_fill(~seen, -math.inf)
        p = torch.softmax(scores, 1)
        o = p @ v64
        dp = d64 @ v64.T
        ds = p * (dp - (d64 * o).sum(1, keepdim=True))
        u = UNIT[dtype]
        # A score: float32's rounding of its 64 products and sums, and of the
        # exponent that it becomes; twice, for the row's largest.
        of_score = (q64.abs() @ k64.abs().T * scale) * 64 * 2.0 ** -24
        loose = u + 2.0 ** -16 + 2 * of_score.amax(1, keepdim=True)
        size = p * (d64.abs() @ v64.abs().T
                    + (d64.abs() * o.abs()).sum(1, keepdim=True))
        # Half precision's shares and slopes below its range (2^-25 of the
        # largest in the row's or the tile's scale).
        tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
        off = 3 * loose * size + tiny * size.amax()
        shares = 2 * loose * p + tiny * seen
        want = [(o, shares @ v64.abs() + u * o.abs()),
                (ds @ k64 * scale, off @ k64.abs() * scale),
                (ds.T @ q64 * scale, off.T @ q64.abs() * scale),
                (p.T @ d64, shares.T @ d64.abs())]
    for name, value, (ref, bound) in zip(('out', 'dq', 'dk', 'dv'), got, want):
        assert_within(value[:, 0], ref, bound + u * ref.abs() + 2.0 ** -25,
                      name)
