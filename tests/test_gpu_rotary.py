"""Rotary positions of several axes against float64."""

from __future__ import annotations

import pytest
import torch
from transformer_reference import assert_within, rotary_f64

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _ops():
    import mlx_lattice_amd.ops as ops

    return ops


def _check(x, positions, dims, interleaved=False, base=10000.0):
    ops = _ops()
    frequencies = ops.rotary_frequencies(dims, base, device='cuda')
    leaf = x.detach().requires_grad_()
    y = ops.rotary_positions(leaf, positions, frequencies, dims=dims,
                             interleaved=interleaved)
    assert y.dtype == x.dtype and y.is_contiguous()
    assert_within(y, *rotary_f64(x, positions, frequencies, dims, interleaved),
                  'y')
    dy = torch.randn(x.shape, device='cuda').to(x.dtype)
    grad, = torch.autograd.grad(y, leaf, dy)
    assert_within(grad, *rotary_f64(dy, positions, frequencies, dims,
                                    interleaved, -1.0), 'dx')
    with torch.no_grad():
        assert torch.equal(y, ops.rotary_positions(
            x, positions, frequencies, dims=dims, interleaved=interleaved))


def _rows(rows, heads, dim, dtype, axes, high=300):
    x = torch.randn((rows, heads, dim), device='cuda').to(dtype)
    return x, torch.randint(-high, high, (rows, axes), dtype=torch.int32,
                            device='cuda')


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('interleaved', (False, True))
@pytest.mark.parametrize('rows, heads, dim, dims', [
    (1, 1, 2, (2,)), (1, 8, 64, (64,)), (5, 3, 32, (12, 10, 10)),
    (700, 16, 32, (12, 10, 10)), (33, 5, 48, (16, 16, 16)),
    (3000, 6, 64, (24, 20, 20)), (9, 2, 128, (44, 42, 42)),
    (17, 3, 80, (20, 0, 22, 18)), (11, 4, 24, (4, 6)), (6, 2, 33, (10, 12)),
    (7, 1, 130, (130,)), (4, 3, 1024, (512, 256, 256)), (0, 4, 32, (32,))])
def test_rows(rows, heads, dim, dims, interleaved, dtype):
    _check(*_rows(rows, heads, dim, dtype, len(dims)), dims, interleaved)


@pytest.mark.parametrize('dtype', DTYPES)
def test_slices_of_packed_rows(dtype):
    packed = torch.randn((60, 7, 40), device='cuda').to(dtype)
    coords = torch.randint(0, 500, (60, 4), dtype=torch.int32, device='cuda')
    _check(packed[:, :5, :32], coords[:, 1:], (12, 10, 10))
    _check(packed[:, 1:4, 8:], coords[:, 1:], (12, 10, 10))
    _check(packed[:, :, 1:33], coords[:, 1:], (12, 10, 10))
    _check(packed.transpose(0, 1)[:, :32].contiguous().transpose(0, 1),
           coords[:32, 1:], (12, 10, 10))
    _check(packed[:, :1].expand(60, 4, 40), coords[:, 1:], (40, 0, 0))


def test_far_coordinates_keep_their_angle():
    """Angles of tens of millions of radians, reduced in float64."""
    x, _ = _rows(64, 2, 64, torch.float32, 3)
    positions = torch.randint(-2 ** 26, 2 ** 26, (64, 3), dtype=torch.int32,
                              device='cuda')
    _check(x, positions, (24, 20, 20))


def test_float_positions():
    x, _ = _rows(100, 2, 32, torch.float32, 2)
    _check(x, torch.randn((100, 2), device='cuda') * 50, (16, 16), base=100.0)


def test_relative_positions():
    """A turned pair of rows has a product that depends on their distance."""
    ops = _ops()
    dims = (24, 20, 20)
    frequencies = ops.rotary_frequencies(dims, device='cuda')
    q, k = (torch.randn((1, 1, 64), device='cuda') for _ in range(2))
    products = []
    for shift in (0, 1000):
        a = torch.tensor([[3, 5, 7]], dtype=torch.int32, device='cuda') + shift
        b = torch.tensor([[9, 1, 4]], dtype=torch.int32, device='cuda') + shift
        turned = (ops.rotary_positions(q, a, frequencies, dims=dims)
                  * ops.rotary_positions(k, b, frequencies, dims=dims))
        products.append(float(turned.double().sum()))
    # 64 products of size about 1, each a few float32 roundings off.
    assert abs(products[0] - products[1]) < 64 * 8 * 2.0 ** -22


def test_refusals():
    ops = _ops()
    x, positions = _rows(4, 2, 32, torch.float32, 2)
    f = ops.rotary_frequencies((16, 16), device='cuda')
    for args, dims, message in (
            ((x[0], positions, f), (16, 16), r'shape \(N, heads, dim\)'),
            ((x.double(), positions, f), (16, 16), 'float32, float16'),
            ((x, positions, f), (15, 17), 'even'),
            ((x, positions, f), (32, 32), 'fit the head'),
            ((x, positions, f), (), 'between 1 and 4 axes'),
            ((x, positions[:3], f), (16, 16), 'positions must have shape'),
            ((x, positions.long(), f), (16, 16), 'positions must have shape'),
            ((x, positions, f.float()), (16, 16), 'frequencies must have'),
            ((x, positions, f[:3]), (16, 16), 'frequencies must have'),
            ((x, positions.cpu(), f), (16, 16), 'HIP device tensor')):
        with pytest.raises(ValueError, match=message):
            ops.rotary_positions(*args, dims=dims)
    with pytest.raises(ValueError, match='even'):
        ops.rotary_frequencies((3,))
    with pytest.raises(ValueError, match='base'):
        ops.rotary_frequencies((4,), 0.0)


def test_more_rows_than_blocks_of_a_launch():
    """Rows of many pairs, a block each: 2^24 blocks of 256 threads are more
    than a launch takes."""
    rows, dim = 2 ** 24 + 5, 1022
    x = torch.randn((1, 1, dim), device='cuda').half()
    places = torch.full((1, 1), 7, dtype=torch.int32, device='cuda')
    kwargs = {'frequencies': _ops().rotary_frequencies((dim,), device='cuda'),
              'dims': (dim,)}
    want = _ops().rotary_positions(x, places, **kwargs)
    got = _ops().rotary_positions(x.expand(rows, 1, dim),
                                  places.expand(rows, 1), **kwargs)
    for part in got.split(1 << 20):
        assert torch.equal(part, want.expand_as(part))
