"""Layer norm and its gradients against float64."""

from __future__ import annotations

import pytest
import torch
from transformer_reference import assert_within, layer_norm_f64

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _ops():
    import mlx_lattice_amd.ops as ops

    return ops


def _inputs(rows, channels, dtype, seed=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device='cuda')

    x = (normal(rows, channels) * (torch.arange(rows, device='cuda')[:, None]
                                   % 5 + 0.5) + 2 * normal(1, channels))
    return (x.to(dtype), (1 + 0.3 * normal(channels)).to(dtype),
            normal(channels).to(dtype), normal(rows, channels).to(dtype))


def _check(x, weight, bias, dy, eps=1e-5, active=None):
    ops = _ops()
    count = (None if active is None else torch.tensor(
        [active], dtype=torch.int32, device='cuda'))
    leaves = [t.detach().requires_grad_() if t is not None else None
              for t in (x, weight, bias)]
    with torch.no_grad():
        plain = ops.layer_norm(*leaves, eps=eps, active_rows=count)
    y = ops.layer_norm(*leaves, eps=eps, active_rows=count)
    assert torch.equal(plain, y)
    want = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, want, dy))
    refs = layer_norm_f64(x, weight, bias, eps, dy, active)
    got = [y] + [next(grads) if t is not None else None for t in leaves]
    for name, value, (ref, bound) in zip(('y', 'dx', 'dw', 'db'), got, refs):
        if value is not None:
            assert value.dtype == x.dtype
            assert_within(value, ref, bound, name)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows, channels', [
    (1, 1), (1, 8), (5, 3), (257, 7), (17, 30), (1000, 32), (33, 96),
    (513, 128), (7, 130), (10, 1000), (31, 1024), (3, 2049), (5, 2056),
    (3, 8200), (4500, 16)])
def test_rows(rows, channels, dtype):
    _check(*_inputs(rows, channels, dtype))


@pytest.mark.parametrize('dtype', DTYPES)
def test_without_weight_or_bias(dtype):
    x, weight, bias, dy = _inputs(77, 48, dtype)
    _check(x, None, None, dy)
    _check(x, weight, None, dy)
    _check(x, None, bias, dy)


@pytest.mark.parametrize('dtype', DTYPES)
def test_strided_and_misaligned_rows(dtype):
    wide, weight, bias, dy = _inputs(65, 131, dtype)
    _check(wide[:, 1:65], weight[:64], bias[1:65], dy[:, 3:67])
    _check(wide[:, :64], weight[3:67], bias[:64], dy[:, :64])
    _check(wide.t()[:128], *_inputs(128, 65, dtype)[1:])
    _check(wide[:1].expand(9, 131), weight, bias, dy[:9])


@pytest.mark.parametrize('channels', (24, 3000))
@pytest.mark.parametrize('active', (0, 1, 40, 64, 99))
def test_inactive_rows_are_zero_and_take_no_part(active, channels):
    x, weight, bias, dy = _inputs(64, channels, torch.float32)
    x[active:] = float('nan')
    dy[active:] = float('inf')
    _check(x, weight, bias, dy, active=active)


def test_no_rows():
    x, weight, bias, dy = _inputs(3, 20, torch.float16)
    _check(x[:0], weight, bias, dy[:0])


def test_large_mean_does_not_cancel():
    x, weight, bias, dy = _inputs(50, 256, torch.float32)
    _check(x + 4096.0, weight, bias, dy)


def test_constant_rows_and_eps():
    _, weight, bias, dy = _inputs(9, 64, torch.float32)
    _check(torch.full((9, 64), 3.0, device='cuda'), weight, bias, dy,
           eps=1e-3)


def test_gradient_against_differences():
    x, weight, bias, dy = _inputs(12, 40, torch.float32)
    ops = _ops()
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    grads = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        way = torch.randn_like(leaf)
        way = way / way.norm()
        ends = []
        for step in (0.02, -0.02):
            moved = [t.detach() for t in leaves]
            moved[i] = moved[i] + step * way
            ends.append((ops.layer_norm(*moved).double() * dy).sum())
        slope = float((ends[0] - ends[1]) / 0.04)
        # Central differences of step 0.02 leave a third-order term of about
        # 0.02^2 of the slope's size; the float32 forward, 480 roundings of
        # 2^-24 over 0.04, is smaller.
        size = float(grad.norm())
        assert abs(slope - float((grad.double() * way).sum())) < 5e-3 * size


def test_same_result_each_time():
    x, weight, bias, dy = _inputs(70001, 64, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    runs = [torch.autograd.grad(_ops().layer_norm(*leaves), leaves, dy)
            for _ in range(2)]
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_sparse_tensor():
    from mlx_lattice_amd import SparseTensor

    x, weight, bias, _ = _inputs(20, 16, torch.float32)
    coords = torch.zeros((20, 4), dtype=torch.int32, device='cuda')
    coords[:, 1] = torch.arange(20)
    active = torch.tensor([15], dtype=torch.int32, device='cuda')
    sparse = SparseTensor(coords, x, active_rows=active)
    out = _ops().layer_norm(sparse, weight, bias)
    assert out.same_coords(sparse)
    assert_within(out.feats, *layer_norm_f64(x, weight, bias, 1e-5, active=15))
    with pytest.raises(ValueError, match='its own active_rows'):
        _ops().layer_norm(sparse, weight, bias, active_rows=active)


def test_refusals():
    ops = _ops()
    x, weight, bias, _ = _inputs(4, 8, torch.float32)
    for args, message in (
            ((x[0], weight, bias), r'shape \(N, C\)'),
            ((x.double(), None, None), 'float32, float16 or bfloat16'),
            ((x, weight.half(), bias), 'weight must share a dtype'),
            ((x, weight, bias[:7]), r'bias must have shape \(C,\)'),
            ((x, weight.cpu(), bias), 'HIP device tensor')):
        with pytest.raises(ValueError, match=message):
            ops.layer_norm(*args)
    with pytest.raises(ValueError, match='eps'):
        ops.layer_norm(x, weight, bias, eps=-1.0)
    with pytest.raises(ValueError, match='active_rows'):
        ops.layer_norm(x, active_rows=torch.zeros(2, device='cuda'))


def test_more_channels_than_blocks_of_a_launch():
    """The sums of 2^26 columns and more, 16 a block of 1024 threads."""
    channels = 2 ** 25 + 24
    x, weight, bias, dy = _inputs(2, channels, torch.float16)
    leaves = [t.requires_grad_() for t in (x, weight, bias)]
    y = _ops().layer_norm(*leaves)
    _, dw, db = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        wide = x.double()
        var, mean = torch.var_mean(wide, 1, unbiased=False, keepdim=True)
        normed = (wide - mean) / torch.sqrt(var + 1e-5)
        size = (wide.abs() + wide.abs().mean(1, keepdim=True)) / torch.sqrt(
            var + 1e-5)
        terms = dy.double()
        # As the bounds of layer_norm_f64, of sums of two terms.
        for got, want, most in ((dw, terms * normed, terms.abs() * size),
                                (db, terms, terms.abs())):
            off = (got.double() - want.sum(0)).abs()
            assert (off <= 2.0 ** -11 * want.sum(0).abs()
                    + 2.0 ** -16 * most.sum(0) + 2.0 ** -24).all()
