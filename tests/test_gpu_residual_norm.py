"""The junction of two parts of a block and its gradients against float64."""

from __future__ import annotations

import itertools

import pytest
import torch
from transformer_reference import FLOAT_SUM, TINY, UNIT, assert_within

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)
NAMES = ('weight', 'bias', 'gate', 'post_weight', 'post_bias')


def _ops():
    import mlx_lattice_amd.ops as ops

    return ops


def _inputs(rows, channels, dtype, vectors=NAMES, seed=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device='cuda')

    spread = torch.rand((rows, 1), generator=gen, device='cuda') * 3 + 0.1
    given = {'x': (normal(rows, channels) * spread + 0.3).to(dtype),
             'residual': (normal(rows, channels) - 0.2 * spread).to(dtype)}
    for name in vectors:
        given[name] = (normal(channels) * 0.4
                       + (0.8 if 'weight' in name else 0.1)).to(dtype)
    cotangents = [normal(rows, channels).to(dtype) for _ in range(2)]
    return given, cotangents


def _statistics(z, rms, eps):
    mean = 0.0 if rms else z.mean(1, keepdim=True)
    root = 1 / torch.sqrt(((z - mean) ** 2).mean(1, keepdim=True) + eps)
    # What the mean's own rounding and the difference's reach.
    size = (z.abs() + (0.0 if rms else z.abs().mean(1, keepdim=True))) * root
    return (z - mean) * root, root, size


def _reference(given, total, cotangents, scale, post, rms, eps, active):
    """(value, bound) of every result, float64 on the CPU; ``total`` is the sum
    as it was rounded, which the second norm is of."""
    dtype = given['x'].dtype
    u, tiny = UNIT[dtype], TINY[dtype]
    n, c = given['x'].shape
    live = (torch.arange(n) < (n if active is None else active))[:, None]

    def wide(t):
        return t.detach().cpu().double()

    def rows(t):
        return torch.where(live, wide(t), 0.0)

    x, residual, h = rows(given['x']), rows(given['residual']), rows(total)
    ones, zeros = (torch.full((c,), v, dtype=torch.float64) for v in (1., 0.))
    w, b, gate, pw, pb = (
        wide(given[k]) if k in given else default
        for k, default in zip(NAMES, (ones, zeros, ones, ones, zeros)))
    if post:
        m, post_root, m_size = _statistics(x, rms, eps)
        part, part_size = m * pw + pb, m_size * pw.abs() + pb.abs()
    else:
        part, part_size = x, x.abs()
    f = scale * gate
    want = torch.where(live, residual + f * part, 0.0)
    near = FLOAT_SUM * (residual.abs() + f.abs() * part_size)
    normed, root, size = _statistics(h, rms, eps)
    y = torch.where(live, normed * w + b, 0.0)
    out = {'sum': (want, u * want.abs() + near + tiny),
           'normed': (y, u * y.abs() + FLOAT_SUM * (size * w.abs() + b.abs())
                      + tiny)}
    dh, dy = (torch.zeros_like(h) if t is None else rows(t)
              for t in cotangents)
    g = dy * w

    def back(slope, mag, normed, root, size):
        mean = 0.0 if rms else slope.mean(1, keepdim=True)
        mag_mean = 0.0 if rms else mag.mean(1, keepdim=True)
        value = root * (slope - mean - normed * (slope * normed).mean(
            1, keepdim=True))
        return value, root * (mag + mag_mean + size * (mag * size).mean(
            1, keepdim=True))

    t, t_mag = back(g, g.abs(), normed, root, size)
    t, t_mag = t + dh, t_mag + dh.abs()
    du, du_mag = f * t, f.abs() * t_mag
    values = {'residual': (t, t_mag),
              'weight': ((dy * normed).sum(0), (dy.abs() * size).sum(0)),
              'bias': (dy.sum(0), dy.abs().sum(0)),
              'gate': (scale * (t * part).sum(0),
                       abs(scale) * (t_mag * part_size).sum(0)),
              'x': (du, du_mag)}
    if post:
        values['x'] = back(du * pw, du_mag * pw.abs(), m, post_root, m_size)
        values['post_weight'] = ((du * m).sum(0), (du_mag * m_size).sum(0))
        values['post_bias'] = (du.sum(0), du_mag.sum(0))
    for name, (value, mag) in values.items():
        mask = live if value.ndim == 2 else True
        value = torch.where(torch.as_tensor(mask), value, 0.0)
        out['d_' + name] = (value, u * value.abs() + FLOAT_SUM * mag + tiny)
    return out


def _check(given, cotangents, scale=0.7, post=False, rms=False, eps=1e-5,
           active=None):
    leaves = {k: t.detach().requires_grad_() for k, t in given.items()}
    count = (None if active is None else
             torch.tensor([active], dtype=torch.int32, device='cuda'))
    how = {'scale': scale, 'post_norm': post, 'rms': rms, 'eps': eps,
           'active_rows': count}
    total, normed = _ops().residual_norm(**leaves, **how)
    with torch.no_grad():
        plain = _ops().residual_norm(**given, **how)
    assert torch.equal(plain[0], total) and torch.equal(plain[1], normed)
    used = [(o, t) for o, t in zip((total, normed), cotangents)
            if t is not None]
    grads = torch.autograd.grad([o for o, _ in used], list(leaves.values()),
                                [t for _, t in used])
    got = {'sum': total, 'normed': normed,
           **{'d_' + k: g for k, g in zip(leaves, grads)}}
    want = _reference(given, total, cotangents, scale, post, rms, eps, active)
    for name, value in got.items():
        assert value.dtype == given['x'].dtype
        assert_within(value, *want[name], name)


SHAPES = [(1, 1), (1, 64), (3, 3), (17, 7), (70, 30), (1, 512), (33, 96),
          (300, 128), (65, 257), (129, 513), (10, 1000), (6, 1030), (50, 2048),
          (7, 4100), (5, 6000), (3, 8200), (4, 9001), (9, 20000)]


@pytest.mark.parametrize('rms', (False, True))
@pytest.mark.parametrize('post', (False, True))
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows, channels', SHAPES)
def test_rows(rows, channels, dtype, post, rms):
    names = NAMES if post else NAMES[:3]
    _check(*_inputs(rows, channels, dtype, names), post=post, rms=rms)


@pytest.mark.parametrize('post', (False, True))
@pytest.mark.parametrize('channels', (40, 9000))
def test_any_set_of_vectors(channels, post):
    names = NAMES if post else NAMES[:3]
    for count in range(len(names) + 1):
        for some in itertools.combinations(names, count):
            _check(*_inputs(9, channels, torch.float32, some), post=post,
                   scale=-1.5)


@pytest.mark.parametrize('post', (False, True))
@pytest.mark.parametrize('channels', (64, 700, 9000))
def test_one_cotangent(channels, post):
    names = NAMES if post else NAMES[:3]
    given, (dh, dy) = _inputs(20, channels, torch.float32, names)
    _check(given, (dh, torch.zeros_like(dy)), post=post)
    leaves = {k: t.requires_grad_() for k, t in given.items()}
    total, normed = _ops().residual_norm(**leaves, scale=0.7, post_norm=post)
    want = _reference(given, total, (dh, None), 0.7, post, False, 1e-5, None)
    wants = _reference(given, total, (None, dy), 0.7, post, False, 1e-5, None)
    for out, slope, refs in ((total, dh, want), (normed, dy, wants)):
        grads = torch.autograd.grad(out, list(leaves.values()), slope,
                                    retain_graph=True)
        for name, grad in zip(leaves, grads):
            assert_within(grad, *refs['d_' + name], name)


@pytest.mark.parametrize('rms', (False, True))
@pytest.mark.parametrize('channels', (48, 9000))
@pytest.mark.parametrize('active', (0, 1, 13, 40, 99, -5))
def test_inactive_rows_are_zero_and_take_no_part(active, channels, rms):
    given, cotangents = _inputs(40, channels, torch.float32)
    for t in (given['x'], given['residual'], *cotangents):
        t[max(0, active):] = float('nan')
    _check(given, cotangents, post=True, rms=rms,
           active=min(40, max(0, active)))


def test_no_rows():
    for dtype in DTYPES:
        given, cotangents = _inputs(0, 40, dtype)
        leaves = {k: t.requires_grad_() for k, t in given.items()}
        out = _ops().residual_norm(**leaves, post_norm=True)
        assert out[0].shape == out[1].shape == (0, 40)
        grads = torch.autograd.grad(out, list(leaves.values()), cotangents)
        for leaf, grad in zip(leaves.values(), grads):
            assert grad.shape == leaf.shape and not grad.any()


@pytest.mark.parametrize('dtype', DTYPES)
def test_strided_and_misaligned_rows(dtype):
    given, cotangents = _inputs(50, 64, dtype)
    packed = torch.zeros((50, 200), device='cuda', dtype=dtype)
    for at, gap in ((0, 64), (1, 67), (2, 66), (8, 80)):
        moved = dict(given)
        moved['x'] = packed[:, at:at + 64].copy_(given['x'])
        moved['residual'] = packed[:, at + gap:at + gap + 64].copy_(
            given['residual'])
        _check(moved, cotangents, post=True)
    moved = dict(given)
    moved['x'] = given['x'].T.contiguous().T
    moved['residual'] = given['residual'][:1].expand(50, 64)
    moved['weight'] = torch.stack([given['weight']] * 2, 1)[:, 0]
    moved['gate'] = given['gate'][:1].expand(64)
    _check(moved, [cotangents[0].T.contiguous().T,
                   cotangents[1][:1].expand(50, 64)], post=True)


def test_same_tensor_twice():
    """One tensor as both inputs gets both gradients."""
    given, cotangents = _inputs(30, 96, torch.float32, NAMES[:3])
    x = given.pop('x').requires_grad_()
    given.pop('residual')
    out = _ops().residual_norm(x, x, **given)
    both = torch.autograd.grad(out, x, cotangents)[0]
    a, b = x.detach().requires_grad_(), x.detach().requires_grad_()
    each = torch.autograd.grad(_ops().residual_norm(a, b, **given), (a, b),
                               cotangents)
    assert torch.equal(both, each[0] + each[1])


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('channels', (30, 64, 128, 200, 512))
def test_as_an_addition_and_a_norm(channels, dtype):
    """The sum bit for bit.  The norms' float32 values may differ in their
    last bits (orders of sums, one rounding or two for a value less the mean),
    each within the float32 bound; where such values lie on either side of a
    border of the type, they are one step, two units of rounding, apart."""
    given, _ = _inputs(333, channels, dtype, NAMES[:2])
    total, normed = _ops().residual_norm(**given)
    assert torch.equal(total, given['residual'] + given['x'])
    apart = _ops().layer_norm(total, given['weight'], given['bias'])
    h = total.double()
    _, _, size = _statistics(h, False, 1e-5)
    bound = 2 * FLOAT_SUM * (size * given['weight'].double().abs()
                             + given['bias'].double().abs())
    bound = bound + 2 * UNIT[dtype] * apart.double().abs() + TINY[dtype]
    assert_within(normed, apart.double(), bound)


def test_large_mean_does_not_cancel():
    given, cotangents = _inputs(40, 256, torch.float32)
    given['residual'] += 3000.0
    given['x'] += 500.0
    _check(given, cotangents, post=True)


def test_constant_rows_and_eps():
    given, cotangents = _inputs(8, 64, torch.float32)
    given['x'][:] = 2.0
    given['residual'][:4] = 1.0
    _check(given, cotangents, post=True, eps=1e-3)
    for t in (given['x'], given['residual']):
        t.zero_()
    _check(given, cotangents, post=True, rms=True, eps=1e-2)


def test_infinities_and_nan_stay_in_their_rows():
    given, _ = _inputs(20, 64, torch.float16, NAMES[:3])
    clean = _ops().residual_norm(**given)
    given['x'][3, 5] = float('inf')
    given['residual'][9, 60] = float('nan')
    spoilt = _ops().residual_norm(**given)
    keep = torch.ones(20, dtype=torch.bool)
    keep[[3, 9]] = False
    for a, b in zip(clean, spoilt):
        assert torch.equal(a[keep], b[keep])
    assert torch.isnan(spoilt[1][[3, 9]]).all()


@pytest.mark.parametrize('post, rms', ((False, False), (True, False),
                                       (True, True)))
@pytest.mark.parametrize('channels', (40, 700))
def test_gradient_against_differences(channels, post, rms):
    given, cotangents = _inputs(12, channels, torch.float32,
                                NAMES if post else NAMES[:3])
    how = {'post_norm': post, 'rms': rms, 'scale': 0.7}
    leaves = {k: t.requires_grad_() for k, t in given.items()}
    grads = torch.autograd.grad(_ops().residual_norm(**leaves, **how),
                                list(leaves.values()), cotangents)
    for (name, leaf), grad in zip(leaves.items(), grads):
        way = torch.randn_like(leaf)
        way = way / way.norm()
        ends = []
        for step in (0.02, -0.02):
            moved = {k: t.detach() for k, t in leaves.items()}
            moved[name] = moved[name] + step * way
            ends.append(sum((o.double() * t).sum() for o, t in zip(
                _ops().residual_norm(**moved, **how), cotangents)))
        slope = float((ends[0] - ends[1]) / 0.04)
        # Central differences of step 0.02 leave a third-order term of about
        # 0.02^2 of the slope's size; the float32 forward's roundings of 2^-24
        # over 0.04 are smaller.
        size = float(grad.norm())
        assert abs(slope - float((grad.double() * way).sum())) < 5e-3 * size


def test_same_result_each_time():
    given, cotangents = _inputs(70001, 64, torch.bfloat16)
    leaves = {k: t.requires_grad_() for k, t in given.items()}
    runs = [torch.autograd.grad(
        _ops().residual_norm(**leaves, post_norm=True),
        list(leaves.values()), cotangents) for _ in range(2)]
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize('rows, channels, dtype', [
    (300000, 8, torch.float16), (40000, 128, torch.bfloat16),
    (20011, 300, torch.float32), (5003, 1500, torch.float16)])
def test_many_rows(rows, channels, dtype):
    """More rows than the blocks of a launch."""
    _check(*_inputs(rows, channels, dtype), post=True)


def test_sparse_tensors():
    from mlx_lattice_amd import SparseTensor

    given, cotangents = _inputs(20, 16, torch.float32, NAMES[:3])
    coords = torch.zeros((20, 4), dtype=torch.int32, device='cuda')
    coords[:, 1] = torch.arange(20)
    active = torch.tensor([15], dtype=torch.int32, device='cuda')
    x = SparseTensor(coords, given.pop('x'), active_rows=active)
    residual = x.replace(feats=given.pop('residual'))
    out = _ops().residual_norm(x, residual, **given)
    want = _ops().residual_norm(x.feats, residual.feats, **given,
                                active_rows=active)
    for a, b in zip(out, want):
        assert a.same_coords(x) and torch.equal(a.feats, b)
        assert not a.feats[15:].any()
    with pytest.raises(ValueError, match='own active_rows'):
        _ops().residual_norm(x, residual, active_rows=active)
    with pytest.raises(ValueError, match='sparse residual'):
        _ops().residual_norm(x, residual.feats)
    with pytest.raises(ValueError, match='sparse residual'):
        _ops().residual_norm(x.feats, residual)
    other = SparseTensor(coords.clone(), residual.feats)
    with pytest.raises(ValueError, match='coordinates must match'):
        _ops().residual_norm(x, other)


@pytest.mark.parametrize('channels', (64, 1000, 9000))
def test_captured_graph_replays(channels):
    """Forward and gradients in a captured graph whose inputs change."""
    from mlx_lattice_amd._native import ext

    given, (dh, dy) = _inputs(700, channels, torch.float16)
    vectors = [given[n] for n in NAMES]

    def passes():
        total, normed, stats = ext.residual_norm(
            given['x'], given['residual'], vectors, 0.5, True, False, 1e-5,
            None, True)
        return [total, normed, *ext.residual_norm_grad(
            dh, dy, total, stats, given['x'], given['residual'], vectors, 0.5,
            True, False, 1e-5, None, [True] * 5)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = passes()
    for seed in range(3):
        fresh, slopes = _inputs(700, channels, torch.float16, seed=seed + 5)
        for name, t in given.items():
            t.copy_(fresh[name])
        dh.copy_(slopes[0])
        dy.copy_(slopes[1])
        want = passes()
        graph.replay()
        torch.cuda.synchronize()
        for got, eager in zip(captured, want):
            assert torch.equal(got, eager)


@pytest.mark.parametrize('channels', (96, 2048))
def test_captured_training_step(channels):
    """A differentiated call in a captured graph, each pass with leaves of its
    own over the same memory."""
    given, cotangents = _inputs(300, channels, torch.bfloat16)

    def step():
        leaves = {k: t.detach().requires_grad_() for k, t in given.items()}
        out = _ops().residual_norm(**leaves, scale=0.5, post_norm=True)
        return [*(t.detach() for t in out), *torch.autograd.grad(
            out, list(leaves.values()), cotangents)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        fresh, slopes = _inputs(300, channels, torch.bfloat16, seed=seed + 9)
        for name, t in given.items():
            t.data.copy_(fresh[name])
        for t, new in zip(cotangents, slopes):
            t.copy_(new)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for got, eager in zip(captured, want):
            assert torch.equal(got, eager)


def test_only_the_gradients_asked_for():
    given, cotangents = _inputs(20, 32, torch.float32)
    for names in itertools.chain(itertools.combinations(given, 1),
                                 itertools.combinations(given, 2)):
        leaves = {k: t.detach().requires_grad_(k in names)
                  for k, t in given.items()}
        out = _ops().residual_norm(**leaves, post_norm=True)
        asked = [leaves[n] for n in names]
        some = torch.autograd.grad(out, asked, cotangents)
        every = {k: t.detach().requires_grad_() for k, t in given.items()}
        out = _ops().residual_norm(**every, post_norm=True)
        all_of = dict(zip(every, torch.autograd.grad(
            out, list(every.values()), cotangents)))
        for name, grad in zip(names, some):
            assert torch.equal(grad, all_of[name])


def test_differentiated_once():
    given, (dh, _) = _inputs(9, 32, torch.float32)
    x = given.pop('x').requires_grad_()
    total, _ = _ops().residual_norm(x, **given, post_norm=True)
    grad = torch.autograd.grad(total, x, dh, create_graph=True)[0]
    with pytest.raises(RuntimeError, match='differentiated once'):
        grad.sum().backward()


def test_refusals():
    ops = _ops()
    x = torch.zeros((6, 8), device='cuda')

    def refused(message, *args, error=ValueError, **more):
        with pytest.raises(error, match=message):
            ops.residual_norm(*args, **more)

    refused('shape', x[0], x[0])
    refused('shape', x[:, :0], x[:, :0])
    refused('match the shape', x, x[:5])
    refused('share a dtype', x, x.half())
    refused('float32, float16 or bfloat16', x.double(), x.double())
    refused('HIP device tensor', x, x.cpu())
    refused('shape \\(C,\\)', x, x, x[0, :7])
    refused('share a dtype', x, x, gate=x[0].half())
    refused('need post_norm', x, x, post_weight=x[0])
    refused('non-negative', x, x, eps=-1.0)
    refused('non-negative', x, x, eps=float('nan'))
    refused('active_rows', x, x, active_rows=torch.zeros(
        1, dtype=torch.int64, device='cuda'))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        refused('forward-mode', dual, x, error=RuntimeError)


@pytest.mark.parametrize('channels', (48, 9000))
@pytest.mark.parametrize('rms', (False, True))
def test_what_no_gradient_reads_may_change(rms, channels):
    """The residual and the bias are not read by the backward pass, nor is x
    without the first norm and a gradient of the gate, or the first norm's bias
    without the latter: changing them in place between the passes is fine."""
    for post in (False, True):
        given, cotangents = _inputs(40, channels, torch.float32)
        if not post:
            del given['post_weight'], given['post_bias']
        for wanted, changed in (
                ([n for n in given if n != 'gate'],
                 ['residual', 'bias'] + (['post_bias'] if post else ['x'])),
                (list(given), ['residual', 'bias'])):
            grads = []
            for change in (False, True):
                # Leaves are multiplied first, so that what the call takes may
                # be changed.
                leaves = {k: t.detach().clone().requires_grad_(k in wanted)
                          for k, t in given.items()}
                inputs = {k: t * 1 for k, t in leaves.items()}
                out = _ops().residual_norm(**inputs, scale=0.5, rms=rms,
                                           post_norm=post)
                if change:
                    with torch.no_grad():
                        for name in changed:
                            inputs[name].add_(100.0)
                grads.append(torch.autograd.grad(
                    out, [leaves[n] for n in wanted], cotangents))
            for a, b in zip(*grads):
                assert torch.equal(a, b)


def test_what_a_gradient_reads_may_not_change():
    given, cotangents = _inputs(40, 48, torch.float32)
    for name in ('x', 'weight', 'gate', 'post_weight', 'post_bias'):
        leaves = {k: t.detach().clone().requires_grad_()
                  for k, t in given.items()}
        inputs = {k: t * 1 for k, t in leaves.items()}
        out = _ops().residual_norm(**inputs, post_norm=True)
        with torch.no_grad():
            inputs[name].add_(100.0)
        with pytest.raises(RuntimeError, match='modified by an inplace'):
            torch.autograd.grad(out, list(leaves.values()), cotangents)


def test_gradient_without_x():
    from mlx_lattice_amd._native import ext

    given, (dh, dy) = _inputs(30, 40, torch.float16)
    vectors = [given['weight'], None, given['gate'], None, None]
    total, _, stats = ext.residual_norm(
        given['x'], given['residual'], vectors, 0.5, False, False, 1e-5, None,
        True)

    def grad(x, wanted, post=False):
        return ext.residual_norm_grad(dh, dy, total, stats, x, None, vectors,
                                      0.5, post, False, 1e-5, None, wanted)

    some = [True, True, False, False, False]
    for a, b in zip(grad(None, some), grad(given['x'], some)):
        assert a is None and b is None or torch.equal(a, b)
    for wanted, post in (([True] * 3 + [False] * 2, False), (some, True)):
        with pytest.raises(ValueError, match='x is needed'):
            grad(None, wanted, post)
