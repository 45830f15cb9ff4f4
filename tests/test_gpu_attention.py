"""Windowed attention and its gradients against float64."""

from __future__ import annotations

import pytest
import torch
from transformer_reference import assert_within, attention_f64

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _ops():
    import mlx_lattice_amd.ops as ops

    return ops


def _offsets(lengths, start=0):
    out = [start]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device='cuda')


def _normal(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device='cuda').to(dtype)


def _run(q, k, v, dy, **kwargs):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = _ops().window_attention(*leaves, **kwargs)
    with torch.no_grad():
        plain = _ops().window_attention(q, k, v, **kwargs)
    assert torch.equal(plain.nan_to_num(7.0), out.nan_to_num(7.0))
    return [out, *torch.autograd.grad(out, leaves, dy)]


def _check(q, k, v, dy, spans, left, right, sinks, scale=None, device='cpu',
           **kwargs):
    got = _run(q, k, v, dy, left=left, right=right, sinks=sinks, scale=scale,
               **kwargs)
    want = attention_f64(q, k, v, spans, left, right, sinks,
                         scale or q.shape[-1] ** -0.5, dy, device)
    for name, value, like, (ref, bound) in zip(('out', 'dq', 'dk', 'dv'), got,
                                               (q, q, k, v), want):
        assert value.dtype == like.dtype and value.shape == like.shape
        assert_within(value, ref, bound, name)


def _self(lengths, heads, kv_heads, dim, dtype, left, right, sinks, seed=0,
          device='cpu'):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    rows = sum(lengths)
    qkv = _normal(gen, dtype, rows, heads + 2 * kv_heads, dim)
    spans, at = [], 0
    for n in lengths:
        spans.append((at, n, at, n))
        at += n
    _check(qkv[:, :heads], qkv[:, heads:heads + kv_heads],
           qkv[:, heads + kv_heads:], _normal(gen, dtype, rows, heads, dim),
           spans, left, right, sinks, offsets=_offsets(lengths),
           device=device)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('lengths, heads, kv_heads, dim, left, right, sinks', [
    ((1,), 1, 1, 8, None, None, 0),
    ((1,), 4, 2, 64, 0, 0, 1),
    ((2, 0, 1), 2, 1, 32, None, 0, 0),
    ((63,), 2, 2, 32, 5, 3, 2),
    ((64, 65), 4, 1, 64, 16, 0, 4),
    ((300,), 3, 3, 32, 128, 128, 4),
    ((129, 1, 0, 200), 4, 4, 24, 40, 7, 3),
    ((257,), 8, 2, 128, None, 0, 0),
    ((190, 70), 2, 2, 128, None, None, 0),
    ((333,), 6, 2, 80, 50, 0, 16),
    ((401,), 1, 1, 64, 0, 0, 0),
    ((150,), 2, 1, 16, 0, 5, 300),
    ((500,), 2, 1, 96, 30, 30, 70),
    ((40,) * 9, 2, 2, 40, 9, 2, 1)])
def test_packed_sequences(lengths, heads, kv_heads, dim, left, right, sinks,
                          dtype):
    _self(lengths, heads, kv_heads, dim, dtype, left, right, sinks)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', (1, 2, 7, 33, 36, 100, 127))
def test_any_number_of_channels(dim, dtype):
    _self((50, 21), 2, 1, dim, dtype, 12, 4, 2)


@pytest.mark.parametrize('dtype', DTYPES)
def test_many_short_sequences(dtype):
    _self(tuple(i % 4 for i in range(700)), 2, 1, 32, dtype, 2, 1, 1)


# Rows enough for tiles of 128, 32768 rows of key heads and more; the first
# keys' long sums in a pass of their own (long sequences) and without.
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('lengths, heads, kv_heads, dim, left, right, sinks', [
    ((3000, 2501, 3100), 8, 4, 64, 90, 40, 5),
    ((1500, 0, 700, 1, 411) + (61,) * 110, 8, 4, 32, 70, 9, 3),
    ((4100, 4200), 12, 4, 80, 130, 0, 37),
    ((3400, 33, 5000), 4, 4, 128, 33, 64, 1),
    ((2900, 2800, 2700), 4, 4, 24, 10, 200, 150),
    ((5600,), 6, 6, 96, 300, 0, 0)])
def test_many_rows(lengths, heads, kv_heads, dim, left, right, sinks, dtype):
    _self(lengths, heads, kv_heads, dim, dtype, left, right, sinks,
          device='cuda')


# Few rows that see thousands of keys: tiles of 128 whose keys are split.
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('lengths, heads, kv_heads, dim, left, right, sinks', [
    ((2600,), 2, 1, 64, None, 0, 0), ((3001,), 2, 2, 32, 2500, 100, 7),
    ((2500, 70), 2, 1, 128, None, None, 0), ((2300,), 1, 1, 96, 2290, 0, 1)])
def test_split_keys(lengths, heads, kv_heads, dim, left, right, sinks, dtype):
    _self(lengths, heads, kv_heads, dim, dtype, left, right, sinks,
          device='cuda')


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('value', (float('nan'), float('inf')))
def test_what_is_not_seen_never_arrives_in_large_tiles(value, dtype):
    """A row of k, v, q or the cotangent that is not finite, in tiles of 128:
    rows past two windows of it neither see it nor share a sum with one that
    does.  Those that share a tile with it are made again by themselves and
    differ in rounding; rows some tiles away are those of the clean call."""
    gen = torch.Generator(device='cuda').manual_seed(13)
    kwargs = {'left': 40, 'right': 3, 'sinks': 0, 'offsets': _offsets((9000,))}
    place = torch.arange(9000, device='cuda')
    past = (place - 4321).abs() > 86
    far = (place - 4321).abs() > 86 + 4 * 128
    for name in ('k', 'v', 'dy', 'q'):
        t = {n: _normal(gen, dtype, 9000, 4, 32) for n in ('q', 'k', 'v', 'dy')}
        clean = _run(t['q'], t['k'], t['v'], t['dy'], **kwargs)
        want = attention_f64(t['q'], t['k'], t['v'], [(0, 9000, 0, 9000)], 40,
                             3, 0, 32 ** -0.5, t['dy'], 'cuda')
        t[name][4321] = value
        got = _run(t['q'], t['k'], t['v'], t['dy'], **kwargs)
        for a, b, (ref, bound) in zip(got, clean, want):
            assert torch.equal(a[far], b[far])
            assert_within(a[past], ref[past], bound[past], name)
        assert not torch.isfinite(got[1][4310:4340]).all()


def _cache(q_lengths, k_lengths, capacity, heads, kv_heads, dim, dtype, left,
           right, sinks, seed=1):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    count = len(q_lengths)
    q = _normal(gen, dtype, sum(q_lengths), heads, dim)
    k, v = (_normal(gen, dtype, count * capacity, kv_heads, dim)
            for _ in range(2))
    spans, at = [], 0
    for s, (nq, nk) in enumerate(zip(q_lengths, k_lengths)):
        spans.append((at, nq, s * capacity, nk))
        # What is past a sequence's keys is never read into a result.
        k[s * capacity + nk:(s + 1) * capacity] = float('nan')
        v[s * capacity + nk:(s + 1) * capacity] = float('inf')
        at += nq
    _check(q, k, v, _normal(gen, dtype, at, heads, dim), spans, left, right,
           sinks, offsets=_offsets(q_lengths),
           key_offsets=torch.arange(count + 1, dtype=torch.int32,
                                    device='cuda') * capacity,
           key_lengths=torch.tensor(k_lengths, dtype=torch.int32,
                                    device='cuda'))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize(
    'q_lengths, k_lengths, capacity, heads, kv_heads, dim, left, sinks', [
        ((1,), (1,), 1, 4, 4, 64, None, 0),
        ((1, 1, 1), (5, 0, 130), 130, 8, 2, 64, None, 0),
        ((1, 1), (700, 513), 800, 8, 1, 128, 64, 4),
        ((1, 1), (3000, 1999), 3000, 4, 1, 32, None, 0),
        ((3, 1, 0, 2), (64, 65, 7, 1), 70, 4, 2, 24, 40, 2),
        ((130, 20), (1500, 20), 1600, 2, 1, 64, 600, 8),
        ((5,), (2, ), 9, 2, 1, 80, None, 1),
        ((17, 17), (900, 333), 1000, 16, 1, 128, None, 0)])
def test_cache(q_lengths, k_lengths, capacity, heads, kv_heads, dim, left,
               sinks, dtype):
    _cache(q_lengths, k_lengths, capacity, heads, kv_heads, dim, dtype, left,
           0, sinks)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('left, right, sinks', ((3, 0, 0), (0, 2, 2),
                                                (None, 0, 0)))
def test_queries_before_the_keys_see_nothing(left, right, sinks, dtype):
    _cache((200, 40, 3), (30, 0, 2), 30, 2, 1, 32, dtype, left, right, sinks)


@pytest.mark.parametrize('dtype', DTYPES)
def test_rows_in_no_sequence(dtype):
    gen = torch.Generator(device='cuda').manual_seed(2)
    q, dy = (_normal(gen, dtype, 100, 2, 32) for _ in range(2))
    k, v = (_normal(gen, dtype, 150, 2, 32) for _ in range(2))
    k[:20], v[120:] = float('nan'), float('inf')
    q[:7], dy[60:] = float('nan'), float('inf')
    _check(q, k, v, dy, [(7, 30, 20, 40), (37, 23, 60, 60)], 12, 4, 2,
           offsets=torch.tensor([7, 37, 60], dtype=torch.int32, device='cuda'),
           key_offsets=torch.tensor([20, 60, 120], dtype=torch.int32,
                                    device='cuda'))


@pytest.mark.parametrize('dtype', DTYPES)
def test_no_rows_or_sequences(dtype):
    gen = torch.Generator(device='cuda').manual_seed(2)
    q = _normal(gen, dtype, 6, 2, 32)
    k = _normal(gen, dtype, 9, 1, 32)
    none = _offsets(())
    for a, b in ((q, k), (q[:0], k), (q, k[:0]), (q[:0], k[:0])):
        got = _run(a, b, b, a, offsets=none)
        for value, like in zip(got, (a, a, b, b)):
            assert value.shape == like.shape and not value.any()


@pytest.mark.parametrize('dtype', DTYPES)
def test_layouts(dtype):
    """Packed rows, head-major storage, odd places, heads shared by stride."""
    gen = torch.Generator(device='cuda').manual_seed(3)
    spans = [(0, 70, 0, 70)]
    kwargs = {'offsets': _offsets((70,))}
    q, dy = (_normal(gen, dtype, 4, 70, 32).transpose(0, 1) for _ in range(2))
    kv = _normal(gen, dtype, 70, 2, 2, 40)
    k, v = kv[:, 0, :, 8:], kv[:, 1, :, :32]
    _check(q, k, v, dy, spans, 20, 0, 1, **kwargs)
    _check(q[..., :24], k[..., 8:], kv[:, 1, :, 3:27], dy[..., 1:25], spans,
           20, 0, 1, **kwargs)
    one = kv[:, 0, :1, :32].expand(70, 2, 32)
    _check(q, one, one, dy, spans, 20, 3, 0, **kwargs)
    flat = _normal(gen, dtype, 70 * 4 * 32 + 1)[1:].view(70, 4, 32)
    _check(flat, k, v, dy, spans, None, 0, 0, scale=0.3, **kwargs)


@pytest.mark.parametrize('dtype', DTYPES)
def test_large_scores(dtype):
    """Scores of hundreds: the running maximum carries them."""
    gen = torch.Generator(device='cuda').manual_seed(4)
    q, k, v, dy = (_normal(gen, dtype, 200, 2, 64) for _ in range(4))
    _check(q * 4, k * 4, v, dy, [(0, 200, 0, 200)], 90, 0, 4,
           offsets=_offsets((200,)))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('value', (float('nan'), float('inf')))
def test_what_is_not_seen_never_arrives(value, dtype):
    """Rows of q, k, v and the cotangent that are not finite reach those that
    see them and no others."""
    gen = torch.Generator(device='cuda').manual_seed(5)
    spans = [(0, 150, 0, 150)]
    for name in ('k', 'v', 'dy', 'q'):
        t = {n: _normal(gen, dtype, 150, 2, 32) for n in 'qkv'}
        t['dy'] = _normal(gen, dtype, 150, 2, 32)
        t[name][40] = value
        t[name][97, 1, 5] = value
        got = _run(t['q'], t['k'], t['v'], t['dy'], left=10, right=2, sinks=2,
                   offsets=_offsets((150,)))
        clean = {n: x.nan_to_num(0.0, 0.0, 0.0) for n, x in t.items()}
        want = attention_f64(clean['q'], clean['k'], clean['v'], spans, 10, 2,
                             2, 32 ** -0.5, clean['dy'])
        i = torch.arange(150)
        seen = (i[None] <= i[:, None] + 2) & (
            (i[None] >= i[:, None] - 10) | (i[None] < 2))
        for head, bad in ((0, (40,)), (1, (40, 97))):
            mark = torch.zeros(150, dtype=torch.bool)
            mark[list(bad)] = True
            # A row of k or v spoils the queries that see it and, through
            # their sums, the keys that those see; one of q or the cotangent
            # its own query and the keys that it sees.
            rows = (seen & mark).any(1) if name in 'kv' else mark
            keys = (seen.T & rows).any(1)
            spoilt = {'out': rows if name != 'dy' else mark & False,
                      'dq': rows, 'dk': keys, 'dv': keys}
            for at, (what, (ref, bound)) in enumerate(zip(spoilt, want)):
                clear = ~spoilt[what]
                assert_within(got[at][:, head][clear.cuda()],
                              ref[:, head][clear], bound[:, head][clear],
                              f'{name} {what}')
        if name in 'kv':
            assert not torch.isfinite(got[0][40:51]).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows, start', ((200, 100), (9000, 4100)))
def test_scores_of_minus_infinity(rows, start, dtype):
    """Keys whose scores are -inf have no share, also in rows that are made
    again since a key that they do not see is not finite: such a row starts
    with 64 and more of the former."""
    gen = torch.Generator(device='cuda').manual_seed(17)
    q, k, v = (_normal(gen, dtype, rows, 4, 32) for _ in 'qkv')
    q[..., 0] = q[..., 0].abs() + 0.5
    k[max(0, start - 200):start, :, 0] = float('-inf')
    k[start + 80] = float('nan')
    v[start + 80] = float('nan')
    got = _ops().window_attention(q, k, v, left=170, right=0,
                                  offsets=_offsets((rows,)))
    at = slice(start, start + 80)
    want, bound = attention_f64(q[at], k[at], v[at], [(0, 80, 0, 80)], 170, 0,
                                0, 32 ** -0.5)[0]
    assert_within(got[at], want, bound)


def test_gradient_against_differences():
    gen = torch.Generator(device='cuda').manual_seed(6)
    leaves = [_normal(gen, torch.float32, 60, h, 16).requires_grad_()
              for h in (4, 2, 2)]
    dy = _normal(gen, torch.float32, 60, 4, 16)
    kwargs = {'left': 13, 'right': 4, 'sinks': 3, 'offsets': _offsets((21, 39))}
    grads = torch.autograd.grad(_ops().window_attention(*leaves, **kwargs),
                                leaves, dy)
    for i, grad in enumerate(grads):
        way = _normal(gen, torch.float32, *leaves[i].shape)
        way = way / way.norm()
        ends = []
        for step in (0.02, -0.02):
            moved = [t.detach() for t in leaves]
            moved[i] = moved[i] + step * way
            ends.append((_ops().window_attention(*moved, **kwargs).double()
                         * dy).sum())
        slope = float((ends[0] - ends[1]) / 0.04)
        # A third-order term of about 0.02^2 of the slope's size.
        assert abs(slope - float((grad.double() * way).sum())) < 5e-3 * float(
            grad.norm())


@pytest.mark.parametrize('dtype', DTYPES)
def test_same_result_each_time(dtype):
    gen = torch.Generator(device='cuda').manual_seed(7)
    q, k, v, dy = (_normal(gen, dtype, 3000, h, 64) for h in (4, 1, 1, 4))
    runs = [_run(q, k, v, dy, left=200, right=50, sinks=4,
                 offsets=_offsets((1000, 2000))) for _ in range(2)]
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_cache_past_32_bits():
    """Keys whose place passes 2^31 elements and 2^32 bytes."""
    rows, dim = 17_000_000, 128
    k = torch.zeros((rows, 1, dim), dtype=torch.bfloat16, device='cuda')
    v = torch.zeros_like(k)
    gen = torch.Generator(device='cuda').manual_seed(8)
    k[-500:], v[-500:] = (_normal(gen, torch.bfloat16, 500, 1, dim)
                          for _ in range(2))
    q = _normal(gen, torch.bfloat16, 3, 4, dim)
    for nq in (1, 3):
        got = _ops().window_attention(
            q[:nq], k, v, left=300, right=0,
            offsets=_offsets((0, nq)), key_offsets=torch.tensor(
                [0, rows - 500, rows], dtype=torch.int32, device='cuda'))
        ref, bound = attention_f64(q[:nq], k[-500:], v[-500:],
                                   [(0, nq, 0, 500)], 300, 0, 0,
                                   dim ** -0.5)[0]
        assert_within(got, ref, bound)
        # One sequence from row 0: the window alone is read.
        got = _ops().window_attention(q[:nq], k, v, left=300, right=0, sinks=1,
                                      offsets=_offsets((nq,)),
                                      key_offsets=_offsets((rows,)))
        tail_k, tail_v = (torch.cat([t[:1], t[-500:]]) for t in (k, v))
        ref, bound = attention_f64(q[:nq], tail_k, tail_v, [(0, nq, 0, 501)],
                                   300, 0, 1, dim ** -0.5)[0]
        assert_within(got, ref, bound)


@pytest.mark.parametrize('dim', (32, 128))
def test_rows_and_heads_far_apart(dim):
    """Query heads and rows that no tile's 32-bit places reach."""
    gen = torch.Generator(device='cuda').manual_seed(11)
    store = torch.zeros(5 << 28, dtype=torch.float16, device='cuda')
    q = store.as_strided((70, 4, dim), (dim, 1 << 28, 1))
    k = store[1 << 20:].as_strided((70, 2, dim), (1 << 23, dim, 1))
    for t in (q, k):
        t.copy_(_normal(gen, torch.float16, *t.shape))
    v = _normal(gen, torch.float16, 70, 2, dim)
    dy = _normal(gen, torch.float16, 70, 4, dim)
    _check(q, k, v, dy, [(0, 70, 0, 70)], 20, 3, 2, offsets=_offsets((70,)))


@pytest.mark.parametrize('dtype, dim', ((torch.float32, 128),
                                        (torch.float16, 128),
                                        (torch.bfloat16, 32)))
def test_captured_graph_replays(dtype, dim):
    """Forward and gradients, few queries and many, in a captured graph whose
    inputs change between replays."""
    from mlx_lattice_amd._native import ext

    gen = torch.Generator(device='cuda').manual_seed(12)
    q, dy = (torch.zeros((700, 4, dim), dtype=dtype, device='cuda')
             for _ in range(2))
    k, v = (torch.zeros((700, 2, dim), dtype=dtype, device='cuda')
            for _ in range(2))
    at, token = _offsets((300, 400)), _offsets((1, 1))
    window = (60, 10, 2, dim ** -0.5)

    def passes():
        out, lse, rest = ext.window_attention(q, k, v, at, at, None, *window,
                                              True)
        grads = ext.window_attention_grad(dy, out, lse, rest, q, k, v, at, at,
                                          None, *window)
        few = _ops().window_attention(q[:2], k, v, offsets=token,
                                      key_offsets=at)
        return [out, *grads, few]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = passes()
    for _ in range(3):
        for t in (q, k, v, dy):
            t.copy_(_normal(gen, dtype, *t.shape))
        want = passes()
        graph.replay()
        torch.cuda.synchronize()
        for got, eager in zip(captured, want):
            assert torch.equal(got, eager)


def test_other_stream():
    gen = torch.Generator(device='cuda').manual_seed(9)
    q, k, v, dy = (_normal(gen, torch.float16, 500, h, 32)
                   for h in (4, 2, 2, 4))
    kwargs = {'left': 50, 'right': 0, 'sinks': 1, 'offsets': _offsets((500,))}
    want = _run(q, k, v, dy, **kwargs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, dy, **kwargs)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_offsets_out_of_range_are_clamped():
    gen = torch.Generator(device='cuda').manual_seed(10)
    q, k, v = (_normal(gen, torch.float32, 64, 2, 32) for _ in range(3))
    offsets = torch.tensor([-5, 30, 1000], dtype=torch.int32, device='cuda')
    got = _ops().window_attention(q, k, v, left=9, right=0, offsets=offsets)
    want = _ops().window_attention(q, k, v, left=9, right=0,
                                   offsets=_offsets((30, 34)))
    assert torch.equal(got, want)


def test_batch_offsets():
    from mlx_lattice_amd import SparseTensor

    ops = _ops()
    coords = torch.zeros((10, 4), dtype=torch.int32, device='cuda')
    coords[:, 1] = torch.arange(10)
    feats = torch.zeros((10, 2), device='cuda')
    x = SparseTensor(coords, feats, batch_counts=(3, 0, 7))
    assert ops.batch_offsets(x).tolist() == [0, 3, 3, 10]
    active = torch.tensor([6], dtype=torch.int32, device='cuda')
    x = SparseTensor(coords, feats, active_rows=active)
    assert ops.batch_offsets(x).tolist() == [0, 6]
    assert ops.batch_offsets(x).dtype == torch.int32


def test_refusals():
    ops = _ops()
    q = torch.zeros((6, 4, 32), device='cuda')
    k = torch.zeros((6, 2, 32), device='cuda')
    at = _offsets((6,))

    def refused(message, *args, **kwargs):
        kwargs = {'offsets': at, **kwargs}
        with pytest.raises(ValueError, match=message):
            ops.window_attention(*args, **kwargs)

    refused(r'shape \(N, heads, dim\)', q[0], k, k)
    refused('k and v must have the same shape', q, k, k[:5])
    refused('share the channels', q, k[..., :16], k[..., :16])
    refused('multiple of the number', q[:, :3], k, k)
    refused('between 1 and 128', *(torch.zeros((6, 2, 136), device='cuda'),) * 3)
    refused('share a dtype', q, k.half(), k)
    refused('float32, float16 or bfloat16', q.double(), k.double(), k.double())
    refused('non-negative', q, k, k, left=-1)
    refused('non-negative', q, k, k, right=-1)
    refused('non-negative', q, k, k, sinks=-1)
    refused('offsets must have shape', q, k, k, offsets=at.long())
    refused('key_offsets must have', q, k, k, key_offsets=_offsets((3, 3)))
    refused('key_lengths must have', q, k, k, key_lengths=at)
    refused('HIP device tensor', q.cpu(), k.cpu(), k.cpu())
    refused('HIP device tensor', q, k, k, offsets=at.cpu())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', (1500, 40000))
def test_offsets_that_decrease_stay_inside(rows, dtype):
    """The results are unspecified, but no row outside the tensors is written,
    and none is read: what surrounds the inputs is NaN, what surrounds the
    results and the workspace stays as it is, and what is written is finite.
    (A first key's part would lie some thousand parts before the others.)"""
    import ctypes

    from test_transformer_host import Attention, _library

    lib = _library()
    gen = torch.Generator(device='cuda').manual_seed(23)
    around, dim, heads = 2000, 32, 2
    span = slice(around, around + rows)

    def guarded(count, fill, of=dtype):
        return torch.full((rows + 2 * around, count, dim), fill, dtype=of,
                          device='cuda')

    def at(t):
        return t[span].data_ptr()

    inputs = {n: guarded(c, float('nan'))
              for n, c in (('q', heads), ('k', 1), ('v', 1), ('dy', heads),
                           ('y', heads), ('rest', heads))}
    for t in inputs.values():
        t[span] = _normal(gen, dtype, rows, t.shape[1], dim)
    inputs['rest'][span] = 0
    lse = torch.full((rows + 2 * around, heads), float('nan'), device='cuda')
    lse[span] = 8.0
    results = [guarded(c, 3.0) for c in (heads, heads, 1, 1)]
    states = torch.full((rows + 2 * around, heads), 3.0, device='cuda')
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    for shares in ((0.9, 0.3, 0.35, 0.05, 0.1), (1.0, 0.0), (0.5, 1.0, 0.2)):
        offsets = torch.tensor([int(s * rows) for s in shares],
                               dtype=torch.int32, device='cuda')
        args = Attention(
            dtype=code, queries=rows, keys=rows, heads=heads, kv_heads=1,
            dim=dim, sequences=len(shares) - 1, left=60, right=10, sinks=3,
            scale=dim ** -0.5, q=at(inputs['q']), k=at(inputs['k']),
            v=at(inputs['v']), q_row_stride=heads * dim, q_head_stride=dim,
            k_row_stride=dim, k_head_stride=dim, v_row_stride=dim,
            v_head_stride=dim, offsets=offsets.data_ptr(),
            key_offsets=offsets.data_ptr(), key_lengths=None)
        sizes = [getattr(lib, f'lattice_hip_window_attention{n}'
                         '_workspace_bytes')(ctypes.byref(args))
                 for n in ('', '_grad')]
        guard = 32 << 20
        store = torch.full((max(sizes) + 2 * guard,), 3, dtype=torch.uint8,
                           device='cuda')
        space = store[guard:-guard].zero_()
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

        def pointers(*values):
            return [ctypes.c_void_p(v) for v in values]

        assert lib.lattice_hip_window_attention(
            ctypes.byref(args), *pointers(at(results[0]), at(states), None,
                                          space.data_ptr()),
            ctypes.c_size_t(sizes[0]), stream) == 0
        assert lib.lattice_hip_window_attention_grad(
            ctypes.byref(args), *pointers(
                at(inputs['y']), None if code == 0 else at(inputs['rest']),
                at(lse), at(inputs['dy']), *(at(t) for t in results[1:]),
                space.data_ptr()), ctypes.c_size_t(sizes[1]), stream) == 0
        torch.cuda.synchronize()
        for t in (*results, states):
            assert (t[:around] == 3).all() and (t[span.stop:] == 3).all()
        assert (store[:guard] == 3).all() and (store[-guard:] == 3).all()
        for t in results:
            assert torch.isfinite(t[span]).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('lengths, heads, kv_heads, dim, left, right, sinks', [
    ((300, 77), 4, 2, 32, 40, 3, 2), ((129,), 2, 2, 128, None, 0, 0),
    ((4000, 4600), 8, 4, 64, 90, 0, 5), ((9000,), 4, 4, 32, 33, 64, 0)])
def test_negative_scale(lengths, heads, kv_heads, dim, left, right, sinks,
                        dtype):
    """A negative scale is the positive one with the sign in the queries or the
    keys, bit for bit: no row is made again by itself since a mask met the
    sign.  (A gradient is compared where its sums have the same operands: the
    matrix cores' sums are not symmetric in sign.)"""
    gen = torch.Generator(device='cuda').manual_seed(19)
    rows = sum(lengths)
    q, k, v, dy = (_normal(gen, dtype, rows, h, dim)
                   for h in (heads, kv_heads, kv_heads, heads))
    kwargs = {'left': left, 'right': right, 'sinks': sinks,
              'offsets': _offsets(lengths)}
    out, dq, dk, dv = _run(q, k, v, dy, scale=-0.2, **kwargs)
    of_q = _run(-q, k, v, dy, scale=0.2, **kwargs)
    of_k = _run(q, -k, v, dy, scale=0.2, **kwargs)
    for a, b in ((out, of_q[0]), (out, of_k[0]), (dv, of_q[3]), (dv, of_k[3]),
                 (dq, -of_q[1]), (dk, -of_k[2])):
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('lengths, dim', (((300, 77), 32), ((9000,), 64)))
def test_scale_of_zero(lengths, dim, dtype):
    """Every key that is seen has the same share, as with queries of zero."""
    gen = torch.Generator(device='cuda').manual_seed(20)
    q, k, v, dy = (_normal(gen, dtype, sum(lengths), 4, dim) for _ in range(4))
    kwargs = {'left': 50, 'right': 3, 'sinks': 2, 'offsets': _offsets(lengths)}
    out, dq, dk, dv = _run(q, k, v, dy, scale=0.0, **kwargs)
    want = _run(torch.zeros_like(q), k, v, dy, scale=1.0, **kwargs)
    assert torch.equal(out, want[0]) and torch.equal(dv, want[3])
    assert not dq.any() and not dk.any()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('first', (True, False))
@pytest.mark.parametrize('queries', (1, 300, 66000))
def test_long_tail_under_one_large_score(queries, first, dtype):
    """One key 17.4 above 40,000 others, whose shares of 2^-25 come to a
    thousandth of the result: the first key and the last, few queries, keys
    that are split, and tiles of many queries."""
    keys = 40001
    q = torch.zeros((queries, 1, 32), dtype=dtype, device='cuda')
    k = torch.zeros((keys, 1, 32), dtype=dtype, device='cuda')
    v = torch.ones_like(k)
    # 4 x 4.34375 has the same value in every type.
    at = 0 if first else keys - 1
    q[..., 0], k[at, 0, 0], v[at] = 4, 4.34375, 0
    got = _ops().window_attention(q, k, v, offsets=_offsets((queries,)),
                                  key_offsets=_offsets((keys,)), scale=1.0)
    tail = (keys - 1) * 2.718281828459045 ** -17.375
    want = torch.full(got.shape, tail / (1 + tail), dtype=torch.float64)
    # The result is rounded, and so are the shares: in half precision to
    # eleven bits or, as small as these, at least ten.  The sums are made in
    # float32 over products of two keys (float32) or sixteen, in order.
    unit = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11,
            torch.bfloat16: 2.0 ** -8}[dtype]
    share = 2.0 ** -10 if dtype == torch.float16 else unit
    steps = keys / (2 if dtype == torch.float32 else 16)
    assert_within(got, want, want * (unit + share + steps * 2.0 ** -24))


@pytest.mark.parametrize('dtype', DTYPES)
def test_no_rows_in_any_layout(dtype):
    """Slices without rows are taken in every layout, as slices with rows."""
    gen = torch.Generator(device='cuda').manual_seed(21)
    q, dy = (_normal(gen, dtype, 5, 2, 32) for _ in range(2))
    wide = _normal(gen, dtype, 5, 4, 33)
    none = wide[:0, :2, 1:]
    kwargs = {'offsets': _offsets((5,)), 'key_offsets': _offsets((0,))}
    for value in _run(q, none, none, dy, **kwargs):
        assert not value.any()
    for value, like in zip(_run(none, q, q, none, offsets=_offsets((0,)),
                                key_offsets=_offsets((5,))),
                           (none, none, q, q)):
        assert value.shape == like.shape and not value.any()


def test_more_sequences_than_blocks_of_a_launch():
    """2^24 sequences of a row each: 2^32 threads and more."""
    rows = 2 ** 24 + 3
    gen = torch.Generator(device='cuda').manual_seed(22)
    q, k, v, dy = (_normal(gen, torch.float16, rows, 1, 8) for _ in range(4))
    offsets = torch.arange(rows + 1, dtype=torch.int32, device='cuda')
    out, dq, dk, dv = _run(q, k, v, dy, offsets=offsets)
    # The one key has the whole share.
    assert torch.equal(out, v) and torch.equal(dv, dy)
    # delta is float32's sum of eight products.
    for grad in (dq, dk):
        assert float(grad.abs().max()) < 1e-4
