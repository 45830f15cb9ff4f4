"""Operators of a transformer block over the rows of voxel scans, one pass each:
layer norm, rotary positions by voxel coordinates, attention over a sliding
window with first tokens that stay visible, and counter-based dropout.

``run`` computes them in a plain form of elementary torch operations in
float32, or, where ``own`` is true, through the library's public operators.
A case is a dict of plain values.  Its ``kind``:

* ``attention``: packed sequences.  ``form`` ``self``: every row is a query and
  a key of its scan (``rows`` over ``batches`` scans of unequal length);
  ``cache``: ``q_len`` new tokens of each of ``batches`` sequences against a
  cache of ``cache`` rows a sequence, partly filled.  ``left`` / ``right``: how
  many keys before / after its position a query sees (-1: all); ``sinks``: the
  first keys of a sequence, which every later query sees too; ``grad``: also
  the gradients of q, k and v.
* ``norm``: layer norm of ``rows`` x ``channels``; ``grad``: also the gradients
  of the rows, the weight and the bias.
* ``rotary``: ``heads`` query and ``kv_heads`` key heads of a packed q k v row
  turned by the row's x, y and z; ``grad``: also the gradient.
* ``dropout``: with the ``residual`` it is added to, or without; ``grad``: also
  the gradient.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
_BYTES = {'f32': 4, 'f16': 2, 'bf16': 2}
_EPS = 1e-5
_BASE = 10000.0


def _ops():
    package = str(Path(__file__).resolve().parent.parent / 'mlx-lattice_amd')
    if package not in sys.path:
        sys.path.insert(0, package)
    import mlx_lattice_amd.ops as ops

    return ops


# ----------------------------------------------------------------- cases --


def _attention(dtype, heads, kv_heads, dim, left, right, sinks, *, form='self',
               rows=0, batches=1, q_len=0, cache=0, grad=False):
    return {'kind': 'attention', 'form': form, 'dtype': dtype, 'heads': heads,
            'kv_heads': kv_heads, 'dim': dim, 'left': left, 'right': right,
            'sinks': sinks, 'rows': rows, 'batches': batches, 'q_len': q_len,
            'cache': cache, 'grad': grad}


def listed():
    return [
        # The smallest call: one new token of four streamed scans against
        # their last 512 tokens; launches and host work dominate.
        {'name': 'token_bf16', **_attention(
            'bf16', 8, 2, 64, 512, 0, 4, form='cache', batches=4, q_len=1,
            cache=2048)},
        # Serving with long caches: one new token of 32 sequences, all of
        # whose keys are visible.
        {'name': 'token_long_f16', **_attention(
            'f16', 16, 4, 128, -1, 0, 0, form='cache', batches=32, q_len=1,
            cache=32768)},
        # An encoder level served over four scans: each voxel sees the 128
        # rows before and after it in scan order.
        {'name': 'scan_f16', **_attention(
            'f16', 8, 8, 32, 128, 128, 4, rows=120000, batches=4)},
        # The longest sequence: a causal decoder's first pass.
        {'name': 'causal_bf16', **_attention(
            'bf16', 16, 4, 128, 4096, 0, 16, rows=16384)},
        # Training of the same level in half precision ...
        {'name': 'scan_train_bf16', **_attention(
            'bf16', 4, 2, 64, 256, 256, 4, rows=60001, batches=2, grad=True)},
        # ... and of a small grid in the default type.
        {'name': 'scan_train_f32', **_attention(
            'f32', 4, 4, 32, 100, 27, 1, rows=20000, batches=3, grad=True)},
        # Layer norm of a small grid's narrow rows, and in training over the
        # headline layer's rows.
        {'name': 'norm_f32', 'kind': 'norm', 'dtype': 'f32', 'rows': 20000,
         'channels': 32, 'grad': False},
        {'name': 'norm_train_f16', 'kind': 'norm', 'dtype': 'f16',
         'rows': 400000, 'channels': 128, 'grad': True},
        # Rotary positions of a served level, and in training in the default
        # type.
        {'name': 'rotary_bf16', 'kind': 'rotary', 'dtype': 'bf16',
         'rows': 200000, 'heads': 8, 'kv_heads': 8, 'dim': 32, 'grad': False},
        {'name': 'rotary_train_f32', 'kind': 'rotary', 'dtype': 'f32',
         'rows': 60001, 'heads': 4, 'kv_heads': 2, 'dim': 64, 'grad': True},
        # Dropout into the residual stream in training, and of rows whose
        # width fills no vector.
        {'name': 'dropout_train_f16', 'kind': 'dropout', 'dtype': 'f16',
         'rows': 400000, 'channels': 128, 'percent': 10, 'residual': True,
         'grad': True},
        {'name': 'dropout_f32', 'kind': 'dropout', 'dtype': 'f32',
         'rows': 100003, 'channels': 30, 'percent': 50, 'residual': False,
         'grad': False},
    ]


def draw(rng):
    """A case of the ranges above; sizes are log-uniform and mostly odd."""
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(('token', 'chunk', 'scan', 'scan', 'causal', 'train',
                       'train', 'norm', 'norm', 'rotary', 'dropout'))
    dtype = rng.choice(('f32', 'f16', 'bf16'))
    if kind == 'norm':
        channels = rng.choice((3, 16, 30, 32, 64, 96, 128, 256, 512, 1000))
        return {'kind': 'norm', 'dtype': dtype,
                'rows': size(1, 80_000_000 // (channels * _BYTES[dtype])),
                'channels': channels, 'grad': rng.random() < 0.6}
    if kind == 'rotary':
        heads, kv_heads = rng.choice(((8, 8), (4, 2), (8, 2), (16, 4), (3, 1)))
        dim = rng.choice((16, 32, 48, 64, 128))
        return {'kind': 'rotary', 'dtype': dtype,
                'rows': size(1, 160_000_000 // ((heads + kv_heads) * dim
                                                * _BYTES[dtype])),
                'heads': heads, 'kv_heads': kv_heads, 'dim': dim,
                'grad': rng.random() < 0.5}
    if kind == 'dropout':
        channels = rng.choice((1, 7, 30, 64, 96, 128, 257))
        return {'kind': 'dropout', 'dtype': dtype,
                'rows': size(1, 80_000_000 // (channels * _BYTES[dtype])),
                'channels': channels, 'percent': rng.choice((5, 10, 25, 50)),
                'residual': rng.random() < 0.5, 'grad': rng.random() < 0.5}
    kv_heads = rng.choice((1, 2, 4))
    heads = kv_heads * rng.choice((1, 2, 4))
    dim = rng.choice((16, 24, 32, 64, 64, 80, 128))
    sinks = rng.choice((0, 1, 4, 16))
    if kind == 'token':
        return _attention(dtype, heads, kv_heads, dim,
                          rng.choice((-1, size(16, 4096))), 0, sinks,
                          form='cache', batches=size(1, 32), q_len=1,
                          cache=size(16, 10000))
    if kind == 'chunk':
        return _attention(dtype, heads, kv_heads, dim,
                          rng.choice((-1, size(64, 4096))), 0, sinks,
                          form='cache', batches=rng.choice((1, 2, 4)),
                          q_len=size(2, 500), cache=size(600, 8000))
    if kind == 'causal':
        grad = rng.random() < 0.4
        return _attention(dtype, heads, kv_heads, dim, size(200, 4096), 0,
                          sinks, rows=size(100, 4000 if grad else 10000),
                          grad=grad)
    return _attention(dtype, heads, kv_heads, dim, size(8, 300),
                      size(8, 300), sinks,
                      rows=size(50, 25000 if kind == 'train' else 40000),
                      batches=rng.choice((1, 2, 4, 7)), grad=kind == 'train')


def _lengths(case):
    """(queries, keys) of each sequence."""
    n = case['batches']
    if case['form'] == 'cache':
        longest = case['cache']
        keys = [max(case['q_len'], longest - (b * 977) % (longest // 2 + 1))
                for b in range(n)]
        return [case['q_len']] * n, keys
    shares = [5 + (3 * b) % 7 for b in range(n)]
    ends = [case['rows'] * sum(shares[:b + 1]) // sum(shares)
            for b in range(n)]
    own_rows = [hi - lo for lo, hi in zip([0] + ends, ends)]
    return own_rows, own_rows


def _dims(dim):
    """Channels of a head turned by x, y and z: whole pairs, the rest to x."""
    third = dim // 6 * 2
    return (dim // 2 * 2 - 2 * third, third, third)


# --------------------------------------------------------------- prepare --


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(int(seed))
    dtype = _DTYPES[case['dtype']]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=gen, device='cuda') * scale
                + shift).to(dtype)

    state = {'case': case}
    kind, grad = case['kind'], case['grad']
    if kind == 'norm':
        rows, channels = case['rows'], case['channels']
        # Rows of unequal size whose channels do not average to zero.
        spread = torch.rand((rows, 1), generator=gen, device='cuda') * 2 + 0.2
        shift = torch.randn((1, channels), generator=gen, device='cuda') * 0.5
        x = torch.randn((rows, channels), generator=gen, device='cuda')
        state['x'] = (x * spread + shift).to(dtype).requires_grad_(grad)
        state['weight'] = normal(channels, scale=0.2,
                                 shift=1.0).requires_grad_(grad)
        state['bias'] = normal(channels, scale=0.2).requires_grad_(grad)
        if grad:
            state['dy'] = normal(rows, channels)
        return state
    if kind == 'dropout':
        rows, channels = case['rows'], case['channels']
        state['x'] = normal(rows, channels).requires_grad_(grad)
        state['residual'] = (normal(rows, channels) if case['residual']
                             else None)
        state['seed'] = int(seed) * 0x9E3779B1 + 12345
        state['offset'] = int(seed) % 1000
        if grad:
            state['dy'] = normal(rows, channels)
        return state
    if kind == 'rotary':
        rows, dim = case['rows'], case['dim']
        turned = case['heads'] + case['kv_heads']
        qkv = normal(rows, turned + case['kv_heads'], dim)
        state['x'] = qkv[:, :turned].requires_grad_(grad)
        # The voxels of a scan in a cube of 256.
        state['coords'] = torch.randint(0, 256, (rows, 4), generator=gen,
                                        device='cuda', dtype=torch.int32)
        dims = _dims(dim)
        state['dims'] = dims
        state['frequencies'] = torch.tensor(
            [_BASE ** (-2.0 * i / d) for d in dims for i in range(d // 2)],
            dtype=torch.float64, device='cuda')
        if grad:
            state['dy'] = normal(rows, turned, dim)
        return state
    heads, kv_heads, dim = case['heads'], case['kv_heads'], case['dim']
    queries, keys = _lengths(case)
    offsets = np.concatenate([[0], np.cumsum(queries)])
    state['offsets'] = torch.tensor(offsets, dtype=torch.int32, device='cuda')
    rows = int(offsets[-1])
    if case['form'] == 'cache':
        state['q'] = normal(rows, heads, dim)
        key_rows = case['batches'] * case['cache']
        state['k'] = normal(key_rows, kv_heads, dim)
        state['v'] = normal(key_rows, kv_heads, dim)
        state['key_offsets'] = torch.arange(
            case['batches'] + 1, dtype=torch.int32,
            device='cuda') * case['cache']
        state['key_lengths'] = torch.tensor(keys, dtype=torch.int32,
                                            device='cuda')
    else:
        # One projection makes q, k and v: the three are slices of its rows.
        qkv = normal(rows, heads + 2 * kv_heads, dim)
        state['q'] = qkv[:, :heads].requires_grad_(grad)
        state['k'] = qkv[:, heads:heads + kv_heads].requires_grad_(grad)
        state['v'] = qkv[:, heads + kv_heads:].requires_grad_(grad)
    if grad:
        state['dy'] = normal(rows, heads, dim)
    return state


# ------------------------------------------------------------------- run --


def run(state):
    case = state['case']
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        return {'attention': _plain_attention, 'norm': _plain_norm,
                'rotary': _plain_rotary,
                'dropout': _plain_dropout}[case['kind']](state, case)


def _run_own(state, case):
    ops, kind = _ops(), case['kind']
    if kind == 'norm':
        inputs = (state['x'], state['weight'], state['bias'])
        out = ops.layer_norm(*inputs, eps=_EPS)
    elif kind == 'dropout':
        inputs = (state['x'],)
        out = ops.dropout(state['x'], case['percent'] / 100,
                          seed=state['seed'], offset=state['offset'],
                          residual=state['residual'])
    elif kind == 'rotary':
        inputs = (state['x'],)
        out = ops.rotary_positions(state['x'], state['coords'][:, 1:],
                                   state['frequencies'], dims=state['dims'])
    else:
        inputs = (state['q'], state['k'], state['v'])
        out = ops.window_attention(
            *inputs, left=None if case['left'] < 0 else case['left'],
            right=None if case['right'] < 0 else case['right'],
            sinks=case['sinks'], offsets=state['offsets'],
            key_offsets=state.get('key_offsets'),
            key_lengths=state.get('key_lengths'))
    if not case['grad']:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, inputs, state['dy'])]


def _plain_norm(state, case):
    x, weight = state['x'].float(), state['weight'].float()
    dtype = state['x'].dtype
    centred = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + _EPS)
    normed = centred * rstd
    out = (normed * weight + state['bias'].float()).to(dtype)
    if not case['grad']:
        return [out]
    dy = state['dy'].float()
    scaled = dy * weight
    dx = rstd * (scaled - scaled.mean(1, keepdim=True)
                 - normed * (scaled * normed).mean(1, keepdim=True))
    return [out, dx.to(dtype), (dy * normed).sum(0).to(dtype),
            dy.sum(0).to(dtype)]


def _plain_words(numbers, counter_high, key):
    """The four 32-bit words of Philox 4x32-10 for every counter
    ``(numbers, counter_high)``: (count, 4), in int64."""
    mask = 0xFFFFFFFF

    def product(a, b):
        low = a * (b & 0xFFFF)
        high = a * (b >> 16) + (low >> 16)
        return (high >> 16) & mask, ((high & 0xFFFF) << 16) | (low & 0xFFFF)

    words = [numbers & mask, numbers >> 32,
             torch.full_like(numbers, counter_high & mask),
             torch.full_like(numbers, counter_high >> 32 & mask)]
    for step in range(10):
        key0 = ((key & mask) + step * 0x9E3779B9) & mask
        key1 = ((key >> 32 & mask) + step * 0xBB67AE85) & mask
        high0, low0 = product(0xD2511F53, words[0])
        high1, low1 = product(0xCD9E8D57, words[2])
        words = [high1 ^ words[1] ^ key0, low1, high0 ^ words[3] ^ key1, low0]
    return torch.stack(words, 1)


def _plain_dropout(state, case):
    x = state['x']
    count = x.numel()
    numbers = torch.arange((count + 3) // 4, device=x.device)
    words = _plain_words(numbers, state['offset'], state['seed'])
    keep = (words.reshape(-1)[:count].reshape(x.shape)
            >= round(case['percent'] / 100 * 2 ** 32))
    scale = 1 / (1 - case['percent'] / 100)

    def drop(values):
        return torch.where(keep, values.float() * scale, 0.0)

    out = drop(x)
    if case['residual']:
        out = out + state['residual'].float()
    out = out.to(x.dtype)
    return [out, drop(state['dy']).to(x.dtype)] if case['grad'] else [out]


def _plain_rotary(state, case):
    x, dims = state['x'], state['dims']
    position = state['coords'][:, 1:].float()
    frequency = state['frequencies'].float()
    axis = torch.arange(3, device=x.device).repeat_interleave(
        torch.tensor([d // 2 for d in dims], device=x.device),
        output_size=sum(dims) // 2)
    angle = position[:, axis] * frequency
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    # The channels of the pairs: the first and second half of each axis.
    pair = torch.arange(sum(dims) // 2, device=x.device)
    starts = torch.tensor([0, dims[0], dims[0] + dims[1]], device=x.device)
    halves = torch.tensor([d // 2 for d in dims], device=x.device)
    first = starts[axis] + pair - starts[axis] // 2
    second = first + halves[axis]

    def turn(values, sin):
        values = values.float()
        u, v = values[..., first], values[..., second]
        out = values.clone()
        out[..., first] = u * cos - v * sin
        out[..., second] = u * sin + v * cos
        return out.to(x.dtype)

    out = turn(x, sin)
    return [out, turn(state['dy'], -sin)] if case['grad'] else [out]


def _plain_attention(state, case):
    """Blocks of query rows against the band of keys they can see, and the
    first keys of each row's sequence apart from the band."""
    q, k, v = state['q'], state['k'], state['v']
    dtype, device = q.dtype, q.device
    rows, heads, dim = q.shape
    key_rows, kv_heads = k.shape[:2]
    group = heads // kv_heads
    queries, keys = _lengths(case)
    left = max(keys) if case['left'] < 0 else min(case['left'], max(keys))
    right = max(keys) if case['right'] < 0 else min(case['right'], max(keys))
    step = (case['q_len'] if case['form'] == 'cache'
            else min(rows, 1024, max(64, left + right)))
    blocks = -(-rows // step)
    offsets = state['offsets'].long()
    key_offsets = state.get('key_offsets', state['offsets']).long()
    row = torch.arange(blocks * step, device=device)
    real = (row < rows).reshape(blocks, step)
    row = row.clamp(max=rows - 1).reshape(blocks, step)
    seq = torch.bucketize(row, offsets[1:], right=True)
    starts = key_offsets[seq]
    lengths = (state['key_lengths'].long()[seq] if 'key_lengths' in state
               else key_offsets[seq + 1] - starts)
    position = (row - offsets[seq] + lengths
                - (offsets[seq + 1] - offsets[seq]))

    def seen(index):
        """(in the window, a first key outside it) of key ``index`` of the
        row's own sequence."""
        p = position[..., None]
        valid = (real[..., None] & (index >= 0) & (index <= p + right)
                 & (index < lengths[..., None]))
        return valid & (index >= p - left), valid & (index < p - left)

    band = ((starts + position)[:, :1] - left
            + torch.arange(step + left + right, device=device))
    in_window = seen(band[:, None] - starts[..., None])[0][:, None, None]
    band = band.clamp(0, key_rows - 1)
    sinks = torch.arange(case['sinks'], device=device)
    is_sink = seen(sinks.expand(blocks, step, -1))[1][:, None, None]
    sink_rows = (starts[..., None] + sinks).clamp(max=key_rows - 1)

    def of_queries(x):  # (blocks, kv_heads, group, step, dim)
        return x[row].float().reshape(blocks, step, kv_heads, group,
                                      dim).permute(0, 2, 3, 1, 4)

    def of_band(x):  # (blocks, kv_heads, 1, band, dim)
        return x[band].float().permute(0, 2, 1, 3)[:, :, None].contiguous()

    def of_sinks(x):  # (blocks, kv_heads, step, sinks, dim)
        return x[sink_rows].float().permute(0, 3, 1, 2, 4).contiguous()

    def with_band(a, b):  # a's rows by b's
        flat = a.reshape(blocks, kv_heads, 1, group * step, dim)
        return (flat @ b.transpose(-1, -2)).reshape(blocks, kv_heads, group,
                                                    step, -1)

    def with_sinks(a, b):
        return (a.transpose(2, 3) @ b.transpose(-1, -2)).transpose(2, 3)

    def over_band(p, b):  # the sum of b's rows by p
        return (p.reshape(blocks, kv_heads, 1, group * step, -1)
                @ b).reshape(blocks, kv_heads, group, step, dim)

    def over_sinks(p, b):
        return (p.transpose(2, 3) @ b).transpose(2, 3)

    def to_rows(x):
        return x.permute(0, 3, 1, 2, 4).reshape(
            blocks * step, heads, dim)[:rows].to(dtype)

    scale = dim ** -0.5
    q32, kb, vb = of_queries(q), of_band(k), of_band(v)
    ks, vs = of_sinks(k), of_sinks(v)
    low = -math.inf
    sb = torch.where(in_window, with_band(q32, kb) * scale, low)
    ss = torch.where(is_sink, with_sinks(q32, ks) * scale, low)
    top = sb.amax(-1, keepdim=True)
    if case['sinks']:
        top = torch.maximum(top, ss.amax(-1, keepdim=True))
    top = torch.where(top == low, 0.0, top)
    sb, ss = torch.exp(sb - top), torch.exp(ss - top)
    total = sb.sum(-1, keepdim=True) + ss.sum(-1, keepdim=True)
    total = torch.where(total == 0, 1.0, total)
    sb, ss = sb / total, ss / total
    out = over_band(sb, vb) + over_sinks(ss, vs)
    if not case['grad']:
        return [to_rows(out)]
    dy = of_queries(state['dy'])
    delta = (dy * out).sum(-1, keepdim=True)
    db = sb * (with_band(dy, vb) - delta)
    ds = ss * (with_sinks(dy, vs) - delta)
    dq = (over_band(db, kb) + over_sinks(ds, ks)) * scale

    def to_keys(pb, ps, a):
        """The sum over queries of ``a``'s rows by p, into the key rows."""
        flat = a.reshape(blocks, kv_heads, group * step, dim)
        of_b = (pb.reshape(blocks, kv_heads, group * step, -1).transpose(
            -1, -2) @ flat).permute(0, 2, 1, 3)
        of_s = (ps.transpose(2, 3).transpose(-1, -2)
                @ a.transpose(2, 3)).permute(0, 2, 3, 1, 4)
        out = torch.zeros((key_rows, kv_heads, dim), device=device)
        out.index_add_(0, band.reshape(-1),
                       of_b.reshape(-1, kv_heads, dim))
        out.index_add_(0, sink_rows.reshape(-1),
                       of_s.reshape(-1, kv_heads, dim))
        return out

    dk = to_keys(db, ds, q32) * scale
    dv = to_keys(sb, ss, dy)
    return [to_rows(out), to_rows(dq), dk.to(dtype), dv.to(dtype)]


# ------------------------------------------------------------------ work --


def _pairs(case):
    """(visible query-key pairs, key rows that some query sees)."""
    pairs = touched = 0
    for nq, nk in zip(*_lengths(case)):
        p = np.arange(nq, dtype=np.int64) + nk - nq
        left = nk if case['left'] < 0 else case['left']
        right = nk if case['right'] < 0 else case['right']
        lo = np.maximum(0, p - left)
        hi = np.minimum(nk - 1, p + right)
        seen = np.maximum(0, hi - lo + 1)
        pairs += int((seen + np.minimum(case['sinks'], lo)).sum())
        if nq:
            touched += int(hi[-1] - lo[0] + 1 + min(case['sinks'], lo[0]))
    return pairs, touched


def work(case):
    size = _BYTES[case['dtype']]
    kind, grad = case['kind'], case['grad']
    if kind == 'attention':
        pairs, touched = _pairs(case)
        row = case['dim'] * size
        rows = sum(_lengths(case)[0])
        of_q, of_k = rows * case['heads'] * row, touched * case['kv_heads'] * row
        return {'bytes': 2 * of_q + 2 * of_k + (2 * of_q + 2 * of_k
                                                if grad else 0),
                'flops': pairs * case['heads'] * case['dim']
                * (14 if grad else 4)}
    if kind == 'rotary':
        turned = case['heads'] + case['kv_heads']
        values = case['rows'] * turned * case['dim']
        return {'bytes': 2 * values * size * (2 if grad else 1)
                + case['rows'] * 12, 'flops': 3 * values * (2 if grad else 1)}
    values = case['rows'] * case['channels']
    if kind == 'norm':
        arrays = 4 if grad else 2
        return {'bytes': arrays * values * size + 4 * case['channels'] * size,
                'flops': values * (20 if grad else 8)}
    arrays = 2 + bool(case['residual']) + (2 if grad else 0)
    return {'bytes': arrays * values * size, 'flops': 2 * values}


# ----------------------------------------------------------------- exact --


def exact(case, seed):
    """The outputs of ``run`` in float64, from the definitions."""
    state = prepare(case, seed)
    with torch.no_grad():
        return {'attention': _exact_attention, 'norm': _exact_norm,
                'rotary': _exact_rotary,
                'dropout': _exact_dropout}[case['kind']](state, case)


def _exact_norm(state, case):
    x = state['x'].double()
    weight, bias = state['weight'].double(), state['bias'].double()
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    root = torch.sqrt(var + _EPS)
    normed = (x - mean) / root
    out = normed * weight + bias
    if not case['grad']:
        return [out]
    dy = state['dy'].double()
    g = dy * weight
    channels = x.shape[1]
    along = (g * normed).sum(1, keepdim=True)
    dx = (channels * g - g.sum(1, keepdim=True) - normed * along) / (
        channels * root)
    return [out, dx, torch.einsum('nc,nc->c', dy, normed), dy.sum(0)]


def _exact_dropout(state, case):
    x = state['x']
    count = x.numel()
    number = np.arange((count + 3) // 4, dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    key = [state['seed'] & 0xFFFFFFFF, state['seed'] >> 32 & 0xFFFFFFFF]
    c0, c1 = number & low, number >> half
    c2 = np.full_like(number, state['offset'] & 0xFFFFFFFF)
    c3 = np.full_like(number, state['offset'] >> 32 & 0xFFFFFFFF)
    for _ in range(10):
        a, b = c0 * np.uint64(0xD2511F53), c2 * np.uint64(0xCD9E8D57)
        c0, c1, c2, c3 = ((b >> half) ^ c1 ^ np.uint64(key[0]), b & low,
                          (a >> half) ^ c3 ^ np.uint64(key[1]), a & low)
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF,
               (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    words = np.stack([c0, c1, c2, c3], 1).reshape(-1)[:count]
    share = case['percent'] / 100
    keep = torch.from_numpy(words >= np.uint64(round(share * 2 ** 32)))
    factor = keep.to(x.device).reshape(x.shape).double() / (1 - share)
    out = x.double() * factor
    if case['residual']:
        out += state['residual'].double()
    return [out, state['dy'].double() * factor] if case['grad'] else [out]


def _exact_rotary(state, case):
    coords, dims = state['coords'].double(), state['dims']

    def turn(values, sign):
        out = values.double().clone()
        start = used = 0
        for axis, width in enumerate(dims):
            half = width // 2
            angle = sign * (coords[:, 1 + axis, None]
                            * state['frequencies'][used:used + half])
            turned = torch.polar(torch.ones_like(angle), angle)[:, None]
            values64 = values[..., start:start + width].double()
            pair = torch.complex(values64[..., :half].contiguous(),
                                 values64[..., half:].contiguous()) * turned
            out[..., start:start + width] = torch.cat([pair.real, pair.imag],
                                                      -1)
            start, used = start + width, used + half
        return out

    out = turn(state['x'], 1.0)
    return [out, turn(state['dy'], -1.0)] if case['grad'] else [out]


def _exact_attention(state, case):
    """Sequence by sequence, some query rows at a time, against the keys from
    the first to the last that they can see and the sequence's first keys."""
    q, k, v = (state[n].double() for n in 'qkv')
    grad = case['grad']
    heads, kv_heads, dim = case['heads'], case['kv_heads'], case['dim']
    group = heads // kv_heads
    out = torch.zeros_like(q)
    if grad:
        dy = state['dy'].double()
        dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v))
    first_row = 0
    for b, (nq, nk) in enumerate(zip(*_lengths(case))):
        key_start = (b * case['cache'] if case['form'] == 'cache'
                     else first_row)
        left = nk if case['left'] < 0 else case['left']
        right = nk if case['right'] < 0 else case['right']
        for at in range(0, nq, 1024):
            end = min(nq, at + 1024)
            rows = slice(first_row + at, first_row + end)
            pos = torch.arange(at, end, device=q.device)[:, None] + nk - nq
            lo = max(0, at + nk - nq - left)
            hi = max(lo, min(nk, end + nk - nq + right))
            index = torch.cat([torch.arange(min(case['sinks'], lo)),
                               torch.arange(lo, hi)]).to(q.device)
            visible = (index <= pos + right) & ((index >= pos - left)
                                                | (index < case['sinks']))
            for g in range(kv_heads):
                own_heads = slice(g * group, (g + 1) * group)
                kk, vv = k[key_start + index, g], v[key_start + index, g]
                qq = q[rows, own_heads].transpose(0, 1)
                scores = (qq @ kk.T) / math.sqrt(dim)
                scores = scores.masked_fill(~visible, -math.inf)
                share = torch.softmax(scores, -1)
                share = share.masked_fill(~visible, 0.0)
                result = share @ vv
                out[rows, own_heads] = result.transpose(0, 1)
                if not grad:
                    continue
                dd = dy[rows, own_heads].transpose(0, 1)
                slope = share * (dd @ vv.T - (dd * result).sum(
                    -1, keepdim=True)) / math.sqrt(dim)
                dq[rows, own_heads] = (slope @ kk).transpose(0, 1)
                dk[:, g].index_add_(0, key_start + index, torch.bmm(
                    slope.transpose(1, 2), qq).sum(0))
                dv[:, g].index_add_(0, key_start + index, torch.bmm(
                    share.transpose(1, 2), dd).sum(0))
        first_row += nq
    return [out, dq, dk, dv] if grad else [out]
