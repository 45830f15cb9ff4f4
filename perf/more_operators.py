"""Operators of a transformer block as it is served and trained, one pass each:
a cache of keys and values in 8 bits that is written, read back and attended
to, and the junction of two parts of a block (norm, gate and scale of what one
part gives, the residual sum, the next part's norm).

``run`` computes them in a plain form of elementary torch operations in
float32, or, where ``own`` is true, through the library's public operators.
A case is a dict of plain values.  Its ``kind``:

* ``attention``: ``q_len`` new tokens of each of ``batches`` sequences against
  a cache of ``cache`` tokens a sequence, partly filled; ``left`` / ``right``:
  how many tokens before / after its position a query sees (-1: all);
  ``sinks``: the first tokens, which every later query sees too.
* ``write``: ``rows`` new tokens over ``batches`` sequences of unequal length,
  appended to a cache of ``cache`` tokens a sequence.  Its outputs are the
  codes, in their 8-bit type, and the exponents of two that scale them.
* ``read``: the whole of such a cache in ``dtype``, zeros past the lengths.
* ``junction``: ``rows`` x ``channels``; ``norm`` ``layer`` or ``rms``;
  ``post``: the part's result is normed first; ``gate``: a factor a channel;
  ``grad``: also the gradients of both inputs and of every vector.

``code`` is the cache's 8-bit type: ``e4m3`` or ``int8``.  The cache holds, for
each block of 32 tokens and key head, keys ``(32, width)`` and values ``(width,
32)``, ``width`` being ``dim`` rounded up to 32, and a power of two for each.
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
_CODES = {'e4m3': torch.float8_e4m3fn, 'int8': torch.int8}
_BLOCK = 32
_EPS = 1e-5
_SCALE = 0.5  # of a junction's gated part
_LOW = -126  # the least exponent of a block


def _package():
    package = str(Path(__file__).resolve().parent.parent / 'mlx-lattice_amd')
    if package not in sys.path:
        sys.path.insert(0, package)
    import mlx_lattice_amd.core as core
    import mlx_lattice_amd.ops as ops

    return core, ops


# ----------------------------------------------------------------- cases --


def _attention(code, dtype, heads, kv_heads, dim, batches, q_len, cache,
               left=-1, right=0, sinks=0):
    return {'kind': 'attention', 'code': code, 'dtype': dtype, 'heads': heads,
            'kv_heads': kv_heads, 'dim': dim, 'batches': batches,
            'q_len': q_len, 'cache': cache, 'left': left, 'right': right,
            'sinks': sinks}


def _write(code, dtype, kv_heads, dim, batches, rows, cache):
    return {'kind': 'write', 'code': code, 'dtype': dtype,
            'kv_heads': kv_heads, 'dim': dim, 'batches': batches,
            'rows': rows, 'cache': cache}


def _read(code, dtype, kv_heads, dim, batches, cache):
    return {'kind': 'read', 'code': code, 'dtype': dtype,
            'kv_heads': kv_heads, 'dim': dim, 'batches': batches,
            'cache': cache}


def _junction(dtype, rows, channels, norm='layer', post=False, gate=False,
              grad=False):
    return {'kind': 'junction', 'dtype': dtype, 'rows': rows,
            'channels': channels, 'norm': norm, 'post': post, 'gate': gate,
            'grad': grad}


def listed():
    return [
        # The smallest call: one new token of four streamed scans against
        # their last 512 tokens; launches and host work dominate.
        {'name': 'token_e4m3_bf16', **_attention(
            'e4m3', 'bf16', 8, 2, 64, 4, 1, 2048, left=512, sinks=4)},
        # Serving with long caches: one new token of 32 sequences, all of
        # whose tokens are visible.
        {'name': 'token_long_e4m3_f16', **_attention(
            'e4m3', 'f16', 16, 4, 128, 32, 1, 32768)},
        # The same in the default type, with heads that fill no tile.
        {'name': 'token_int8_f32', **_attention(
            'int8', 'f32', 6, 2, 80, 16, 1, 8000)},
        # A long prompt fed in pieces: causal, against what is cached.
        {'name': 'chunk_e4m3_bf16', **_attention(
            'e4m3', 'bf16', 16, 4, 128, 2, 2048, 16384)},
        # An encoder level's scans streamed slab by slab, in a window.
        {'name': 'chunk_int8_f16', **_attention(
            'int8', 'f16', 8, 8, 32, 4, 333, 4096, left=1024, sinks=4)},
        # One new token of 32 sequences goes into the cache ...
        {'name': 'write_token_e4m3_bf16', **_write(
            'e4m3', 'bf16', 4, 128, 32, 32, 2048)},
        # ... and whole prompts, of unequal length.
        {'name': 'write_prompt_int8_f16', **_write(
            'int8', 'f16', 8, 128, 4, 30001, 16384)},
        # A cache is read back to be attended to in the rows' own type, ...
        {'name': 'read_e4m3_bf16', **_read('e4m3', 'bf16', 4, 128, 8, 8192)},
        # ... and a small one, with heads that fill no tile.
        {'name': 'read_int8_f32', **_read('int8', 'f32', 2, 80, 3, 1000)},
        # The junction behind the attention for one token of 32 sequences,
        {'name': 'junction_token_bf16', **_junction(
            'bf16', 32, 512, norm='rms', post=True, gate=True)},
        # in training over the headline layer's rows,
        {'name': 'junction_train_f16', **_junction(
            'f16', 400000, 128, gate=True, grad=True)},
        # and of wide rows with norms on both sides, in the default type.
        {'name': 'junction_train_f32', **_junction(
            'f32', 25013, 1000, norm='rms', post=True, gate=True,
            grad=True)},
    ]


def draw(rng):
    """A case of the ranges above; sizes are log-uniform and mostly odd."""
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(('token', 'token', 'chunk', 'chunk', 'write_token',
                       'write', 'read', 'junction', 'junction', 'junction'))
    dtype = rng.choice(('f32', 'f16', 'bf16'))
    if kind == 'junction':
        channels = rng.choice((3, 16, 30, 32, 64, 96, 128, 256, 512, 1000,
                               2048))
        return _junction(
            dtype, size(1, 100_000_000 // (channels * _BYTES[dtype])),
            channels, norm=rng.choice(('layer', 'rms')),
            post=rng.random() < 0.4, gate=rng.random() < 0.6,
            grad=rng.random() < 0.6)
    code = rng.choice(('e4m3', 'int8'))
    kv_heads = rng.choice((1, 2, 4, 8))
    dim = rng.choice((16, 24, 32, 64, 64, 80, 96, 128, 128))
    if kind == 'write_token':
        batches = size(1, 64)
        return _write(code, dtype, kv_heads, dim, batches, batches,
                      size(40, 2000))
    if kind == 'write':
        batches = rng.choice((1, 2, 3, 7))
        rows = size(20, 8000) * batches
        return _write(code, dtype, kv_heads, dim, batches, rows,
                      2 * rows // batches + size(1, 2000))
    if kind == 'read':
        return _read(code, dtype, kv_heads, dim, size(1, 16), size(20, 4000))
    heads = kv_heads * rng.choice((1, 2, 4))
    left = rng.choice((-1, size(16, 4096)))
    sinks = rng.choice((0, 1, 4, 16))
    if kind == 'token':
        return _attention(code, dtype, heads, kv_heads, dim, size(1, 32), 1,
                          size(16, 10000), left=left, sinks=sinks)
    return _attention(code, dtype, heads, kv_heads, dim, rng.choice((1, 2, 4)),
                      size(2, 600), size(700, 8000), left=left,
                      right=rng.choice((0, 0, 40)), sinks=sinks)


def _capacity(case):
    return -(-case['cache'] // _BLOCK) * _BLOCK


def _width(case):
    return -(-case['dim'] // 32) * 32


def _lengths(case):
    """(new tokens, tokens with the new ones) of each sequence."""
    n, longest = case['batches'], case['cache']
    if case['kind'] != 'write':
        new = case.get('q_len', 0)
        return [new] * n, [max(new, longest - (b * 977) % (longest // 2 + 1))
                           for b in range(n)]
    if case['rows'] == n:
        return [1] * n, [1 + (b * 977 + longest - 3) % longest
                         for b in range(n)]
    shares = [5 + (3 * b) % 7 for b in range(n)]
    ends = [case['rows'] * sum(shares[:b + 1]) // sum(shares)
            for b in range(n)]
    new = [hi - lo for lo, hi in zip([0] + ends, ends)]
    # Every second sequence goes on behind earlier tokens.
    return new, [c + (b % 2) * ((b * 977 + 5) % max(1, longest - c + 1))
                 for b, c in enumerate(new)]


def _touched(case):
    """(sequence, block) of every block that gets new tokens."""
    return [(b, block) for b, (new, total) in enumerate(zip(*_lengths(case)))
            for block in range((total - new) // _BLOCK,
                               (total - 1) // _BLOCK + 1) if new]


# --------------------------------------------------------------- prepare --


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(int(seed))
    dtype = _DTYPES[case['dtype']]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=gen, device='cuda') * scale
                + shift).to(dtype)

    state = {'case': case}
    if case['kind'] == 'junction':
        rows, channels, grad = case['rows'], case['channels'], case['grad']
        # Rows of unequal size whose channels do not average to zero.
        spread = torch.rand((rows, 1), generator=gen, device='cuda') * 2 + 0.2
        shift = torch.randn((1, channels), generator=gen, device='cuda') * 0.5
        residual = torch.randn((rows, channels), generator=gen, device='cuda')
        state['residual'] = (residual * spread + shift).to(
            dtype).requires_grad_(grad)
        state['x'] = normal(rows, channels).requires_grad_(grad)
        for name, used, middle in (
                ('weight', True, 1.0), ('bias', case['norm'] == 'layer', 0.0),
                ('gate', case['gate'], 0.3), ('post_weight', case['post'], 1.0),
                ('post_bias', case['post'] and case['norm'] == 'layer', 0.0)):
            state[name] = normal(channels, scale=0.2, shift=middle
                                 ).requires_grad_(grad) if used else None
        if grad:
            state['d_sum'] = normal(rows, channels)
            state['d_normed'] = normal(rows, channels)
        return state
    heads, width, n = case['kv_heads'], _width(case), case['batches']
    capacity, dim = _capacity(case), case['dim']
    new, total = _lengths(case)

    def codes(shape, channel):
        """Values of unequal channels, some large, as they lie in a cache."""
        spread = torch.rand(width, generator=gen, device='cuda') + 0.3
        spread[dim:] = 0
        along = [1] * len(shape)
        along[channel] = width
        x = torch.randn(shape, generator=gen, device='cuda')
        x *= spread.view(along)
        if case['code'] == 'int8':
            return x.mul_(24).round_().clamp_(-127, 127).to(torch.int8)
        return x.mul_(80).clamp_(-448, 448).to(torch.float8_e4m3fn)

    state['keys'] = codes((n, heads, capacity, width), 3)
    state['values'] = codes((n, heads, capacity // _BLOCK, width, _BLOCK), 3)
    for name in ('key_exponents', 'value_exponents'):
        state[name] = torch.randint(
            -8, -4, (n, heads, capacity // _BLOCK), generator=gen,
            device='cuda', dtype=torch.int8)
    state['lengths'] = torch.tensor(total, dtype=torch.int32, device='cuda')
    state['offsets'] = torch.tensor(np.concatenate([[0], np.cumsum(new)]),
                                    dtype=torch.int32, device='cuda')
    if case['kind'] == 'attention':
        state['q'] = normal(sum(new), case['heads'], dim)
    if case['kind'] == 'write':
        # One projection makes keys and values: slices of its rows.
        spread = torch.rand((1, 1, dim), generator=gen, device='cuda') + 0.3
        kv = (torch.randn((sum(new), 2 * heads, dim), generator=gen,
                          device='cuda') * spread).to(dtype)
        state['k'], state['v'] = kv[:, :heads], kv[:, heads:]
        state['touched'] = torch.tensor(_touched(case), device='cuda').T
    return state


# ------------------------------------------------------------------- run --


def run(state):
    case = state['case']
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        return {'attention': _plain_attention, 'write': _plain_write,
                'read': _plain_read,
                'junction': _plain_junction}[case['kind']](state, case)


def _run_own(state, case):
    core, ops = _package()
    kind = case['kind']
    if kind == 'junction':
        out = ops.residual_norm(
            state['x'], state['residual'], state['weight'], state['bias'],
            gate=state['gate'], scale=_SCALE, post_norm=case['post'],
            post_weight=state['post_weight'], post_bias=state['post_bias'],
            rms=case['norm'] == 'rms', eps=_EPS)
        if not case['grad']:
            return list(out)
        inputs = [state[n] for n in _junction_inputs(state)]
        return [t.detach() for t in out] + list(torch.autograd.grad(
            out, inputs, (state['d_sum'], state['d_normed'])))
    if 'cache_object' not in state:
        state['cache_object'] = core.QuantizedCache(
            state['keys'], state['values'], state['key_exponents'],
            state['value_exponents'], case['dim'])
    cache = state['cache_object']
    if kind == 'attention':
        return [ops.cache_attention(
            state['q'], cache, offsets=state['offsets'],
            lengths=state['lengths'],
            left=None if case['left'] < 0 else case['left'],
            right=None if case['right'] < 0 else case['right'],
            sinks=case['sinks'])]
    if kind == 'read':
        return list(ops.read_cache(cache, lengths=state['lengths'],
                                   dtype=_DTYPES[case['dtype']]))
    ops.write_cache(cache, state['k'], state['v'], offsets=state['offsets'],
                    lengths=state['lengths'])
    return [cache.keys, cache.values, cache.key_exponents,
            cache.value_exponents]


def _junction_inputs(state):
    return [n for n in ('x', 'residual', 'weight', 'bias', 'gate',
                        'post_weight', 'post_bias') if state[n] is not None]


def _plain_norm(x, rms):
    """(normed rows, 1 / deviation)."""
    if not rms:
        x = x - x.mean(1, keepdim=True)
    root = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + _EPS)
    return x * root, root


def _plain_norm_grad(slope, normed, root, rms):
    along = (slope * normed).mean(1, keepdim=True)
    if not rms:
        slope = slope - slope.mean(1, keepdim=True)
    return (slope - normed * along) * root


def _plain_junction(state, case):
    dtype, rms = state['x'].dtype, case['norm'] == 'rms'
    x, residual = state['x'].float(), state['residual'].float()
    w, b, gate, post_w, post_b = (
        None if state[n] is None else state[n].float()
        for n in ('weight', 'bias', 'gate', 'post_weight', 'post_bias'))
    part = x
    if case['post']:
        before, post_root = _plain_norm(x, rms)
        part = before * post_w + (0.0 if post_b is None else post_b)
    factor = _SCALE if gate is None else gate * _SCALE
    total = (residual + part * factor).to(dtype)
    normed, root = _plain_norm(total.float(), rms)
    out = [total, (normed * w + (0.0 if b is None else b)).to(dtype)]
    if not case['grad']:
        return out
    dy = state['d_normed'].float()
    d_total = state['d_sum'].float() + _plain_norm_grad(dy * w, normed, root,
                                                        rms)
    d_part = d_total * factor
    grads = {'residual': d_total, 'weight': (dy * normed).sum(0),
             'bias': dy.sum(0), 'x': d_part,
             'gate': (d_total * part).sum(0) * _SCALE}
    if case['post']:
        grads['x'] = _plain_norm_grad(d_part * post_w, before, post_root, rms)
        grads['post_weight'] = (d_part * before).sum(0)
        grads['post_bias'] = d_part.sum(0)
    return out + [grads[n].to(dtype) for n in _junction_inputs(state)]


def _power(exponent):
    """2 ** exponent of whole numbers from -126 to 127, from its bits."""
    return ((exponent.int() + 127) << 23).view(torch.float32)


def _plain_write(state, case):
    _plain_append(state, case, state['k'], state['keys'].view(
        *state['key_exponents'].shape, _BLOCK, -1), state['key_exponents'])
    _plain_append(state, case, state['v'], state['values'].transpose(-1, -2),
                  state['value_exponents'])
    return [state['keys'], state['values'], state['key_exponents'],
            state['value_exponents']]


def _plain_append(state, case, x, codes, exponents):
    """``codes`` (sequences, heads, blocks, 32, width) and ``exponents``
    (sequences, heads, blocks) get the new rows ``x``."""
    seq, block = state['touched']
    offsets, lengths = state['offsets'].long(), state['lengths'].long()
    first = (lengths - (offsets[1:] - offsets[:-1]))[seq, None]
    place = block[:, None] * _BLOCK + torch.arange(_BLOCK, device=x.device)
    is_old = (place < first)[:, None, :, None]
    is_new = ((place >= first)
              & (place < lengths[seq, None]))[:, None, :, None]
    row = (offsets[seq, None] + place - first).clamp(0, len(x) - 1)
    rows = x[row].float().transpose(1, 2)  # (touched, heads, 32, dim)
    rows = torch.nn.functional.pad(rows, (0, codes.shape[-1] - rows.shape[-1]))
    rows = torch.where(is_new, rows, 0.0)
    is_int = case['code'] == 'int8'
    most = rows.abs().amax((-1, -2))
    mantissa, power = torch.frexp(most)
    power = power - (7 if is_int else 9)
    power = torch.where(mantissa <= (127 / 128 if is_int else 0.875), power,
                        power + 1)
    power = torch.where(most > 0, power.clamp(min=_LOW), _LOW)
    before = exponents[seq, :, block].int()
    power = torch.where(is_old[:, :, 0, 0],
                        torch.maximum(power, before), power)
    bits = codes.view(torch.uint8)
    kept = bits[seq, :, block]
    old = kept.view(codes.dtype).float()
    moved = _power((before - power).clamp(min=_LOW))[..., None, None]
    value = torch.where(is_new, rows * _power(-power)[..., None, None],
                        old * moved)
    if is_int:
        value = torch.round(value).clamp(-127, 127)
    bits[seq, :, block] = torch.where(
        is_new | is_old, value.to(codes.dtype).view(torch.uint8), kept)
    exponents[seq, :, block] = power.to(torch.int8)


def _plain_values(state, case):
    """The cache's keys and values, (sequences, heads, tokens, dim)."""
    shape = state['key_exponents'].shape
    keys = state['keys'].view(*shape, _BLOCK, -1).float()
    values = state['values'].transpose(-1, -2).float()
    return [(codes * _power(e)[..., None, None]).flatten(2, 3)[
        ..., :case['dim']] for codes, e in (
            (keys, state['key_exponents']), (values, state['value_exponents']))]


def _plain_read(state, case):
    filled = (torch.arange(_capacity(case), device='cuda')
              < state['lengths'][:, None])[:, None, :, None]
    return [torch.where(filled, t, 0.0).transpose(1, 2).to(
        _DTYPES[case['dtype']]).contiguous()
        for t in _plain_values(state, case)]


def _plain_attention(state, case):
    q, n, count = state['q'], case['batches'], case['q_len']
    heads, kv_heads, dim = case['heads'], case['kv_heads'], case['dim']
    group = heads // kv_heads
    keys, values = _plain_values(state, case)
    lengths = state['lengths'].long()
    position = (lengths[:, None] - count
                + torch.arange(count, device=q.device))[..., None]
    token = torch.arange(keys.shape[2], device=q.device)
    seen = token < lengths[:, None, None]
    if case['right'] >= 0:
        seen = seen & (token <= position + case['right'])
    if case['left'] >= 0:
        seen = seen & ((token >= position - case['left'])
                       | (token < case['sinks']))
    rows = q.float().view(n, count, kv_heads, group, dim).permute(
        0, 2, 3, 1, 4).reshape(n, kv_heads, group * count, dim)
    scores = (rows @ keys.transpose(-1, -2)).view(
        n, kv_heads, group, count, -1) * dim ** -0.5
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = scores.sum(-1, keepdim=True)
    shares = scores / torch.where(total == 0, 1.0, total)
    out = shares.view(n, kv_heads, group * count, -1) @ values
    return [out.view(n, kv_heads, group, count, dim).permute(
        0, 3, 1, 2, 4).reshape(n * count, heads, dim).to(q.dtype)]


# ------------------------------------------------------------------ work --


def work(case):
    size = _BYTES[case['dtype']]
    if case['kind'] == 'junction':
        values = case['rows'] * case['channels']
        arrays = 8 if case['grad'] else 4
        vectors = 1 + (case['norm'] == 'layer') + case['gate'] + case['post']
        vectors += case['post'] and case['norm'] == 'layer'
        return {'bytes': (arrays * values + vectors * case['channels']
                          * (2 if case['grad'] else 1)) * size,
                'flops': values * (12 + 8 * case['post'])
                * (3 if case['grad'] else 1)}
    new, total = _lengths(case)
    row = case['kv_heads'] * case['dim']
    if case['kind'] == 'write':
        rows = sum(new)
        blocks = len(_touched(case)) * case['kv_heads']
        return {'bytes': 2 * rows * row * (size + 1) + 2 * blocks,
                'flops': 6 * rows * row}
    if case['kind'] == 'read':
        blocks = sum(-(-t // _BLOCK) for t in total) * case['kv_heads']
        return {'bytes': 2 * sum(total) * row + 2 * blocks
                + 2 * case['batches'] * _capacity(case) * row * size,
                'flops': 2 * sum(total) * row}
    pairs = touched = 0
    for count, tokens in zip(new, total):
        p = np.arange(count, dtype=np.int64) + tokens - count
        left = tokens if case['left'] < 0 else case['left']
        right = tokens if case['right'] < 0 else case['right']
        lo, hi = np.maximum(0, p - left), np.minimum(tokens - 1, p + right)
        pairs += int((hi - lo + 1 + np.minimum(case['sinks'], lo)).sum())
        touched += int(hi[-1] - lo[0] + 1 + min(case['sinks'], lo[0]))
    of_q = sum(new) * case['heads'] * case['dim'] * size
    return {'bytes': 2 * of_q + 2 * touched * row
            + touched // _BLOCK * 2 * case['kv_heads'],
            'flops': 4 * pairs * case['heads'] * case['dim']}


# ----------------------------------------------------------------- exact --


def exact(case, seed):
    """The outputs of ``run`` in float64, from the definitions."""
    state = prepare(case, seed)
    with torch.no_grad():
        return {'attention': _exact_attention, 'write': _exact_write,
                'read': _exact_read,
                'junction': _exact_junction}[case['kind']](state, case)


def _exact_normed(x, rms):
    if rms:
        return x * torch.rsqrt(x.square().mean(1, keepdim=True) + _EPS)
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    return (x - mean) / torch.sqrt(var + _EPS)


def _exact_junction(state, case):
    """The gradients through torch's own differentiation in float64."""
    rms, dtype = case['norm'] == 'rms', state['x'].dtype
    with torch.enable_grad():
        v = {n: state[n].detach().double().requires_grad_()
             for n in _junction_inputs(state)}
        part = v['x']
        if case['post']:
            part = _exact_normed(part, rms) * v['post_weight']
            part = part + v.get('post_bias', 0.0)
        total = v['residual'] + _SCALE * v.get('gate', 1.0) * part
        # The norm is that of the sum as it is returned.
        rounded = total + (total.to(dtype).double() - total).detach()
        normed = _exact_normed(rounded, rms) * v['weight'] + v.get('bias', 0.0)
        out = [total.detach(), normed.detach()]
        if case['grad']:
            out += torch.autograd.grad(
                (total, normed), list(v.values()),
                (state['d_sum'].double(), state['d_normed'].double()))
    return out


def _exact_decoded(state, case, b, tokens):
    """The first ``tokens`` keys and values of sequence ``b``, (heads, tokens,
    dim)."""
    blocks = -(-tokens // _BLOCK)
    keys = state['keys'][b, :, :blocks * _BLOCK].double()
    values = state['values'][b, :, :blocks].double().movedim(3, 2)
    values = values.reshape(keys.shape)

    def factor(exponents):
        return torch.exp2(exponents[b, :, :blocks].double()).repeat_interleave(
            _BLOCK, 1)[..., None]

    return [(codes * factor(e))[:, :tokens, :case['dim']]
            for codes, e in ((keys, state['key_exponents']),
                             (values, state['value_exponents']))]


def _exact_read(state, case):
    out = [torch.zeros((case['batches'], _capacity(case), case['kv_heads'],
                        case['dim']), dtype=torch.float64, device='cuda')
           for _ in range(2)]
    for b, tokens in enumerate(_lengths(case)[1]):
        for whole, part in zip(out, _exact_decoded(state, case, b, tokens)):
            whole[b, :tokens] = part.transpose(0, 1)
    return out


def _exact_rounded(x, is_int):
    """Half to even, to whole numbers or to four significant bits (steps of
    2 ** -9 below 2 ** -6)."""
    if is_int:
        return x.round()
    step = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3
    step = torch.exp2(step)
    return (x / step).round() * step


def _exact_write(state, case):
    is_int = case['code'] == 'int8'
    most_code = 127.0 if is_int else 448.0
    dim, heads = case['dim'], case['kv_heads']
    out = []
    for x, codes, exponents, transposed in (
            (state['k'], state['keys'], state['key_exponents'], False),
            (state['v'], state['values'], state['value_exponents'], True)):
        codes, exponents = codes.double(), exponents.double()
        tokens = (codes.movedim(4, 3).flatten(2, 3) if transposed
                  else codes).clone()
        at = 0
        for b, (new, total) in enumerate(zip(*_lengths(case))):
            start = total - new
            for block in range(start // _BLOCK, -(-total // _BLOCK)):
                lo, hi = block * _BLOCK, min(total, (block + 1) * _BLOCK)
                mid = max(lo, start)
                rows = x[at + mid - start:at + hi - start].double().movedim(
                    1, 0)
                most = rows.abs().amax((1, 2)).clamp(min=2.0 ** -149)
                power = torch.ceil(torch.log2(most / most_code))
                # The logarithm's own rounding.
                power += (most > most_code * torch.exp2(power)).double()
                power -= (most <= most_code * torch.exp2(power - 1)).double()
                power = power.clamp(min=_LOW)
                if mid > lo:
                    power = torch.maximum(power, exponents[b, :, block])
                    moved = torch.exp2(exponents[b, :, block] - power)
                    tokens[b, :, lo:mid] = _exact_rounded(
                        tokens[b, :, lo:mid] * moved[:, None, None], is_int)
                tokens[b, :, mid:hi, :dim] = _exact_rounded(
                    rows / torch.exp2(power)[:, None, None], is_int)
                exponents[b, :, block] = power
            at += new
        if transposed:
            tokens = tokens.view(len(tokens), heads, -1, _BLOCK,
                                 tokens.shape[-1]).movedim(3, 4)
        out.append((tokens.contiguous(), exponents))
    codes = [c.to(torch.int8) if is_int else c for c, _ in out]
    return codes + [e.to(torch.int8) for _, e in out]


def _exact_attention(state, case):
    """Sequence by sequence and key head by key head, some queries at a time."""
    count, dim = case['q_len'], case['dim']
    group = case['heads'] // case['kv_heads']
    q = state['q'].double()
    out = torch.zeros_like(q)
    for b, tokens in enumerate(_lengths(case)[1]):
        keys, values = _exact_decoded(state, case, b, tokens)
        index = torch.arange(tokens, device=q.device)
        for at in range(0, count, 512):
            end = min(count, at + 512)
            pos = torch.arange(at, end, device=q.device)[:, None] + (
                tokens - count)
            hidden = torch.zeros((end - at, tokens), dtype=torch.bool,
                                 device=q.device)
            if case['right'] >= 0:
                hidden |= index > pos + case['right']
            if case['left'] >= 0:
                hidden |= (index < pos - case['left']) & (index
                                                          >= case['sinks'])
            rows = slice(b * count + at, b * count + end)
            for g in range(case['kv_heads']):
                own_heads = slice(g * group, (g + 1) * group)
                scores = q[rows, own_heads].transpose(0, 1) @ keys[g].T
                scores = (scores / math.sqrt(dim)).masked_fill(hidden,
                                                               -math.inf)
                result = torch.softmax(scores, -1) @ values[g]
                out[rows, own_heads] = result.transpose(0, 1)
    return [out]
