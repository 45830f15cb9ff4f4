"""Plain float64 forms of the transformer operators, with a bound on how far a
result in a given type may be from them (test infrastructure).

Bounds follow from the arithmetic: results are rounded once to their type
(unit roundoff ``u``), sums are float32 (relative error far under 2^-16 of the
sum of the terms' magnitudes at these sizes), the attention's softmax shares
and their slopes may be rounded to the type before the matrix products, and
its ``delta`` is made from the rounded output."""

from __future__ import annotations

import math

import numpy as np
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11,
        torch.bfloat16: 2.0 ** -8}
FLOAT_SUM = 2.0 ** -16
# The smallest steps of the types, where values or products underflow.
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -24,
        torch.bfloat16: 1e-37}


def assert_within(got, want, bound, what=''):
    got = got.detach().cpu().double()
    want, bound = want.detach().cpu(), bound.detach().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = torch.isnan(got) == torch.isnan(want)
    assert same.all(), f'{what}: {int((~same).sum())} NaN differ'
    finite = torch.isfinite(want)
    assert (got[~finite & ~torch.isnan(want)]
            == want[~finite & ~torch.isnan(want)]).all(), what
    excess = ((got - want).abs() - bound)[finite]
    if excess.numel():
        worst = float(excess.max())
        assert worst <= 0, f'{what}: {worst:.3e} over the bound'


def layer_norm_f64(x, weight, bias, eps, dy=None, active=None):
    """(y, its bound) or, with ``dy``, (value, bound) of y, dx, dw and db."""
    u = UNIT[x.dtype]
    tiny = TINY[x.dtype]
    x64 = x.detach().cpu().double()
    n, c = x64.shape
    active = n if active is None else active
    w = (torch.ones(c, dtype=torch.float64) if weight is None
         else weight.detach().cpu().double())
    b = (torch.zeros(c, dtype=torch.float64) if bias is None
         else bias.detach().cpu().double())
    live = (torch.arange(n) < active).double()[:, None]
    x64 = torch.where(live > 0, x64, 0.0)
    mean = x64.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x64 - mean) ** 2).mean(1, keepdim=True) + eps)
    h = (x64 - mean) * rstd
    y = (h * w + b) * live
    # The mean's own rounding reaches every channel of the row.
    size = (x64.abs() + x64.abs().mean(1, keepdim=True)) * rstd
    near = FLOAT_SUM * (size * w.abs() + b.abs())
    y_bound = u * y.abs() + near + tiny
    if dy is None:
        return y, y_bound
    d = dy.detach().cpu().double()
    d = torch.where(live > 0, d, 0.0)
    g = d * w
    dx = rstd * (g - g.mean(1, keepdim=True)
                 - h * (g * h).mean(1, keepdim=True)) * live
    mags = rstd * (g.abs() + g.abs().mean(1, keepdim=True)
                   + size * (g.abs() * size).mean(1, keepdim=True))
    dw, db = (d * h).sum(0), d.sum(0)
    return [(y, y_bound), (dx, u * dx.abs() + FLOAT_SUM * mags + tiny),
            (dw, u * dw.abs() + FLOAT_SUM * (d.abs() * size).sum(0) + tiny),
            (db, u * db.abs() + FLOAT_SUM * d.abs().sum(0) + tiny)]


def philox_words(count, seed, offset):
    """The first ``count`` words, in Python's whole numbers."""
    out = []
    low = 0xFFFFFFFF
    for number in range((count + 3) // 4):
        c = [number & low, number >> 32, offset & low, offset >> 32 & low]
        k = [seed & low, seed >> 32 & low]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1],
                 a & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        out += c
    return np.array(out[:count], dtype=np.uint64)


def rotary_f64(x, positions, frequencies, dims, interleaved, sign=1.0):
    u, tiny = UNIT[x.dtype], TINY[x.dtype]
    x64 = x.detach().cpu().double()
    positions = positions.detach().cpu().double()
    frequencies = frequencies.detach().cpu()
    out = x64.clone()
    bound = torch.zeros_like(out)
    start = used = 0
    for axis, width in enumerate(dims):
        half = width // 2
        angle = sign * positions[:, axis, None] * frequencies[used:used + half]
        cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        at = torch.arange(half)
        first = start + (2 * at if interleaved else at)
        second = first + (1 if interleaved else half)
        a, b = x64[..., first], x64[..., second]
        out[..., first] = a * cos - b * sin
        out[..., second] = a * sin + b * cos
        # cos, sin and the products are float32: a few roundings of 2^-24.
        both = 2.0 ** -21 * (a.abs() + b.abs())
        bound[..., first] = u * out[..., first].abs() + both + tiny
        bound[..., second] = u * out[..., second].abs() + both + tiny
        start, used = start + width, used + half
    return out, bound


def visible(nq, nk, left, right, sinks):
    p = torch.arange(nq)[:, None] + nk - nq
    j = torch.arange(nk)[None]
    seen = torch.ones((nq, nk), dtype=torch.bool)
    if right is not None:
        seen &= j <= p + right
    if left is not None:
        seen &= (j >= p - left) | (j < sinks)
    return seen


def attention_f64(q, k, v, spans, left, right, sinks, scale, dy=None,
                  device='cpu'):
    """``spans``: (first query row, queries, first key row, keys) of each
    sequence.  A list of (value, bound): out, or out, dq, dk and dv.  What a
    query does not see is left out of its sums altogether."""
    u, tiny = UNIT[q.dtype], TINY[q.dtype]
    step = u + FLOAT_SUM
    q64, k64, v64 = (t.detach().to(device).double() for t in (q, k, v))
    heads, group = q64.shape[1], q64.shape[1] // k64.shape[1]
    grad = dy is not None
    zero = [torch.zeros_like(q64) for _ in range(4)]
    out, out_bound, dq, dq_bound = zero
    dk, dk_bound, dv, dv_bound = (torch.zeros_like(k64) for _ in range(4))
    d64 = dy.detach().to(device).double() if grad else None
    for q0, nq, k0, nk in spans:
        if not nq or not nk:
            continue
        seen = visible(nq, nk, left, right, sinks).to(device)
        for h in range(heads):
            g = h // group
            rows, keys = slice(q0, q0 + nq), slice(k0, k0 + nk)
            qq, kk, vv = q64[rows, h], k64[keys, g], v64[keys, g]

            def over(p, values):
                """p @ values over what is seen, without 0 * inf."""
                if torch.isfinite(values).all():
                    return p @ values
                return torch.where(seen[..., None], p[..., None] * values,
                                   0.0).sum(1)

            def under(p, values):
                if torch.isfinite(values).all() and torch.isfinite(p).all():
                    return p.T @ values
                return torch.where(seen[..., None],
                                   p[..., None] * values[:, None], 0.0).sum(0)

            scores = (qq @ kk.T) * scale
            scores = scores.masked_fill(~seen, -math.inf)
            p = torch.softmax(scores, 1).masked_fill(~seen, 0.0)
            # An error of the scores is a relative error of the shares.
            loose = step * (1 + ((qq.abs() @ kk.abs().T) * scale).masked_fill(
                ~seen, 0.0).nan_to_num(0, 0, 0).amax() * 2.0 ** -4)
            o = over(p, vv)
            out[rows, h] = o
            out_bound[rows, h] = (3 * loose * over(p, vv.abs())
                                  + u * o.abs() + 8 * tiny)
            if not grad:
                continue
            dd = d64[rows, h]
            dp = (dd @ vv.T).masked_fill(~seen, 0.0)
            delta = (dd * o).sum(1, keepdim=True)
            ds = (p * (dp - delta)).masked_fill(~seen, 0.0)
            size = p * ((dd.abs() @ vv.abs().T)
                        + (dd.abs() * o.abs()).sum(1, keepdim=True))
            # The shares' rounding, delta's, and the underflow of a slope.
            off = (3 * loose * size + 2 * tiny).masked_fill(~seen, 0.0)
            dq[rows, h] = over(ds, kk) * scale
            dq_bound[rows, h] = (over(off, kk.abs()) * scale
                                 + u * dq[rows, h].abs() + tiny)
            dk[keys, g] += under(ds, qq) * scale
            dk_bound[keys, g] += under(off, qq.abs()) * scale + tiny
            dv[keys, g] += under(p, dd)
            dv_bound[keys, g] += (3 * loose * under(p, dd.abs())
                                  + under(2 * tiny * seen.double(), dd.abs())
                                  + tiny)
    if not grad:
        return [(out, out_bound)]
    return [(out, out_bound), (dq, dq_bound), (dk, dk_bound + u * dk.abs()),
            (dv, dv_bound + u * dv.abs())]
