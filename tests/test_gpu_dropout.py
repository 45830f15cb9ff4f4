"""Counter-based dropout: its mask word for word, its gradient, its edges."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from transformer_reference import philox_words

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _ops():
    import mlx_lattice_amd.ops as ops

    return ops


def _mask(shape, p, seed, offset):
    words = philox_words(int(np.prod(shape)), seed, offset)
    return torch.from_numpy(words >= np.uint64(round(p * 2 ** 32))).reshape(
        shape)


def _want(x, p, seed, offset, residual=None):
    """One product and one sum in float32, rounded once: exact."""
    keep = _mask(x.shape, p, seed, offset)
    scale = np.float32(1 / (1 - p)) if p < 1 else np.float32(0)
    out = torch.where(keep, x.cpu().double() * float(scale), 0.0)
    if residual is None:
        return out.float().to(x.dtype)
    return out, residual.cpu().double()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', [(1, 1), (3, 1), (5, 7), (64, 30), (33, 64),
                                   (1000, 9)])
@pytest.mark.parametrize('p', (0.0, 0.1, 0.5, 0.999))
def test_mask_is_the_generators(shape, p, dtype):
    x = torch.randn(shape, device='cuda').to(dtype)
    seed, offset = 0x1234_5678_9ABC_DEF0, 0xFEDC_BA98_7654_3210
    got = _ops().dropout(x, p, seed=seed, offset=offset)
    assert torch.equal(got.cpu(), _want(x, p, seed, offset))


def test_words_are_those_of_the_paper():
    # The authors' known answer for a counter and key of zeros.
    assert [int(w) for w in philox_words(4, 0, 0)] == [
        0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize('dtype', DTYPES)
def test_residual_and_gradient(dtype):
    ops = _ops()
    x = torch.randn((129, 31), device='cuda').to(dtype).requires_grad_()
    r = torch.randn((129, 31), device='cuda').to(dtype).requires_grad_()
    dy = torch.randn((129, 31), device='cuda').to(dtype)
    out = ops.dropout(x, 0.25, seed=9, offset=4, residual=r)
    dx, dr = torch.autograd.grad(out, (x, r), dy)
    assert torch.equal(dx.cpu(), _want(dy, 0.25, 9, 4))
    assert torch.equal(dr, dy)
    part, rest = _want(x.detach(), 0.25, 9, 4, residual=r.detach())
    size = part.abs() + rest.abs()
    unit = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11,
            torch.bfloat16: 2.0 ** -8}[dtype]
    off = (out.detach().cpu().double() - (part + rest)).abs()
    assert (off <= (unit + 2.0 ** -23) * size + 2.0 ** -25).all()


def test_dropped_values_leave_no_trace():
    x = torch.full((64, 64), float('nan'), device='cuda')
    x[1::2] = float('inf')
    out = _ops().dropout(x, 0.5, seed=3)
    keep = _mask((64, 64), 0.5, 3, 0)
    assert (out.cpu()[~keep] == 0).all()
    assert (~torch.isfinite(out.cpu()[keep])).all()
    assert (_ops().dropout(x, 1.0, seed=3) == 0).all()


def test_strided_misaligned_and_empty():
    base = torch.randn((41, 66), device='cuda', dtype=torch.float16)
    for x in (base[:, 1:], base.t(), base[::3], base.reshape(-1)[1:],
              base[:0], base.reshape(41, 6, 11)):
        got = _ops().dropout(x, 0.3, seed=17, offset=1)
        assert got.shape == x.shape
        assert torch.equal(got.cpu(), _want(x, 0.3, 17, 1))


def test_places_past_32_bits():
    """The counter of an element past 2^34 has its high word set."""
    rows = (1 << 34) // 4096 + 2
    x = torch.ones((rows, 4096), dtype=torch.float16, device='cuda')
    got = _ops().dropout(x, 0.5, seed=5)
    tail = got.reshape(-1)[1 << 34:(1 << 34) + 64].cpu()
    del got, x
    torch.cuda.empty_cache()
    low = 0xFFFFFFFF
    for number in range(16):
        c, k = [number, 1, 0, 0], [5, 0]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1],
                 a & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        want = [2.0 if w >= 1 << 31 else 0.0 for w in c]
        assert tail[4 * number:4 * number + 4].tolist() == want


def test_share_and_independence():
    x = torch.ones((2000, 512), device='cuda')
    kept = [_ops().dropout(x, 0.2, seed=s, offset=o) > 0
            for s, o in ((1, 0), (1, 1), (2, 0))]
    for mask in kept:
        # Five standard deviations of a million draws.
        assert abs(float(mask.float().mean()) - 0.8) < 5 * 0.4 / 1012
    for a, b in ((0, 1), (0, 2), (1, 2)):
        both = float((kept[a] & kept[b]).float().mean())
        assert abs(both - 0.64) < 5 * 0.48 / 1012


def test_negative_and_large_seeds_wrap():
    x = torch.ones((8, 8), device='cuda')
    a = _ops().dropout(x, 0.5, seed=-1, offset=-2)
    b = _ops().dropout(x, 0.5, seed=2 ** 64 - 1, offset=2 ** 64 - 2)
    assert torch.equal(a, b)


def test_refusals():
    ops = _ops()
    x = torch.ones((4, 8), device='cuda')
    for p in (-0.1, 1.1, float('nan')):
        with pytest.raises(ValueError, match='between 0 and 1'):
            ops.dropout(x, p, seed=0)
    with pytest.raises(ValueError, match='shape of x'):
        ops.dropout(x, 0.1, seed=0, residual=x[:2])
    with pytest.raises(ValueError, match='share a dtype'):
        ops.dropout(x, 0.1, seed=0, residual=x.half())
    with pytest.raises(ValueError, match='float32, float16 or bfloat16'):
        ops.dropout(x.double(), 0.1, seed=0)
    with pytest.raises(ValueError, match='HIP device tensor'):
        ops.dropout(x.cpu(), 0.1, seed=0)
