"""The attention layer and its block with an 8-bit cache: what goes into the
cache, what is seen of it, and that a block is its parts."""

from __future__ import annotations

import pytest
import torch
from cache_reference import decoded
from test_gpu_serving import _gated, _ints, _scans
from transformer_reference import assert_within, attention_f64

pytestmark = pytest.mark.gpu
CODES = (torch.float8_e4m3fn, torch.int8)


def _layer(dtype, **how):
    """A layer whose scores are far from equal and whose last product gives
    its rows as they are."""
    import mlx_lattice_amd.nn as lnn

    torch.manual_seed(7)
    layer = lnn.WindowAttention(64, 4, kv_heads=2, device='cuda', dtype=dtype,
                                **how)
    with torch.no_grad():
        layer.project.weight *= 8
        layer.out.weight.zero_()
        layer.out.weight[torch.arange(64), 0, 0, 0, torch.arange(64)] = 1
    return layer


def _projected(layer, x):
    """The layer's queries, keys and values, turned and not turned."""
    import mlx_lattice_amd.ops as ops

    packed = layer.project(x).feats.view(x.capacity, -1, layer.dim)
    turned = ops.rotary_positions(
        packed[:, :layer.heads + layer.kv_heads].contiguous(), x.coords[:, 1:],
        ops.rotary_frequencies(layer.dims, device='cuda'), dims=layer.dims)
    heads = layer.heads
    return (turned[:, :heads], turned[:, heads:],
            packed[:, heads + layer.kv_heads:],
            packed[:, heads:heads + layer.kv_heads])


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', (torch.float32, torch.float16))
def test_layer_writes_and_sees_its_own_keys(dtype, code):
    import mlx_lattice_amd.ops as ops
    from mlx_lattice_amd import QuantizedCache

    gen = torch.Generator(device='cuda').manual_seed(7)
    layer = _layer(dtype, left=24, right=0, sinks=2)
    cache = layer.make_cache(2, 160, dtype=code)
    own, unturned = (QuantizedCache.empty(2, 160, 2, 16, dtype=code,
                                          device='cuda') for _ in range(2))
    lengths = torch.zeros(2, dtype=torch.int32, device='cuda')
    total = 0
    for rows in (70, 1, 1, 45, 1):
        x = _scans(gen, rows, 64, dtype, start=total)
        total += rows
        lengths += rows
        at = _ints(0, rows, 2 * rows)
        got = layer(x, cache=cache, lengths=lengths).feats.view(-1, 4, 16)
        queries, keys, values, plain = _projected(layer, x)
        ops.write_cache(own, keys, values, offsets=at, lengths=lengths)
        ops.write_cache(unturned, plain, values, offsets=at, lengths=lengths)
        for a, b in zip(cache.parts, own.parts):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        spans = [(s * rows, rows, s * cache.capacity, total)
                 for s in range(2)]

        def wanted(held, left, sinks):
            flat = [t.reshape(-1, 2, 16) for t in decoded(held)]
            return attention_f64(queries, *flat, spans, left, 0, sinks,
                                 16 ** -0.5)[0]

        want, bound = wanted(own, 24, 2)
        # The last product is by ones and zeros: what it adds is float32's.
        bound = bound + 2.0 ** -20 * want.abs()
        assert_within(got, want, bound)
        # A layer without the first tokens, the window or the keys' rotation
        # would be outside the bound.  (Two tokens of 27 carry a far from equal
        # softmax of few rows, and the first rows see all there is: not each
        # single row tells.)
        if rows > 1:
            for other, _ in (wanted(own, 24, 0), wanted(own, None, 2),
                             wanted(unturned, 24, 2)):
                assert ((other - want).abs() > 4 * bound).any()


@pytest.mark.parametrize('gated', (False, True))
def test_block_with_a_cache_is_its_parts(gated):
    import mlx_lattice_amd.nn as lnn
    import mlx_lattice_amd.ops as ops

    gen = torch.Generator(device='cuda').manual_seed(8)
    if gated:
        block = _gated(torch.float16)
    else:
        torch.manual_seed(8)
        block = lnn.VoxelTransformerBlock(64, 4, left=20, right=20,
                                          device='cuda', dtype=torch.float16)
    block.eval()
    caches = [block.attention.make_cache(2, 96) for _ in range(2)]
    lengths = torch.zeros(2, dtype=torch.int32, device='cuda')
    for start, rows in ((0, 40), (40, 1), (41, 7)):
        x = _scans(gen, rows, 64, torch.float16, start=start)
        lengths += rows
        got = block(x, cache=caches[0], lengths=lengths).feats
        mixed = block.attention(block.norm1(x), cache=caches[1],
                                lengths=lengths)
        if gated:
            stream, normed = ops.residual_norm(
                mixed, x, block.norm2.weight, block.norm2.bias,
                gate=block.gate1, eps=block.norm2.eps)
            inner = block.contract(block.expand(normed, activation='relu'))
            want = torch.addcmul(stream.feats, inner.feats, block.gate2)
        else:
            stream = x.replace(feats=mixed.feats + x.feats)
            inner = block.contract(block.expand(block.norm2(stream),
                                                activation='relu'))
            want = inner.feats + stream.feats
        assert torch.equal(got, want)
        for a, b in zip(*(c.parts for c in caches)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
