"""Streamed scans through the transformer block's layers with an 8-bit cache:
writing, attending and joining as they are used together."""

from __future__ import annotations

import pytest
import torch
from cache_reference import decoded
from transformer_reference import assert_within, attention_f64

pytestmark = pytest.mark.gpu
CODES = (torch.float8_e4m3fn, torch.int8)


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _scans(gen, rows, channels, dtype, batches=2, start=0):
    """``rows`` successive voxels of each scan, with features."""
    import mlx_lattice_amd.ops as ops

    place = torch.arange(start, start + rows, device='cuda')
    coords = torch.stack([place // 64, place % 64, place * 7 % 64], 1).int()
    feats = [torch.randn((rows, channels), generator=gen, device='cuda').to(
        dtype) for _ in range(batches)]
    return ops.sparse_collate([coords] * batches, feats)


@pytest.mark.parametrize('code', CODES)
@pytest.mark.parametrize('dtype', (torch.float32, torch.bfloat16))
def test_steps_of_any_size_see_what_the_cache_holds(dtype, code):
    """A prompt, then single rows and pieces: each step's attention is that of
    its queries over the cache's values as they then are."""
    import mlx_lattice_amd.ops as ops

    gen = torch.Generator(device='cuda').manual_seed(0)
    heads, kv_heads, dim, total = 4, 2, 40, 0
    from mlx_lattice_amd import QuantizedCache

    cache = QuantizedCache.empty(2, 200, kv_heads, dim, dtype=code,
                                 device='cuda')
    lengths = torch.zeros(2, dtype=torch.int32, device='cuda')
    for rows in (70, 1, 1, 33, 1, 60, 1, 1, 1):
        total += rows
        packed = torch.randn((2 * rows, heads + 2 * kv_heads, dim),
                             generator=gen, device='cuda').to(dtype)
        lengths += rows
        at = _ints(0, rows, 2 * rows)
        q = packed[:, :heads]
        ops.write_cache(cache, packed[:, heads:heads + kv_heads],
                        packed[:, heads + kv_heads:], offsets=at,
                        lengths=lengths)
        out = ops.cache_attention(q, cache, offsets=at, lengths=lengths,
                                  left=64, right=0, sinks=4)
        flat = [t.reshape(-1, kv_heads, dim) for t in decoded(cache)]
        spans = [(s * rows, rows, s * cache.capacity, total)
                 for s in range(2)]
        want, bound = attention_f64(q, *flat, spans, 64, 0, 4, dim ** -0.5)[0]
        assert_within(out, want, bound, rows)
        # The same over rows that were read back.
        k, v = (t.view(-1, kv_heads, dim) for t in ops.read_cache(
            cache, lengths=lengths, dtype=dtype))
        again = ops.window_attention(
            q, k, v, offsets=at, key_lengths=lengths,
            key_offsets=_ints(0, cache.capacity, 2 * cache.capacity), left=64,
            right=0, sinks=4)
        assert_within(again, want, bound, rows)


@pytest.mark.parametrize('code', CODES)
def test_layer_with_a_cache_is_near_the_layer_without(code):
    """Row by row against the scans' single pass: off by the codes'
    rounding."""
    import mlx_lattice_amd.nn as lnn
    import mlx_lattice_amd.ops as ops

    torch.manual_seed(1)
    gen = torch.Generator(device='cuda').manual_seed(1)
    block = lnn.VoxelTransformerBlock(64, 4, kv_heads=2, left=32, right=0,
                                      sinks=2, device='cuda').eval()
    whole = _scans(gen, 60, 64, torch.float32)
    want = block(whole).feats.view(2, 60, 64)
    cache = block.attention.make_cache(2, 60, dtype=code)
    assert cache.capacity == 64 and cache.dtype == code
    feats = whole.feats.view(2, 60, 64)
    coords = whole.coords.view(2, 60, 4)
    lengths = torch.zeros(2, dtype=torch.int32, device='cuda')
    out = []
    at = 0
    for rows in (40,) + (1,) * 20:
        step = ops.sparse_collate(
            [c[at:at + rows, 1:] for c in coords],
            [f[at:at + rows] for f in feats])
        at += rows
        lengths += rows
        out.append(block(step, cache=cache, lengths=lengths).feats.view(
            2, rows, 64))
    got = torch.cat(out, 1)
    # A code is off by 2^-4 of its value (e4m3) or 2^-7 of the block's largest
    # (int8, at most half a step of 2^-6); scores and values are averages of
    # such errors, and the residual stream carries none.
    assert (got - want).norm() < 2.0 ** -4 * want.norm()


def test_layer_refuses_half_a_cache():
    import mlx_lattice_amd.nn as lnn

    gen = torch.Generator(device='cuda').manual_seed(2)
    layer = lnn.WindowAttention(32, 2, device='cuda')
    x = _scans(gen, 5, 32, torch.float32)
    with pytest.raises(ValueError, match='go together'):
        layer(x, cache=layer.make_cache(2, 64))
    with pytest.raises(ValueError, match='go together'):
        layer(x, lengths=_ints(5, 5))


def _gated(dtype, p=0.0):
    import mlx_lattice_amd.nn as lnn

    torch.manual_seed(3)
    block = lnn.VoxelTransformerBlock(
        64, 4, left=20, right=20, p=p, seed=5, layer_scale=0.5, device='cuda',
        dtype=dtype)
    with torch.no_grad():
        for gate in (block.gate1, block.gate2):
            gate += torch.randn_like(gate) * 0.2
    return block


# A chain of some twenty rounded operations: the type's roundoff times that.
@pytest.mark.parametrize('dtype, relative', [
    (torch.float32, 2e-5), (torch.float16, 2.0 ** -11 * 20),
    (torch.bfloat16, 2.0 ** -8 * 20)])
@pytest.mark.parametrize('p', (0.0, 0.3))
def test_gated_block(p, dtype, relative):
    """The block with gates against its parts one by one."""
    import mlx_lattice_amd.ops as ops

    gen = torch.Generator(device='cuda').manual_seed(3)
    x = _scans(gen, 90, 64, dtype)
    block = _gated(dtype, p)
    got = block(x).feats

    def drop(rows, index):
        kept = ops.dropout(torch.ones_like(rows, dtype=torch.float32), p,
                           seed=10 + index)
        return rows.double() * kept.double()

    mixed = block.attention(block.norm1(x)).feats
    stream = x.feats.double() + block.gate1.double() * drop(mixed, 0)
    normed = x.replace(feats=torch.nn.functional.layer_norm(
        stream, (64,), block.norm2.weight.double(), block.norm2.bias.double(),
        block.norm2.eps).to(dtype))
    inner = block.contract(block.expand(normed, activation='relu')).feats
    want = stream + block.gate2.double() * drop(inner, 1)
    assert (got.double() - want).norm() < relative * want.norm()


def test_gated_block_trains():
    """The loss along the gradients, by a step of the parameters, gates among
    them."""
    gen = torch.Generator(device='cuda').manual_seed(4)
    x = _scans(gen, 90, 64, torch.float32)
    block = _gated(torch.float32)
    parameters = list(block.parameters())
    assert any(p is block.gate1 for p in parameters)
    for parameter in parameters:
        parameter.requires_grad_()
    slope = torch.randn(x.feats.shape, generator=gen, device='cuda')

    def loss():
        return (block(x).feats.double() * slope).sum()

    grads = torch.autograd.grad(loss(), parameters)
    size = sum(float((g.double() ** 2).sum()) for g in grads) ** 0.5
    ends = []
    with torch.no_grad():
        for sign in (1, -2):
            for parameter, grad in zip(parameters, grads):
                parameter += sign * 1e-3 * grad / size
            ends.append(float(loss()))
    # Central differences over 1e-3: float32 values of the loss's size leave
    # about 1e-7 / 1e-3 of it, a ReLU's kinks and curvature less.
    assert abs((ends[0] - ends[1]) / 2e-3 - size) < 2e-2 * size


def test_block_without_gates_keeps_its_state():
    import mlx_lattice_amd.nn as lnn

    block = lnn.VoxelTransformerBlock(32, 2)
    assert not any('gate' in name for name in block.state_dict())
    gated = lnn.VoxelTransformerBlock(32, 2, layer_scale=1e-4)
    assert {name for name in gated.state_dict()} - {
        name for name in block.state_dict()} == {'gate1', 'gate2'}


def test_captured_step():
    """One step of a block and its cache in a graph: replays follow the
    lengths, which the graph counts up."""
    import mlx_lattice_amd.nn as lnn
    import mlx_lattice_amd.ops as ops

    torch.manual_seed(4)
    gen = torch.Generator(device='cuda').manual_seed(4)
    block = lnn.VoxelTransformerBlock(64, 4, kv_heads=2, left=48, right=0,
                                      device='cuda',
                                      dtype=torch.float16).eval()
    eager_cache, cache = (block.attention.make_cache(2, 128)
                          for _ in range(2))
    lengths = torch.zeros(2, dtype=torch.int32, device='cuda')
    at = _ints(0, 1, 2)
    x = _scans(gen, 1, 64, torch.float16)

    def step(cache):
        return block(x, offsets=at, cache=cache, lengths=lengths).feats

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lengths += 1
        out = step(cache)
    lengths.zero_()
    for part in cache.parts:
        part.view(torch.uint8).zero_()
    for index in range(70):
        x.feats.copy_(torch.randn(x.feats.shape, generator=gen,
                                  device='cuda'))
        x.coords[:, 1:] += 1
        graph.replay()
        assert lengths.tolist() == [index + 1] * 2
        assert torch.equal(out, step(eager_cache))
    for a, b in zip(cache.parts, eager_cache.parts):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    k, _ = ops.read_cache(cache, lengths=lengths)
    assert k[:, :70].any() and not k[:, 70:].any()


def test_two_captured_attentions_with_parts():
    """Calls whose tokens are split, in two graphs that replay in turn."""
    import mlx_lattice_amd.ops as ops
    from cache_reference import random_cache

    gen = torch.Generator(device='cuda').manual_seed(5)
    caches = [random_cache(gen, c, 2, 4096, 2, 64) for c in CODES]
    q = torch.zeros((2, 8, 64), device='cuda', dtype=torch.bfloat16)
    args = {'offsets': _ints(0, 1, 2), 'lengths': _ints(4096, 3001)}
    graphs = []
    for cache in caches:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.cache_attention(q, cache, **args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.cache_attention(q, cache, **args)
        graphs.append((graph, out))
    for _ in range(3):
        q.copy_(torch.randn(q.shape, generator=gen, device='cuda'))
        want = [ops.cache_attention(q, cache, **args) for cache in caches]
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, got), eager in zip(graphs, want):
            assert torch.equal(got, eager)
