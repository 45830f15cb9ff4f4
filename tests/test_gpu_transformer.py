"""The transformer block's modules, and the example that trains and serves
with them."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
EXAMPLE = (Path(__file__).resolve().parent.parent / 'examples'
           / 'voxel_transformer.py')


def _example():
    spec = importlib.util.spec_from_file_location('voxel_transformer', EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _scans(channels, dtype=torch.float32):
    import mlx_lattice_amd.ops as ops

    generator = torch.Generator().manual_seed(3)
    example = _example()
    coords = [example.scan(n, generator).cuda() for n in (150, 1, 70)]
    feats = [torch.randn((len(c), channels), generator=generator).cuda().to(
        dtype) for c in coords]
    return ops.sparse_collate(coords, feats)


def _plain_block(block, x, drop):
    """The block in float64, row by row of torch's own operations."""
    def wide(t):
        return t.detach().double()

    def linear(conv, rows):
        return rows @ wide(conv.weight).flatten(1).T + wide(conv.bias)

    def norm(module, rows):
        return torch.nn.functional.layer_norm(
            rows, rows.shape[1:], wide(module.weight), wide(module.bias),
            module.eps)

    attention = block.attention
    heads, kv, dim = attention.heads, attention.kv_heads, attention.dim
    rows = wide(x.feats)
    packed = linear(attention.project, norm(block.norm1, rows)).view(
        len(rows), -1, dim)
    turned = packed.clone()
    start = used = 0
    for axis, width in enumerate(attention.dims):
        half = width // 2
        angle = wide(x.coords[:, 1 + axis])[:, None] * (
            attention._frequencies[used:used + half].to(rows.device))
        cos, sin = angle.cos()[:, None], angle.sin()[:, None]
        u = packed[:, :heads + kv, start:start + half]
        v = packed[:, :heads + kv, start + half:start + width]
        turned[:, :heads + kv, start:start + half] = u * cos - v * sin
        turned[:, :heads + kv, start + half:start + width] = u * sin + v * cos
        start, used = start + width, used + half
    k = turned[:, heads:heads + kv].repeat_interleave(heads // kv, 1)
    v = packed[:, heads + kv:].repeat_interleave(heads // kv, 1)
    scores = torch.einsum('ihd,jhd->hij', turned[:, :heads], k) / dim ** 0.5
    scan = x.coords[:, 0]
    place = torch.arange(len(rows), device=rows.device)
    first = torch.searchsorted(scan.contiguous(), scan.contiguous())
    local = place - first
    seen = (scan[:, None] == scan[None]) & (
        local[None] <= local[:, None] + attention.right) & (
        (local[None] >= local[:, None] - attention.left)
        | (local[None] < attention.sinks))
    share = torch.softmax(scores.masked_fill(~seen, -torch.inf), -1)
    mixed = torch.einsum('hij,jhd->ihd', share, v).reshape(len(rows), -1)
    rows = rows + drop(0, linear(attention.out, mixed))
    inner = torch.relu(linear(block.expand, norm(block.norm2, rows)))
    return rows + drop(1, linear(block.contract, inner))


def _close(got, want, relative):
    off = (got.double() - want).norm() / want.norm()
    assert off < relative, float(off)


# A chain of some twenty rounded operations: the type's roundoff times that.
@pytest.mark.parametrize('dtype, relative', [
    (torch.float32, 2e-5), (torch.float16, 2.0 ** -11 * 20),
    (torch.bfloat16, 2.0 ** -8 * 20)])
def test_block_matches_its_plain_form(dtype, relative):
    import mlx_lattice_amd.nn as lnn

    torch.manual_seed(0)
    x = _scans(48, dtype)
    block = lnn.VoxelTransformerBlock(48, 4, kv_heads=2, hidden=96, left=20,
                                      right=9, sinks=2, device='cuda',
                                      dtype=dtype).eval()
    _close(block(x).feats, _plain_block(block, x, lambda i, rows: rows),
           relative)


def test_block_trains_with_the_masks_of_its_counters():
    import mlx_lattice_amd.nn as lnn
    import mlx_lattice_amd.ops as ops

    torch.manual_seed(0)
    x = _scans(32)
    block = lnn.VoxelTransformerBlock(32, 2, left=30, right=30, sinks=1, p=0.3,
                                      seed=11, device='cuda')
    for parameter in block.parameters():
        parameter.requires_grad_()
    for step in range(2):
        def drop(index, rows, step=step):
            kept = ops.dropout(torch.ones_like(rows, dtype=torch.float32), 0.3,
                               seed=22 + index, offset=step)
            return rows * kept.double()

        out = block(x)
        _close(out.feats.detach(), _plain_block(block, x, drop), 2e-5)
    loss = (out.feats ** 2).sum()
    grads = torch.autograd.grad(loss, list(block.parameters()))
    # The loss along the gradients, by a step of the parameters.
    size = sum(float((g.double() ** 2).sum()) for g in grads) ** 0.5
    ends = []
    for sign in (1, -1):
        with torch.no_grad():
            for parameter, grad in zip(block.parameters(), grads):
                parameter += sign * 1e-3 * grad / size
        block.drop1.calls = block.drop2.calls = 1
        ends.append(float((block(x).feats.double() ** 2).sum()))
        with torch.no_grad():
            for parameter, grad in zip(block.parameters(), grads):
                parameter -= sign * 1e-3 * grad / size
    slope = (ends[0] - ends[1]) / 2e-3
    # Central differences over 1e-3: float32 values of the loss's size leave
    # about 1e-7 / 1e-3 of it, a ReLU's kinks and curvature less.
    assert abs(slope - size) < 2e-2 * size


def test_modules_follow_dtype_and_mode():
    import mlx_lattice_amd.nn as lnn

    x = _scans(24, torch.float16)
    block = lnn.VoxelTransformerBlock(24, 2, p=0.5, seed=1,
                                      device='cuda').half()
    assert block.attention._frequencies.dtype == torch.float64
    assert not torch.equal(block(x).feats, block(x).feats)
    block.eval()
    assert torch.equal(block(x).feats, block(x).feats)
    drop = lnn.Dropout(0.5, seed=4)
    first = drop(x).feats
    drop.calls = 0
    assert torch.equal(first, drop(x).feats)
    assert drop.eval()(x) is x


def test_attention_after_a_strided_conv():
    """A downsampled level: cells as coordinates, rows up to the active count,
    the scans found in the batch column."""
    import mlx_lattice_amd.nn as lnn
    import mlx_lattice_amd.ops as ops

    torch.manual_seed(1)
    x = _scans(16)
    down = lnn.Conv3d(16, 32, kernel_size=2, stride=2, device='cuda')(x)
    active = int(down.active_rows)
    assert active < down.capacity
    offsets = ops.batch_offsets(down, 3)
    scans = down.coords[:active, 0].tolist()
    assert scans == sorted(scans)
    assert offsets.tolist() == [sum(s < b for s in scans) for b in range(4)]
    layer = lnn.WindowAttention(32, 2, left=9, right=9, sinks=1,
                                device='cuda')
    got = layer(down, offsets=offsets).feats
    for scan in range(3):
        rows = slice(*offsets[scan:scan + 2].tolist())
        alone = ops.sparse_collate([down.coords[rows, 1:]], [down.feats[rows]])
        _close(got[rows], layer(alone).feats.double(), 2e-5)
    with pytest.raises(ValueError, match='positive'):
        ops.batch_offsets(down, 0)


def test_gradients_cannot_be_differentiated_again():
    """With create_graph the first gradients are as ever; a second
    differentiation says that it cannot."""
    import mlx_lattice_amd.ops as ops

    x = torch.randn((12, 2, 16), device='cuda', requires_grad=True)
    at = torch.tensor([0, 12], dtype=torch.int32, device='cuda')
    places = torch.arange(12, dtype=torch.int32, device='cuda')[:, None]
    frequencies = ops.rotary_frequencies((16,), device='cuda')
    for call in (lambda: ops.window_attention(x, x, x, offsets=at),
                 lambda: ops.rotary_positions(x, places, frequencies,
                                              dims=(16,)),
                 lambda: ops.layer_norm(x.view(12, 32)),
                 lambda: ops.dropout(x, 0.5, seed=1)):
        out = call()
        dy = torch.ones_like(out)
        plain, = torch.autograd.grad(call(), x, dy)
        kept, = torch.autograd.grad(out, x, dy, create_graph=True)
        assert torch.equal(plain, kept.detach())
        with pytest.raises(RuntimeError, match='differentiated once'):
            kept.square().sum().backward()


def test_only_the_gradients_asked_for():
    import mlx_lattice_amd.ops as ops

    x, y = (torch.randn((9, 8), device='cuda', requires_grad=True)
            for _ in range(2))
    w = torch.ones(8, device='cuda', requires_grad=True)
    out = ops.dropout(ops.layer_norm(x.detach(), w), 0.25, seed=2, residual=y)
    dw, dy = torch.autograd.grad(out.sum(), (w, y))
    assert dw.shape == w.shape and torch.equal(dy, torch.ones_like(y))
    ops.layer_norm(x, None, w).sum().backward()
    assert torch.equal(w.grad, torch.full_like(w, 9.0))


def test_refusals():
    import mlx_lattice_amd.nn as lnn

    with pytest.raises(ValueError, match='even number'):
        lnn.WindowAttention(30, 4)
    with pytest.raises(ValueError, match='multiple of the number'):
        lnn.WindowAttention(32, 4, kv_heads=3)
    with pytest.raises(ValueError, match='between 0 and 1'):
        lnn.Dropout(1.5, seed=0)


def test_example():
    example = _example()
    losses = example.train(steps=12)
    assert losses[-1] < losses[0]
    # Outputs of size one in bfloat16: two roundings of 2^-8, and the shares'.
    assert example.serve(rows=90) < 2.0 ** -5


def test_rows_too_wide_are_refused():
    """Rows of 2^32 values and some, whose count in 32 bits is the some."""
    import mlx_lattice_amd.ops as ops

    one = torch.zeros((1, 1, 1), dtype=torch.float16, device='cuda')
    many = 2 ** 32 + 8
    with pytest.raises(ValueError, match='too wide'):
        ops.layer_norm(one[0].expand(1, many))
    heads = one.expand(1, many, 8)
    places = torch.zeros((1, 1), dtype=torch.int32, device='cuda')
    with pytest.raises(ValueError, match='too wide'):
        ops.rotary_positions(heads, places,
                             ops.rotary_frequencies((8,), device='cuda'),
                             dims=(8,))
    at = torch.tensor([0, 1], dtype=torch.int32, device='cuda')
    with pytest.raises(ValueError, match='too wide'):
        ops.window_attention(heads, heads, heads, offsets=at)
    with pytest.raises(ValueError, match='too wide'):
        ops.window_attention(heads[:, :8], heads, heads, offsets=at)


@pytest.mark.parametrize('grad', (False, True))
def test_forward_mode_is_refused(grad):
    """A tangent of any input would be lost."""
    import torch.autograd.forward_ad as fwd

    import mlx_lattice_amd.ops as ops

    rows = torch.randn((12, 32), device='cuda', requires_grad=grad)
    heads = rows.view(12, 2, 16)
    weight = torch.ones(32, device='cuda')
    at = torch.tensor([0, 12], dtype=torch.int32, device='cuda')
    places = torch.arange(12., device='cuda')[:, None]
    frequencies = ops.rotary_frequencies((16,), device='cuda')
    for call, *inputs in (
            (ops.layer_norm, rows, weight, weight),
            (lambda x, r: ops.dropout(x, 0.5, seed=1, residual=r), rows, rows),
            (lambda x, p: ops.rotary_positions(x, p, frequencies, dims=(16,)),
             heads, places),
            (lambda q, k, v: ops.window_attention(q, k, v, offsets=at),
             heads, heads, heads)):
        plain = call(*inputs)
        with fwd.dual_level():
            assert torch.equal(call(*inputs), plain)
            for i, primal in enumerate(inputs):
                dual = fwd.make_dual(primal, torch.ones_like(primal))
                with pytest.raises(RuntimeError, match='forward-mode'):
                    call(*inputs[:i], dual, *inputs[i + 1:])
            if grad:
                dual = fwd.make_dual(plain.detach(), torch.ones_like(plain))
                with pytest.raises(RuntimeError, match='forward-mode'):
                    torch.autograd.grad(plain, rows, dual)
