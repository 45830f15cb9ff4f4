"""Dropout layers' masks: passes that checkpointing makes again, seeds, and
states that are saved and loaded."""

from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint


def _masked(x, p, *, seed, offset, residual=None):
    """Stands in for the operator: a mask made from the two numbers."""
    generator = torch.Generator().manual_seed(seed % 2 ** 50 * 1000 + offset)
    mask = torch.rand(x.shape, generator=generator) >= p
    return x * mask / (1 - p) + (0 if residual is None else residual)


@pytest.fixture
def layers(monkeypatch):
    from mlx_lattice_amd.nn import transformer

    monkeypatch.setattr(transformer, 'dropout', _masked)
    return transformer


@pytest.mark.parametrize('reentrant', (False, True))
def test_a_pass_made_again_has_the_first_mask(layers, reentrant):
    torch.manual_seed(0)
    drop = layers.Dropout(0.5, seed=3)
    x = torch.randn(64, requires_grad=True)
    kept = [_masked(torch.ones(64), 0.5, seed=3, offset=i) for i in range(6)]
    for step in range(0, 6, 2):
        # Two passes, whose gradients are made in the opposite order.
        outs = [checkpoint(drop, x, use_reentrant=reentrant)
                for _ in range(2)]
        grads = [torch.autograd.grad(out.sum(), x)[0] if not reentrant
                 else _backward(out, x) for out in reversed(outs)]
        for i, (out, grad) in enumerate(zip(outs, reversed(grads))):
            assert torch.equal(out, x * kept[step + i])
            assert torch.equal(grad, kept[step + i])
    assert drop.calls == 6


def _backward(out, x):
    x.grad = None
    out.sum().backward()
    return x.grad.clone()


def test_passes_that_cannot_be_told_apart_are_refused(layers):
    x = torch.randn(8, requires_grad=True)
    drop = layers.Dropout(0.5, seed=3)
    out = checkpoint(drop, x, use_reentrant=False, preserve_rng_state=False)
    with pytest.raises(RuntimeError, match='earlier one'):
        out.sum().backward()
    outs = []
    for _ in range(2):
        torch.manual_seed(1)
        outs.append(checkpoint(drop, x, use_reentrant=False))
    with pytest.raises(RuntimeError, match='earlier one'):
        outs[0].sum().backward()
    # The same state with the same count is the same pass.
    drop = layers.Dropout(0.5, seed=3)
    for _ in range(2):
        torch.manual_seed(1)
        drop.calls = 0
        checkpoint(drop, x, use_reentrant=False).sum().backward()


def test_only_the_last_passes_are_kept(layers):
    drop = layers.Dropout(0.5, seed=3)
    x = torch.randn(1, requires_grad=True)
    first = checkpoint(drop, x, use_reentrant=False)
    for _ in range(4100):
        drop(x)
    assert len(drop._offsets) == 4096 and drop.calls == 4101
    with pytest.raises(RuntimeError, match='earlier one'):
        first.sum().backward()


def _blocks(layers, count=2, **kwargs):
    return [layers.VoxelTransformerBlock(8, 2, **kwargs) for _ in range(count)]


def test_layers_without_a_seed_draw_their_own(layers):
    torch.manual_seed(5)
    blocks = _blocks(layers, 3, p=0.1)
    seeds = [d.seed for b in blocks for d in (b.drop1, b.drop2)]
    assert len(set(seeds)) == 6
    torch.manual_seed(5)
    again = _blocks(layers, 3, p=0.1)
    assert seeds == [d.seed for b in again for d in (b.drop1, b.drop2)]
    given, = _blocks(layers, 1, p=0.1, seed=4)
    assert (given.drop1.seed, given.drop2.seed) == (8, 9)


def test_no_dropout_draws_nothing(layers):
    torch.manual_seed(5)
    want = torch.get_rng_state()
    drop = layers.Dropout(0.0)
    assert torch.equal(torch.get_rng_state(), want)
    x = torch.ones(4)
    assert drop(x) is x and torch.equal(torch.get_rng_state(), want)
    # Turned on later, in passes that are made again.
    drops = torch.nn.Sequential(drop, layers.Dropout(0.0))
    drops[0].p = drops[1].p = 0.5
    x.requires_grad_()
    out = checkpoint(drops, x, use_reentrant=False)
    grad, = torch.autograd.grad(out.sum(), x)
    assert torch.equal(grad, out.detach())
    assert drops[0].seed != drops[1].seed


def test_a_resumed_run_goes_on_with_the_masks(layers, tmp_path):
    x = torch.ones(64)
    torch.manual_seed(6)
    block, = _blocks(layers, 1, p=0.5)
    for _ in range(3):
        block.drop1(x)
    torch.save(block.state_dict(), tmp_path / 'state.pt')
    want = [block.drop1(x), block.drop2(x)]
    other, = _blocks(layers, 1, p=0.5)
    state = torch.load(tmp_path / 'state.pt', weights_only=True)
    other.load_state_dict(state)
    assert (other.drop1.calls, other.drop2.calls) == (3, 0)
    for a, b in zip(want, [other.drop1(x), other.drop2(x)]):
        assert torch.equal(a, b)
    # A seed that was given is the caller's; the count goes on.
    given, = _blocks(layers, 1, p=0.5, seed=2)
    given.load_state_dict(state)
    assert (given.drop1.seed, given.drop1.calls) == (4, 3)
    for seed in (-1, 2 ** 63 + 5, 2 ** 64 - 1, 2 ** 70 + 3):
        drop = layers.Dropout(0.5, seed=seed)
        fresh = layers.Dropout(0.5)
        fresh.load_state_dict(drop.state_dict())
        assert (fresh.seed - seed) % 2 ** 64 == 0


def test_states_without_masks_still_load(layers):
    block, other = _blocks(layers, p=0.5)
    state = {k: v for k, v in block.state_dict().items()
             if not k.endswith('_extra_state')}
    seed = other.drop1.seed
    other.load_state_dict(state)
    assert other.drop1.seed == seed
    assert torch.equal(other.expand.weight, block.expand.weight)
    with pytest.raises(RuntimeError, match='expand.weight'):
        other.load_state_dict({k: v for k, v in state.items()
                               if k != 'expand.weight'})


@pytest.mark.gpu
@pytest.mark.parametrize('reentrant', (False, True))
def test_checkpointed_block(reentrant):
    """The gradients of a stack of blocks with and without checkpoints."""
    import mlx_lattice_amd.nn as lnn
    import mlx_lattice_amd.ops as ops

    torch.manual_seed(0)
    places = torch.stack([torch.arange(300), torch.arange(300) % 7,
                          torch.arange(300) % 5], 1).int().cuda()
    x = ops.sparse_collate([places], [torch.randn(300, 32).cuda()])
    blocks = [lnn.VoxelTransformerBlock(32, 2, left=30, right=30, p=0.3,
                                        seed=i, device='cuda')
              for i in range(2)]
    parameters = [p.requires_grad_() for b in blocks for p in b.parameters()]
    grads = []
    for again in (False, True):
        feats = x.feats.clone().requires_grad_()
        for block in blocks:
            block.drop1.calls = block.drop2.calls = 0
        h = feats
        for block in blocks:
            def run(t, block=block):
                return block(x.replace(feats=t)).feats

            h = checkpoint(run, h, use_reentrant=reentrant) if again else run(h)
        for p in parameters:
            p.grad = None
        (h ** 2).sum().backward()
        grads.append([h.detach(), feats.grad, *(p.grad for p in parameters)])
        assert all(b.drop1.calls == 1 == b.drop2.calls for b in blocks)
    for a, b in zip(*grads):
        assert torch.equal(a, b)
