"""The scans of a sparse tensor for the attention over its rows."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rows(scans):
    column = torch.tensor(scans, dtype=torch.int32)
    coords = torch.stack([column, *(torch.arange(len(scans)).int(),) * 3], 1)
    return coords.cuda(), torch.randn(len(scans), 16).cuda()


@pytest.mark.parametrize('scans, active, want', [
    ([0] * 6, 6, [0, 6]), ([0] * 6, 4, [0, 4]), ([0] * 3 + [1] * 4, 7, [0, 3, 7]),
    ([0, 0, 2, 2, 2, 9], 5, [0, 2, 2, 5]), ([1, 1], 2, [0, 0, 2]),
    ([5, 5], 0, [0, 0]), ([], 0, [0, 0])])
def test_scans_are_found_in_the_batch_column(scans, active, want):
    import mlx_lattice_amd.ops as ops
    from mlx_lattice_amd import SparseTensor

    coords, feats = _rows(scans)
    x = SparseTensor(coords.view(-1, 4), feats, active_rows=torch.tensor(
        [active], dtype=torch.int32, device='cuda'))
    got = ops.batch_offsets(x)
    assert got.tolist() == want and got.dtype == torch.int32
    with pytest.raises(ValueError, match='positive'):
        ops.batch_offsets(x, 0)
    assert ops.batch_offsets(x, 1).tolist() == [0, active]


def test_rows_that_are_not_active_are_in_no_scan():
    import mlx_lattice_amd.ops as ops
    from mlx_lattice_amd import SparseTensor

    coords, feats = _rows([0, 0, 0, 1, 1, 1, 1])
    for active, want in ((7, [0, 3, 7]), (5, [0, 3, 5]), (2, [0, 2, 2])):
        x = SparseTensor(coords, feats, batch_counts=(3, 4),
                         active_rows=torch.tensor([active], dtype=torch.int32,
                                                  device='cuda'))
        assert ops.batch_offsets(x).tolist() == want


def test_a_strided_level_keeps_its_scans_apart():
    import mlx_lattice_amd.nn as lnn
    import mlx_lattice_amd.ops as ops

    torch.manual_seed(2)
    clouds = [torch.stack([torch.arange(n), torch.arange(n) * 3 % 50,
                           torch.arange(n) * 7 % 60], 1).int().cuda()
              for n in (200, 77, 130)]
    x = ops.sparse_collate(clouds, [torch.randn(len(c), 16).cuda()
                                    for c in clouds])
    down = lnn.Conv3d(16, 32, kernel_size=2, stride=2, device='cuda')(x)
    assert down.batch_counts is None
    layer = lnn.WindowAttention(32, 2, left=20, right=20, sinks=1,
                                device='cuda')
    want = layer(down, offsets=ops.batch_offsets(down, 3)).feats
    assert torch.equal(layer(down).feats, want)


def test_a_captured_graph_refuses_to_count(monkeypatch):
    import mlx_lattice_amd.ops as ops
    from mlx_lattice_amd import SparseTensor

    coords, feats = _rows([0, 1])
    x = SparseTensor(coords, feats)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing',
                        lambda: True)
    with pytest.raises(ValueError, match='captured graph'):
        ops.batch_offsets(x)
    assert ops.batch_offsets(x, 2).tolist() == [0, 1, 2]
    x = SparseTensor(coords, feats, batch_counts=(1, 1))
    with pytest.raises(ValueError, match='captured graph'):
        ops.batch_offsets(x)


def test_counts_reach_the_device_without_a_host_wait():
    import mlx_lattice_amd.nn as lnn
    import mlx_lattice_amd.ops as ops
    from mlx_lattice_amd import SparseTensor

    coords, feats = _rows([0] * 30 + [1] * 20)
    x = SparseTensor(coords, feats, batch_counts=(30, 20))
    layer = lnn.WindowAttention(16, 2, left=5, right=5, device='cuda')
    want = layer(x).feats
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode('error')
    try:
        offsets = [ops.batch_offsets(x) for _ in range(50)]
        got = layer(x).feats
    finally:
        torch.cuda.set_sync_debug_mode(0)
    assert all(o.tolist() == [0, 30, 50] for o in offsets)
    assert torch.equal(got, want)
