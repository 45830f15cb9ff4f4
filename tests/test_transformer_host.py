"""Host-side checks of the transformer operators that need no GPU: what the C
ABI refuses before it touches a device, its workspace sizes, and the argument
checks of the Python operators."""

from __future__ import annotations

import ctypes
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
LIB = ROOT / 'mlx-lattice_amd' / 'mlx_lattice_amd' / 'liblattice_hip.so'


class Attention(ctypes.Structure):  # lattice_attention
    _fields_ = (
        [(n, ctypes.c_int) for n in ('dtype', 'queries', 'keys', 'heads',
                                     'kv_heads', 'dim', 'sequences', 'left',
                                     'right', 'sinks')]
        + [('scale', ctypes.c_float)]
        + [(n, ctypes.c_void_p) for n in 'qkv']
        + [(n, ctypes.c_longlong) for n in (
            'q_row_stride', 'q_head_stride', 'k_row_stride', 'k_head_stride',
            'v_row_stride', 'v_head_stride')]
        + [(n, ctypes.c_void_p) for n in ('offsets', 'key_offsets',
                                          'key_lengths')])


def _library():
    lib = ctypes.CDLL(str(LIB))
    lib.lattice_hip_last_error.restype = ctypes.c_char_p
    for name in ('layer_norm_grad', 'window_attention',
                 'window_attention_grad'):
        getattr(lib, f'lattice_hip_{name}_workspace_bytes'
                ).restype = ctypes.c_size_t
    return lib


def _attention(**changes):
    values = dict(dtype=1, queries=8, keys=8, heads=4, kv_heads=2, dim=64,
                  sequences=1, left=4, right=0, sinks=0, scale=1.0, q=4096,
                  k=4096, v=4096, q_row_stride=256, q_head_stride=64,
                  k_row_stride=128, k_head_stride=64, v_row_stride=128,
                  v_head_stride=64, offsets=4096, key_offsets=4096,
                  key_lengths=None)
    values.update(changes)
    return Attention(**values)


@pytest.mark.parametrize('changes, message', [
    ({'dtype': 5}, b'float32, float16 and bfloat16'),
    ({'queries': -1}, b'2^29'),
    ({'keys': 1 << 29}, b'2^29'),
    ({'queries': 1 << 28, 'heads': 16, 'kv_heads': 16}, b'2^31'),
    ({'heads': 5}, b'multiple of the number of key heads'),
    ({'kv_heads': 0}, b'multiple of the number of key heads'),
    ({'dim': 136}, b'between 1 and 128'),
    ({'dim': 0}, b'between 1 and 128'),
    ({'left': -1}, b'non-negative'),
    ({'q': None}, b'non-null'),
    ({'offsets': None}, b'non-null'),
    ({'v': None}, b'non-null'),
    ({'dim': 60}, b'whole 16-byte pieces'),
    ({'k_row_stride': 129}, b'whole 16-byte pieces'),
    ({'k_row_stride': -128}, b'whole 16-byte pieces'),
    ({'q': 4098}, b'16-byte boundaries'),
    ({'v_row_stride': 1 << 21}, b'under 4 MiB'),
    ({'heads': 65536, 'q_row_stride': 256}, b'under 4 MiB'),
    ({'q_head_stride': 1 << 28}, b'within 512 MiB')])
def test_attention_refusals(changes, message):
    lib = _library()
    args = _attention(**changes)
    rc = lib.lattice_hip_window_attention(
        ctypes.byref(args), 4096, None, None, None, ctypes.c_size_t(0), None)
    assert rc == 1 and message in lib.lattice_hip_last_error()
    rc = lib.lattice_hip_window_attention_grad(
        ctypes.byref(args), 4096, None, 4096, 4096, 4096, 4096, 4096, None,
        ctypes.c_size_t(0), None)
    assert rc == 1 and message in lib.lattice_hip_last_error()
    assert lib.lattice_hip_window_attention_workspace_bytes(
        ctypes.byref(args)) == 0


def test_attention_workspaces():
    lib = _library()
    rc = lib.lattice_hip_window_attention(None, None, None, None, None,
                                          ctypes.c_size_t(0), None)
    assert rc == 1 and b'non-null' in lib.lattice_hip_last_error()
    # Enough rows of their own: no workspace.
    args = _attention(queries=100000, keys=100000)
    assert lib.lattice_hip_window_attention_workspace_bytes(
        ctypes.byref(args)) == 0
    # One query against many keys: parts of a float32 row and two states.
    args = _attention(queries=1, keys=100000, left=1 << 30)
    size = lib.lattice_hip_window_attention_workspace_bytes(ctypes.byref(args))
    assert size >= 2 * 4 * (64 * 4 + 8)
    rc = lib.lattice_hip_window_attention(
        ctypes.byref(args), 4096, None, None, 4096, ctypes.c_size_t(size - 1),
        None)
    assert rc == 1 and b'workspace' in lib.lattice_hip_last_error()
    size = lib.lattice_hip_window_attention_grad_workspace_bytes(
        ctypes.byref(args))
    assert size >= 4 * 8
    rc = lib.lattice_hip_window_attention_grad(
        ctypes.byref(args), 4096, None, 4096, 4096, 4096, 4096, 4096, 4096,
        ctypes.c_size_t(size - 1), None)
    assert rc == 1 and b'workspace' in lib.lattice_hip_last_error()


def test_row_operator_refusals():
    lib = _library()
    long, double = ctypes.c_longlong, ctypes.c_float

    def refused(rc, message):
        assert rc == 1 and message in lib.lattice_hip_last_error()

    refused(lib.lattice_hip_layer_norm(
        7, 4096, long(8), 1, 8, None, None, double(0), None, 4096, None,
        None), b'float32')
    refused(lib.lattice_hip_layer_norm(
        0, 4096, long(8), 1, 0, None, None, double(0), None, 4096, None,
        None), b'positive')
    refused(lib.lattice_hip_layer_norm(
        0, 4096, long(8), 1, 8, None, None, double(-1), None, 4096, None,
        None), b'eps')
    refused(lib.lattice_hip_layer_norm(
        0, None, long(8), 1, 8, None, None, double(0), None, 4096, None,
        None), b'non-null')
    size = lib.lattice_hip_layer_norm_grad_workspace_bytes(1000, 64)
    assert size > 0
    assert lib.lattice_hip_layer_norm_grad_workspace_bytes(0, 64) == 0
    refused(lib.lattice_hip_layer_norm_grad(
        0, 4096, long(64), 4096, long(64), 1000, 64, None, 4096, None, 4096,
        4096, 4096, 4096, ctypes.c_size_t(size - 1), None), b'workspace')
    word = ctypes.c_uint64
    refused(lib.lattice_hip_dropout(
        0, 4096, None, long(-1), word(0), word(0), word(0), double(1), 4096,
        None), b'non-negative')
    refused(lib.lattice_hip_dropout(
        0, 4096, None, long(1), word(0), word(0), word((1 << 32) + 1),
        double(1), 4096, None), b'2^32')
    refused(lib.lattice_hip_dropout(
        0, None, None, long(1), word(0), word(0), word(0), double(1), 4096,
        None), b'non-null')

    def rotary(*dims, axes=None, dim=32, pointer=4096):
        return lib.lattice_hip_rotary_positions(
            0, pointer, long(64), long(32), 2, 2, dim, 4096, 0, long(3), 4096,
            len(dims) if axes is None else axes,
            (ctypes.c_int32 * max(1, len(dims)))(*dims), 0, 0, 4096, None)

    refused(rotary(16, 18), b'fit the head')
    refused(rotary(15), b'even')
    refused(rotary(-2), b'even')
    refused(rotary(axes=0), b'between 1 and 4 axes')
    refused(rotary(2, axes=5), b'between 1 and 4 axes')
    refused(rotary(16, dim=1025), b'between 1 and 1024')
    refused(rotary(16, pointer=None), b'non-null')


def test_operators_refuse_host_tensors():
    import mlx_lattice_amd.ops as ops

    x = torch.zeros((3, 2, 8))
    at = torch.tensor([0, 3], dtype=torch.int32)
    with pytest.raises(ValueError, match='HIP device tensor'):
        ops.window_attention(x, x, x, offsets=at)
    with pytest.raises(ValueError, match='HIP device tensor'):
        ops.layer_norm(x.view(6, 8))
    with pytest.raises(ValueError, match='HIP device tensor'):
        ops.dropout(x, 0.5, seed=0)
    with pytest.raises(ValueError, match='HIP device tensor'):
        ops.rotary_positions(x, at[:, None].expand(2, 1)[:0].new_zeros((3, 1)),
                             ops.rotary_frequencies((8,)), dims=(8,))
    with pytest.raises(ValueError, match='even'):
        ops.rotary_frequencies((5,))


@pytest.mark.parametrize('shape', ((3, 2, 0), (3, 0), (0,), ()))
def test_attention_refuses_heads_without_channels(shape):
    """With the default scale, which has no value there."""
    import mlx_lattice_amd.ops as ops

    x = torch.zeros(shape)
    at = torch.tensor([0, 3], dtype=torch.int32)
    with pytest.raises(ValueError, match='attention heads must have|shape'):
        ops.window_attention(x, x, x, offsets=at)


def test_rotary_rows_of_too_many_values():
    lib = _library()
    long = ctypes.c_longlong
    rc = lib.lattice_hip_rotary_positions(
        0, 4096, long(64), long(32), 2, 1 << 26, 32, 4096, 0, long(3), 4096, 1,
        (ctypes.c_int32 * 1)(16), 0, 0, 4096, None)
    assert rc == 1 and b'2^31' in lib.lattice_hip_last_error()
