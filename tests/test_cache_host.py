"""Host-side checks of the 8-bit cache and the junction that need no GPU: what
the C ABI refuses before it touches a device, workspace sizes, and the
container's checks."""

from __future__ import annotations

import ctypes
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
LIB = ROOT / 'mlx-lattice_amd' / 'mlx_lattice_amd' / 'liblattice_hip.so'
int_, long_, void = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p


class Cache(ctypes.Structure):  # lattice_cache
    _fields_ = ([(n, int_) for n in ('code', 'sequences', 'kv_heads', 'blocks',
                                     'dim')]
                + [(n, void) for n in ('keys', 'values', 'key_exponents',
                                       'value_exponents')])


class Attention(ctypes.Structure):  # lattice_cache_attention
    _fields_ = ([(n, int_) for n in ('dtype', 'queries', 'heads', 'left',
                                     'right', 'sinks')]
                + [('scale', ctypes.c_float), ('q', void),
                   ('q_row_stride', long_), ('q_head_stride', long_),
                   ('offsets', void), ('lengths', void)])


class Junction(ctypes.Structure):  # lattice_residual_norm
    _fields_ = ([(n, int_) for n in ('dtype', 'rows', 'channels', 'rms',
                                     'post_norm')]
                + [('scale', ctypes.c_float), ('eps', ctypes.c_float)]
                + [(n, void) for n in ('x', 'residual')]
                + [(n, long_) for n in ('x_stride', 'residual_stride')]
                + [(n, void) for n in ('weight', 'bias', 'gate', 'post_weight',
                                       'post_bias', 'active_rows')])


def _library():
    lib = ctypes.CDLL(str(LIB))
    lib.lattice_hip_last_error.restype = ctypes.c_char_p
    for name in ('cache_attention', 'residual_norm_grad'):
        getattr(lib, f'lattice_hip_{name}_workspace_bytes'
                ).restype = ctypes.c_size_t
    return lib


def _cache(**changes):
    values = dict(code=0, sequences=2, kv_heads=2, blocks=4, dim=64, keys=4096,
                  values=4096, key_exponents=4096, value_exponents=4096)
    values.update(changes)
    return Cache(**values)


def _attention(**changes):
    values = dict(dtype=1, queries=8, heads=4, left=100, right=0, sinks=0,
                  scale=1.0, q=4096, q_row_stride=256, q_head_stride=64,
                  offsets=4096, lengths=4096)
    values.update(changes)
    return Attention(**values)


CACHE_FAULTS = [
    ({'code': 2}, b'e4m3 or int8'), ({'sequences': -1}, b'positive'),
    ({'kv_heads': 0}, b'positive'), ({'blocks': -1}, b'positive'),
    ({'blocks': 1 << 23}, b'2^28 tokens'), ({'sequences': 1 << 24}, b'2^24'),
    ({'kv_heads': 1 << 16}, b'2^16'), ({'dim': 0}, b'between 1 and 128'),
    ({'dim': 129}, b'between 1 and 128'), ({'keys': None}, b'non-null'),
    ({'value_exponents': None}, b'non-null'), ({'values': 4104}, b'16-byte')]


@pytest.mark.parametrize('changes, message', CACHE_FAULTS)
def test_cache_refusals(changes, message):
    lib = _library()
    cache = _cache(**changes)
    rc = lib.lattice_hip_cache_write(
        ctypes.byref(cache), 1, void(4096), long_(128), long_(64), void(4096),
        long_(128), long_(64), 8, void(4096), void(4096), None)
    assert rc == 1 and message in lib.lattice_hip_last_error()
    rc = lib.lattice_hip_cache_read(ctypes.byref(cache), 1, void(4096),
                                    void(4096), void(4096), None)
    assert rc == 1 and message in lib.lattice_hip_last_error()
    args = _attention()
    assert lib.lattice_hip_cache_attention_workspace_bytes(
        ctypes.byref(cache), ctypes.byref(args)) == 0
    rc = lib.lattice_hip_cache_attention(
        ctypes.byref(cache), ctypes.byref(args), void(4096), None,
        ctypes.c_size_t(0), None)
    assert rc == 1 and message in lib.lattice_hip_last_error()


def test_write_and_read_refusals():
    lib = _library()
    cache = _cache()

    def write(dtype=1, k=4096, k_stride=128, rows=8, offsets=4096,
              lengths=4096):
        return lib.lattice_hip_cache_write(
            ctypes.byref(cache), dtype, void(k), long_(k_stride), long_(64),
            void(4096), long_(128), long_(64), rows, void(offsets),
            void(lengths), None)

    for changes, message in (
            ({'dtype': 3}, b'float32, float16 or bfloat16'),
            ({'rows': -1}, b'2^29'), ({'rows': 1 << 29}, b'2^29'),
            ({'k_stride': -1}, b'non-negative'), ({'k': None}, b'non-null'),
            ({'offsets': None}, b'non-null'), ({'lengths': None}, b'non-null')):
        assert write(**changes) == 1, changes
        assert message in lib.lattice_hip_last_error()
    # Nothing to do: no pointer is needed.
    assert write(rows=0, k=None, offsets=None, lengths=None) == 0
    assert lib.lattice_hip_cache_write(None, 1, None, long_(0), long_(0), None,
                                       long_(0), long_(0), 0, None, None,
                                       None) == 1
    assert b'non-null' in lib.lattice_hip_last_error()
    for args, message in (((7, 4096, 4096), b'float32'),
                          ((1, None, 4096), b'non-null'),
                          ((1, 4096, None), b'non-null')):
        assert lib.lattice_hip_cache_read(
            ctypes.byref(cache), args[0], void(args[1]), void(args[2]),
            void(4096), None) == 1
        assert message in lib.lattice_hip_last_error()


@pytest.mark.parametrize('changes, message', [
    ({'dtype': 5}, b'float32, float16 and bfloat16'),
    ({'queries': -1}, b'2^28'), ({'queries': 1 << 28}, b'2^28'),
    ({'heads': 3}, b'multiple of the number of key heads'),
    ({'heads': 0}, b'multiple of the number of key heads'),
    ({'queries': 1 << 27, 'heads': 16}, b'2^31'),
    ({'left': -1}, b'non-negative'), ({'right': -1}, b'non-negative'),
    ({'sinks': -1}, b'non-negative'), ({'q': None}, b'non-null'),
    ({'offsets': None}, b'non-null'), ({'lengths': None}, b'non-null'),
    ({'q': 4104}, b'16-byte boundaries'),
    ({'q_row_stride': 260}, b'whole 16-byte pieces'),
    ({'q_head_stride': -64}, b'whole 16-byte pieces')])
def test_attention_refusals(changes, message):
    lib = _library()
    cache, args = _cache(), _attention(**changes)
    rc = lib.lattice_hip_cache_attention(
        ctypes.byref(cache), ctypes.byref(args), void(4096), None,
        ctypes.c_size_t(0), None)
    assert rc == 1 and message in lib.lattice_hip_last_error()
    assert lib.lattice_hip_cache_attention_workspace_bytes(
        ctypes.byref(cache), ctypes.byref(args)) == 0


def test_more_blocks_than_a_launch_has():
    lib = _library()
    message = b'too many sequences and heads'
    cache = _cache(sequences=1 << 23, kv_heads=(1 << 16) - 1)
    assert lib.lattice_hip_cache_write(
        ctypes.byref(cache), 1, void(4096), long_(128), long_(64), void(4096),
        long_(128), long_(64), 8, void(4096), void(4096), None) == 1
    assert message in lib.lattice_hip_last_error()
    assert lib.lattice_hip_cache_read(ctypes.byref(cache), 1, void(4096),
                                      void(4096), void(4096), None) == 1
    assert message in lib.lattice_hip_last_error()
    args = _attention(queries=1, heads=(1 << 16) - 1)
    assert lib.lattice_hip_cache_attention(
        ctypes.byref(cache), ctypes.byref(args), void(4096), None,
        ctypes.c_size_t(0), None) == 1
    assert message in lib.lattice_hip_last_error()


def test_attention_workspaces():
    lib = _library()
    cache = _cache(dim=60)
    args = _attention()
    rc = lib.lattice_hip_cache_attention(
        ctypes.byref(cache), ctypes.byref(args), void(4096), None,
        ctypes.c_size_t(0), None)
    assert rc == 1 and b'16-byte pieces' in lib.lattice_hip_last_error()
    # One query against many tokens: parts of a float32 row and its states.
    cache = _cache(sequences=1, blocks=4000)
    args = _attention(queries=1, left=1 << 30)
    size = lib.lattice_hip_cache_attention_workspace_bytes(
        ctypes.byref(cache), ctypes.byref(args))
    assert size >= 2 * 4 * (64 * 4 + 8)
    rc = lib.lattice_hip_cache_attention(
        ctypes.byref(cache), ctypes.byref(args), void(4096), void(4096),
        ctypes.c_size_t(size - 1), None)
    assert rc == 1 and b'workspace' in lib.lattice_hip_last_error()
    # Enough rows of their own: none.
    args = _attention(queries=1 << 20)
    assert lib.lattice_hip_cache_attention_workspace_bytes(
        ctypes.byref(cache), ctypes.byref(args)) == 0
    assert lib.lattice_hip_cache_attention(
        ctypes.byref(cache), None, void(4096), None, ctypes.c_size_t(0),
        None) == 1


def _junction(**changes):
    values = dict(dtype=1, rows=8, channels=64, rms=0, post_norm=0, scale=1.0,
                  eps=1e-5, x=4096, residual=4096, x_stride=64,
                  residual_stride=64)
    values.update(changes)
    return Junction(**values)


@pytest.mark.parametrize('changes, message', [
    ({'dtype': 9}, b'float32, float16 and bfloat16'),
    ({'rows': -1}, b'positive'), ({'channels': 0}, b'positive'),
    ({'x_stride': -64}, b'positive'), ({'channels': 1 << 26}, b'2^26'),
    ({'eps': -1.0}, b'non-negative'), ({'eps': float('nan')}, b'non-negative'),
    ({'x': None}, b'non-null'), ({'residual': None}, b'non-null')])
def test_junction_refusals(changes, message):
    lib = _library()
    args = _junction(**changes)
    rc = lib.lattice_hip_residual_norm(ctypes.byref(args), void(4096),
                                       void(4096), None, None)
    assert rc == 1 and message in lib.lattice_hip_last_error()
    pointers = [void(4096)] * 6 + [None] * 5
    rc = lib.lattice_hip_residual_norm_grad(
        ctypes.byref(args), *pointers, None, ctypes.c_size_t(0), None)
    assert rc == 1 and message in lib.lattice_hip_last_error()


def test_junction_workspaces_and_results():
    lib = _library()
    args = _junction()
    for results in ((None, 4096), (4096, None)):
        assert lib.lattice_hip_residual_norm(
            ctypes.byref(args), void(results[0]), void(results[1]), None,
            None) == 1
        assert b'non-null' in lib.lattice_hip_last_error()
    size = lib.lattice_hip_residual_norm_grad_workspace_bytes(8, 64)
    assert size >= 8 * 5 * 64 * 4
    assert lib.lattice_hip_residual_norm_grad_workspace_bytes(0, 64) == 0
    # Partial rows are bounded for wide rows.
    assert lib.lattice_hip_residual_norm_grad_workspace_bytes(
        1 << 20, 1 << 20) < 1 << 31

    def grad(vectors, workspace, bytes_):
        return lib.lattice_hip_residual_norm_grad(
            ctypes.byref(args), *[void(4096)] * 6, *vectors, workspace,
            ctypes.c_size_t(bytes_), None)

    weight = [void(4096)] + [None] * 4
    assert grad(weight, void(4096), size - 1) == 1
    assert b'workspace' in lib.lattice_hip_last_error()
    assert grad(weight, None, size) == 1
    assert grad([None] * 4 + [void(4096)], void(4096), size) == 1
    assert b'post_norm' in lib.lattice_hip_last_error()
    # No rows and no vectors: nothing is launched.
    args = _junction(rows=0, x=None, residual=None)
    assert grad([None] * 5, None, 0) == 0
    assert lib.lattice_hip_residual_norm(ctypes.byref(args), None, None, None,
                                         None) == 0


def test_junction_statistics_off_their_boundaries():
    lib = _library()
    args = _junction()
    for rc in (lib.lattice_hip_residual_norm(
            ctypes.byref(args), void(4096), void(4096), void(4104), None),
            lib.lattice_hip_residual_norm_grad(
                ctypes.byref(args), void(4096), void(4104),
                *[void(4096)] * 4, *[None] * 5, None, ctypes.c_size_t(0),
                None)):
        assert rc == 1
        assert b'16-byte boundaries' in lib.lattice_hip_last_error()


def test_cache_shapes():
    from mlx_lattice_amd import QuantizedCache

    for dtype in (torch.float8_e4m3fn, torch.int8):
        cache = QuantizedCache.empty(3, 50, 2, 80, dtype=dtype)
        assert cache.keys.shape == (3, 2, 64, 96)
        assert cache.values.shape == (3, 2, 2, 96, 32)
        assert cache.key_exponents.shape == (3, 2, 2)
        assert (cache.batches, cache.kv_heads, cache.capacity, cache.dim
                ) == (3, 2, 64, 80)
        assert cache.dtype == dtype and cache.device == torch.device('cpu')
        assert cache.nbytes == 2 * 3 * 2 * (64 * 96 + 2)
        assert not any(p.view(torch.uint8).any() for p in cache.parts)
    for args, message in (((-1, 5, 1, 8), 'non-negative'),
                          ((1, -5, 1, 8), 'non-negative'),
                          ((1, 5, 0, 8), 'key head'),
                          ((1, 5, 1, 0), 'between 1 and 128'),
                          ((1, 5, 1, 129), 'between 1 and 128')):
        with pytest.raises(ValueError, match=message):
            QuantizedCache.empty(*args)
    with pytest.raises(ValueError, match='float8_e4m3fn or int8'):
        QuantizedCache.empty(1, 5, 1, 8, dtype=torch.uint8)


def test_cache_refuses_parts_that_do_not_fit():
    from mlx_lattice_amd import QuantizedCache

    good = dict(zip(('keys', 'values', 'key_exponents', 'value_exponents'),
                    QuantizedCache.empty(2, 64, 2, 40).parts), dim=40)
    keys, values = good['keys'], good['values']
    assert QuantizedCache(**good).capacity == 64
    for changes, message in (
            ({'dim': 30}, 'rounded'), ({'dim': 200}, 'between 1 and 128'),
            ({'keys': keys.view(torch.uint8)}, 'float8_e4m3fn or int8'),
            ({'keys': keys[0]}, 'shape'),
            ({'keys': keys[:, :0]}, 'key head'),
            ({'keys': keys[:, :, :40]}, 'multiple of 32'),
            ({'values': values[:1]}, 'cache values'),
            ({'values': values.view(torch.int8)}, 'cache values'),
            ({'key_exponents': good['key_exponents'].int()}, 'int8 dtype'),
            ({'value_exponents': good['value_exponents'][:, :, :1]},
             'int8 dtype'),
            ({'values': values.transpose(3, 4).contiguous().transpose(3, 4)},
             'contiguous'),
            ({'key_exponents': good['key_exponents'].to('meta')},
             'one device')):
        with pytest.raises(ValueError, match=message):
            QuantizedCache(**{**good, **changes})


def test_operators_refuse_host_tensors():
    import mlx_lattice_amd.ops as ops
    from mlx_lattice_amd import QuantizedCache

    cache = QuantizedCache.empty(1, 64, 2, 8)
    x = torch.zeros((3, 2, 8))
    at = torch.tensor([0, 3], dtype=torch.int32)
    args = {'offsets': at, 'lengths': at[1:]}
    with pytest.raises(ValueError, match='HIP device tensor'):
        ops.write_cache(cache, x, x, **args)
    with pytest.raises(ValueError, match='HIP device tensor'):
        ops.read_cache(cache, lengths=at[1:])
    with pytest.raises(ValueError, match='HIP device tensor'):
        ops.cache_attention(x, cache, **args)
    with pytest.raises(ValueError, match='HIP device tensor'):
        ops.residual_norm(x.view(6, 8), x.view(6, 8))
