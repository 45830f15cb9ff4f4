"""A cache of attention keys and values in 8 bits (no reference counterpart)."""

from __future__ import annotations

from dataclasses import dataclass

import torch

__all__ = ['QuantizedCache']

_CODES = (torch.float8_e4m3fn, torch.int8)
_BLOCK = 32


@dataclass(frozen=True, slots=True)
class QuantizedCache:
    """Keys and values of ``B`` sequences in one byte each, ``float8_e4m3fn``
    or ``int8``, with a power of two for each block of 32 tokens and key head:
    code ``c`` of a block with exponent ``e`` stands for ``c * 2 ** e``.

    ``keys`` has shape ``(B, kv_heads, capacity, width)``, ``width`` being the
    head's ``dim`` channels rounded up to 32 with zeros behind; ``values``
    ``(B, kv_heads, capacity / 32, width, 32)``, a block's tokens innermost, as
    the product with the attention's shares reads them; the exponents, int8,
    ``(B, kv_heads, capacity / 32)``.  How many tokens of a sequence are filled
    is its caller's to keep, on the device: ``lengths``.
    """

    keys: torch.Tensor
    values: torch.Tensor
    key_exponents: torch.Tensor
    value_exponents: torch.Tensor
    dim: int

    def __post_init__(self) -> None:
        if not 1 <= self.dim <= 128:
            raise ValueError(
                'cache heads must have between 1 and 128 channels.')
        if self.keys.dtype not in _CODES:
            raise ValueError('cache codes must be float8_e4m3fn or int8.')
        if self.keys.ndim != 4:
            raise ValueError('cache keys must have shape (B, kv_heads, '
                             'capacity, width).')
        batches, heads, capacity, width = self.keys.shape
        if heads < 1:
            raise ValueError('a cache must have a key head.')
        if capacity % _BLOCK:
            raise ValueError("a cache's capacity must be a multiple of 32.")
        if width != _rounded(self.dim):
            raise ValueError("cache rows must be the head's channels rounded "
                             'up to a multiple of 32.')
        blocks = capacity // _BLOCK
        if (self.values.dtype != self.keys.dtype
                or self.values.shape != (batches, heads, blocks, width,
                                         _BLOCK)):
            raise ValueError('cache values must have shape (B, kv_heads, '
                             "capacity / 32, width, 32) and the keys' dtype.")
        for exponents in (self.key_exponents, self.value_exponents):
            if (exponents.dtype != torch.int8
                    or exponents.shape != (batches, heads, blocks)):
                raise ValueError('cache exponents must have shape (B, '
                                 'kv_heads, capacity / 32) and int8 dtype.')
        for part in self.parts[1:]:
            if part.device != self.keys.device:
                raise ValueError('the parts of a cache must be on one device.')
        if not all(part.is_contiguous() for part in self.parts):
            raise ValueError('the parts of a cache must be contiguous.')

    @classmethod
    def empty(cls, batches: int, capacity: int, kv_heads: int, dim: int, *,
              dtype: torch.dtype = torch.float8_e4m3fn,
              device=None) -> QuantizedCache:
        """A cache of zeros for ``batches`` sequences of up to ``capacity``
        tokens (rounded up to whole blocks of 32)."""
        if batches < 0 or capacity < 0:
            raise ValueError('batches and capacity must be non-negative.')
        if dtype not in _CODES:
            raise ValueError('cache codes must be float8_e4m3fn or int8.')
        blocks, width = _rounded(capacity) // _BLOCK, _rounded(dim)

        def zeros(*shape):
            return torch.zeros((batches, kv_heads, *shape), dtype=torch.int8,
                               device=device)

        return cls(zeros(blocks * _BLOCK, width).view(dtype),
                   zeros(blocks, width, _BLOCK).view(dtype), zeros(blocks),
                   zeros(blocks), dim)

    @property
    def parts(self) -> tuple[torch.Tensor, ...]:
        return (self.keys, self.values, self.key_exponents,
                self.value_exponents)

    @property
    def batches(self) -> int:
        return int(self.keys.shape[0])

    @property
    def kv_heads(self) -> int:
        return int(self.keys.shape[1])

    @property
    def capacity(self) -> int:
        return int(self.keys.shape[2])

    @property
    def dtype(self) -> torch.dtype:
        return self.keys.dtype

    @property
    def device(self) -> torch.device:
        return self.keys.device

    @property
    def nbytes(self) -> int:
        return sum(part.numel() for part in self.parts)


def _rounded(count: int) -> int:
    return (count + _BLOCK - 1) // _BLOCK * _BLOCK
