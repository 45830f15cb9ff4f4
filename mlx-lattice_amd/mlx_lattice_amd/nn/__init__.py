from mlx_lattice_amd.nn.conv import (
    Conv3d,
    ConvTranspose3d,
    GenerativeConvTranspose3d,
    SubmConv3d,
)
from mlx_lattice_amd.nn.quantized_conv import (
    QuantizedConv3d,
    QuantizedConvTranspose3d,
    QuantizedGenerativeConvTranspose3d,
    QuantizedSubmConv3d,
)
from mlx_lattice_amd.nn.transformer import (
    Dropout,
    LayerNorm,
    VoxelTransformerBlock,
    WindowAttention,
)

__all__ = [
    'Conv3d',
    'ConvTranspose3d',
    'Dropout',
    'GenerativeConvTranspose3d',
    'LayerNorm',
    'QuantizedConv3d',
    'QuantizedConvTranspose3d',
    'QuantizedGenerativeConvTranspose3d',
    'QuantizedSubmConv3d',
    'SubmConv3d',
    'VoxelTransformerBlock',
    'WindowAttention',
]
