"""The dense block-scaled FP8 linear map of the compiler's dense contract, for the projections around the routed-MoE layer:
E4M3 weights with one FP32 scale per ``BLOCK`` x ``BLOCK`` = 128 x 128 block (a frozen checkpoint), activations quantised per token
and 128 columns by the layer's own quantiser, FP32 accumulation, one rounding to the activations' type.  Sums repeat bit for bit;
K-blocks are added in ascending order except for few rows or few output tiles, which join several parts in a fixed order.

    codes, scale = quantize_rows(x)                                   # x [..., K] -> E4M3 [M, K], FP32 [M, ceil(K/128)]
    y = block_scaled_matmul(codes, scale, weight, weight_scale)       # [M, N]
    y = fp8_linear(x, weight, weight_scale)                           # both; differentiable with respect to x

Every call enqueues on torch's current stream of the operands' device and may be captured in a CUDA graph; nothing is kept
between calls.  A backward pass cannot be captured while an eager graph of one of its leaves, made on the default stream, is alive
(RuntimeError; an operand that is such a leaf is refused in the forward call, unless under ``torch.no_grad()``).  There is no CPU
implementation.  Sizes are up to 2^26; weights (and codes) need rows that are contiguous and start on 16-byte boundaries, so a
width that is no multiple of 16 is stored with padded rows; activations may have any strides.  Bad operands raise ValueError,
operands that carry a forward-mode tangent NotImplementedError, failures of the C ABI RuntimeError.
"""
from __future__ import annotations

import ctypes
from contextlib import nullcontext
from typing import Optional

import torch

from . import abi

_ext = abi.torch_binding()

BLOCK = 128


def quantize_rows(x: torch.Tensor):
    """``x`` [..., K] (BF16, FP16 or FP32) -> (E4M3 codes [M, K], FP32 scales [M, ceil(K/128)]), M the product of the leading
    sizes: ``scale = max(amax of the row's 128 columns, 1e-10) * fl(1/448)``, ``code = e4m3_rne_sat(x * fl(1/scale))``.
    The rows of the codes are padded to 128 bytes and the scales stored block by block, the forms the product reads best.
    A NaN stays at its element; an infinity makes its block's scale infinite.  Codes and scales carry no gradient."""
    return _ext.quantize_rows(x)


def block_scaled_matmul(a: torch.Tensor, a_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                        transpose_weight: bool = False, out_dtype: torch.dtype = torch.bfloat16,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a`` [M, K] E4M3 with scales [M, ceil(K/128)] times a block-scaled weight: ``a @ weight.T`` [M, N] for ``weight``
    [N, K], or with ``transpose_weight`` ``a`` [M, N] times ``weight`` as it is stored -> [M, K].  ``weight_scale`` is
    [ceil(N/128), ceil(K/128)] either way.  ``out`` (row-major, no memory of an operand) takes the result in its own type.  The
    product carries no gradient and refuses operands that require one, unless gradients are off."""
    return _ext.block_scaled_matmul(a, a_scale, weight, weight_scale, transpose_weight, out_dtype, out)


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor) -> torch.Tensor:
    """``x`` [..., K] -> [..., N] in x's type (BF16, FP16 or FP32), through ``weight`` [N, K] E4M3 and ``weight_scale``
    [ceil(N/128), ceil(K/128)].  The rows of x are quantised in the call (``quantize_rows``).

    Differentiable with respect to x: the incoming gradient's rows are quantised the same way and multiplied by the weight as
    it is stored (``block_scaled_matmul(..., transpose_weight=True)``); the rounding of x to E4M3 passes gradients unchanged.
    The weight is frozen.  The gradient cannot be differentiated again with respect to the incoming one: that raises
    RuntimeError."""
    return _ext.fp8_linear(x, weight, weight_scale)


def check_status(device: Optional[torch.device] = None) -> None:
    """Raises if a bounded wait inside a dense kernel of the device ran out.  Waits for all work enqueued on the device, on every
    stream; refused while a graph is being captured."""
    words = (ctypes.c_uint32 * 4)()
    with torch.cuda.device(device) if device is not None else nullcontext():
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("check_status waits for the device, which a stream that is being captured does not allow")
        abi.check(abi.load().netra_dense_status(ctypes.byref(words)), "dense_status")
    if any(words):
        raise abi.NetraError(f"device status words {list(words)}: a bounded wait expired inside a dense FP8 product")
