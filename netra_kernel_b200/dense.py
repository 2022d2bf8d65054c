"""The dense block-scaled FP8 linear map of the compiler's dense contract, for the projections around the routed-MoE layer:
E4M3 weights with one FP32 scale per 128 x 128 block (a frozen checkpoint), activations quantised per token and 128
columns by the layer's own quantiser, FP32 accumulation, one rounding to the activations' type.

    codes, scale = quantize_rows(x)                                   # x [..., K] -> E4M3 [M, K], FP32 [M, ceil(K/128)]
    y = block_scaled_matmul(codes, scale, weight, weight_scale)       # [M, N]
    y = fp8_linear(x, weight, weight_scale)                           # both; differentiable with respect to x

Every call enqueues on torch's current stream of the operands' device and may be captured in a CUDA graph; nothing is kept
between calls.  There is no CPU implementation.
"""
from __future__ import annotations

import ctypes
from contextlib import nullcontext
from typing import Optional

import torch

from . import abi

BLOCK = 128
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _on(device: torch.device):
    """Makes ``device`` the current one for a launch (nothing to do in the usual case)."""
    return nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """``x`` as a matrix whose rows the kernels can walk: unit column stride, rows that do not overlap."""
    if not x.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what} must be bfloat16, float16 or float32")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{what} must have at least one column")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 and x.shape[1] > 1 or x.stride(0) < x.shape[1] and x.shape[0] > 1:
        x = x.contiguous()
    return x


def _check_weight(weight: torch.Tensor, weight_scale: torch.Tensor, device: torch.device) -> None:
    if weight.device != device or weight_scale.device != device:
        raise ValueError("weight and weight_scale must be on the activations' device")
    if weight.dtype != torch.float8_e4m3fn or weight.dim() != 2 or 0 in weight.shape:
        raise ValueError("weight must be float8_e4m3fn [N, K]")
    n, k = weight.shape
    if weight.stride(1) != 1 and k > 1 or weight.stride(0) % 16 or weight.stride(0) < k or weight.data_ptr() % 16:
        raise ValueError("weight rows must be contiguous and start on 16-byte boundaries")
    if weight_scale.dtype != torch.float32 or tuple(weight_scale.shape) != (-(-n // BLOCK), -(-k // BLOCK)):
        raise ValueError("weight_scale must be float32 [ceil(N/128), ceil(K/128)]")
    if weight_scale.stride(1) != 1 and weight_scale.shape[1] > 1 or weight_scale.stride(0) < weight_scale.shape[1] and weight_scale.shape[0] > 1:
        raise ValueError("weight_scale must be row-major")
    if weight.requires_grad or weight_scale.requires_grad:
        raise ValueError("the FP8 weight is frozen: it cannot require a gradient")


def quantize_rows(x: torch.Tensor):
    """``x`` [..., K] (BF16, FP16 or FP32) -> (E4M3 codes [M, K], FP32 scales [M, ceil(K/128)]), M the product of the leading
    sizes: ``scale = max(amax of the row's 128 columns, 1e-10) * fl(1/448)``, ``code = e4m3_rne_sat(x * fl(1/scale))``.
    The rows of the codes are padded to 16 bytes and the scales stored block by block, the forms the product reads best."""
    x = _rows(x, "x")
    m, k = x.shape
    blocks = -(-k // BLOCK)
    codes = torch.empty((m, -(-k // 16) * 16), dtype=torch.float8_e4m3fn, device=x.device)[:, :k]
    scale = torch.empty((blocks, m), dtype=torch.float32, device=x.device).t()
    if m:
        with _on(x.device):
            abi.check(abi.load().netra_dense_quantize_rows_launch(
                codes.data_ptr(), codes.stride(0), scale.data_ptr(), scale.stride(0), scale.stride(1), x.data_ptr(), _DTYPES[x.dtype],
                x.stride(0), m, k, torch.cuda.current_stream(x.device).cuda_stream), "dense_quantize_rows_launch")
    return codes, scale


def block_scaled_matmul(a: torch.Tensor, a_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                        transpose_weight: bool = False, out_dtype: torch.dtype = torch.bfloat16,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a`` [M, K] E4M3 with scales [M, ceil(K/128)] times a block-scaled weight: ``a @ weight.T`` [M, N] for ``weight``
    [N, K], or with ``transpose_weight`` ``a`` [M, N] times ``weight`` as it is stored -> [M, K]."""
    if not a.is_cuda or a.dtype != torch.float8_e4m3fn or a.dim() != 2:
        raise ValueError("a must be a float8_e4m3fn CUDA matrix")
    _check_weight(weight, weight_scale, a.device)
    m = a.shape[0]
    k, n = weight.shape if transpose_weight else weight.shape[::-1]
    if a.shape[1] != k:
        raise ValueError(f"a has {a.shape[1]} columns, the weight reduces over {k}")
    if a_scale.device != a.device or a_scale.dtype != torch.float32 or tuple(a_scale.shape) != (m, -(-k // BLOCK)):
        raise ValueError("a_scale must be float32 [M, ceil(K/128)] on a's device")
    if a.stride(1) != 1 and k > 1 or a.stride(0) % 16 and m > 1 or a.stride(0) < k and m > 1 or a.data_ptr() % 16:
        raise ValueError("the rows of a must be contiguous and start on 16-byte boundaries")
    if out is None:
        if out_dtype not in _DTYPES:
            raise ValueError("out_dtype must be bfloat16, float16 or float32")
        out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    elif out.device != a.device or out.dtype not in _DTYPES or tuple(out.shape) != (m, n) or out.stride(1) != 1 and n > 1 or out.stride(0) < n and m > 1:
        raise ValueError("out must be a row-major [M, N] matrix of BF16, FP16 or FP32 on a's device")
    if m:
        pitch = a.stride(0) if m > 1 else -(-k // 16) * 16
        with _on(a.device):
            abi.check(abi.load().netra_dense_fp8_matmul_launch(
                out.data_ptr(), _DTYPES[out.dtype], max(out.stride(0), n), a.data_ptr(), pitch, a_scale.data_ptr(), a_scale.stride(0),
                a_scale.stride(1), weight.data_ptr(), weight.stride(0), weight_scale.data_ptr(), max(weight_scale.stride(0), weight_scale.shape[1]),
                int(transpose_weight), m, weight.shape[0], weight.shape[1], torch.cuda.current_stream(a.device).cuda_stream),
                "dense_fp8_matmul_launch")
    return out


def _linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, transposed: bool) -> torch.Tensor:
    rows, cols = weight.shape
    k, n = (rows, cols) if transposed else (cols, rows)
    lead = x.shape[:-1]
    x = _rows(x, "x")
    m = x.shape[0]
    out = torch.empty((m, n), dtype=x.dtype, device=x.device)
    if m:
        lib = abi.load()
        size = lib.netra_dense_fp8_linear_workspace_bytes(m, k)
        workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
        with _on(x.device):
            abi.check(lib.netra_dense_fp8_linear_launch(
                out.data_ptr(), n, x.data_ptr(), _DTYPES[x.dtype], max(x.stride(0), k), weight.data_ptr(), weight.stride(0),
                weight_scale.data_ptr(), max(weight_scale.stride(0), weight_scale.shape[1]), int(transposed), m, rows, cols, workspace.data_ptr(), size,
                torch.cuda.current_stream(x.device).cuda_stream), "dense_fp8_linear_launch")
    return out if len(lead) == 1 else out.view(*lead, n)


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, weight_scale):
        ctx.save_for_backward(weight, weight_scale)
        return _linear(x, weight, weight_scale, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        weight, weight_scale = ctx.saved_tensors
        return _linear(grad, weight, weight_scale, True), None, None


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor) -> torch.Tensor:
    """``x`` [..., K] -> [..., N] in x's type (BF16, FP16 or FP32), through ``weight`` [N, K] E4M3 and ``weight_scale``
    [ceil(N/128), ceil(K/128)].  The rows of x are quantised in the call (``quantize_rows``).

    Differentiable with respect to x: the incoming gradient's rows are quantised the same way and multiplied by the weight as
    it is stored (``block_scaled_matmul(..., transpose_weight=True)``); the rounding of x to E4M3 passes gradients unchanged.
    The weight is frozen."""
    if x.dim() == 0 or x.shape[-1] != weight.shape[-1]:
        raise ValueError(f"x must have {weight.shape[-1]} columns")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    _check_weight(weight, weight_scale, x.device)
    if x.requires_grad and torch.is_grad_enabled():
        return _Fp8Linear.apply(x, weight, weight_scale)
    return _linear(x, weight, weight_scale, False)


def check_status(device: Optional[torch.device] = None) -> None:
    """Raises if a bounded wait inside a dense kernel of the device ran out (synchronises)."""
    words = (ctypes.c_uint32 * 4)()
    with torch.cuda.device(device) if device is not None else nullcontext():
        abi.check(abi.load().netra_dense_status(ctypes.byref(words)), "dense_status")
    if any(words):
        raise abi.NetraError(f"device status words {list(words)}: a bounded wait expired inside a dense FP8 product")
