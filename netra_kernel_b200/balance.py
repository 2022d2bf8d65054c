"""The router's load and the loss that keeps it even, for fine-tuning the router of a routed-MoE layer.

    counts = expert_counts(topk_ids, 256, token_mask)                 # int32 [256]
    loss = balance_loss(logits, counts, token_mask)                   # FP32 scalar, differentiable with respect to logits

With f = counts / sum counts and P_e the mean softmax probability of expert e over the counted tokens,
``loss = E * sum_e f_e * P_e``: 1 when both are even.  The counts carry no gradient; a data- or expert-parallel program adds
up the ranks' counts before it calls ``balance_loss``.  Calls enqueue on torch's current stream of the operands' device and may
be captured in a CUDA graph; results do not depend on the order in which blocks run.  There is no CPU implementation.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import abi
from .dense import _DTYPES, _on, _rows

MAX_EXPERTS = 1024


def _mask_ptr(token_mask: Optional[torch.Tensor], tokens: int, device: torch.device) -> Optional[int]:
    if token_mask is None:
        return None
    if token_mask.dtype != torch.bool or token_mask.device != device or tuple(token_mask.shape) != (tokens,) or not token_mask.is_contiguous():
        raise ValueError("token_mask must be a contiguous bool [tokens] tensor on the same device (True = counted)")
    return token_mask.data_ptr()


def expert_counts(topk_ids: torch.Tensor, num_experts: int, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``topk_ids`` int32 or int64 [tokens, slots] -> int32 [num_experts]: how often each expert was chosen by the tokens that
    ``token_mask`` (bool [tokens]) counts.  Ids outside 0..num_experts-1 are not counted, so the layer's nine-slot ids can be
    passed as they are: slot 8 holds the shared expert's id 256."""
    if not topk_ids.is_cuda or topk_ids.dtype not in (torch.int32, torch.int64) or topk_ids.dim() != 2:
        raise ValueError("topk_ids must be an int32 or int64 CUDA matrix [tokens, slots]")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts must be 1..{MAX_EXPERTS}")
    tokens, slots = topk_ids.shape
    mask = _mask_ptr(token_mask, tokens, topk_ids.device)
    if slots > 1 and topk_ids.stride(1) != 1 or tokens > 1 and topk_ids.stride(0) < slots:
        topk_ids = topk_ids.contiguous()
    counts = torch.empty(num_experts, dtype=torch.int32, device=topk_ids.device)
    with _on(topk_ids.device):
        abi.check(abi.load().netra_expert_counts_launch(
            counts.data_ptr(), topk_ids.data_ptr(), topk_ids.element_size(), max(topk_ids.stride(0), slots), mask, tokens, slots, num_experts,
            torch.cuda.current_stream(topk_ids.device).cuda_stream), "expert_counts_launch")
    return counts


def _forward(logits: torch.Tensor, counts: torch.Tensor, token_mask: Optional[torch.Tensor]):
    """(loss, E / counted tokens) of a matrix that _rows() has seen."""
    tokens, experts = logits.shape
    if tokens == 0:
        return torch.zeros((), dtype=torch.float32, device=logits.device), None
    lib = abi.load()
    size = lib.netra_balance_loss_workspace_bytes()
    loss = torch.empty((), dtype=torch.float32, device=logits.device)
    scale = torch.empty((), dtype=torch.float32, device=logits.device)
    workspace = torch.empty(size, dtype=torch.uint8, device=logits.device)
    with _on(logits.device):
        abi.check(lib.netra_balance_loss_launch(
            loss.data_ptr(), scale.data_ptr(), logits.data_ptr(), _DTYPES[logits.dtype], max(logits.stride(0), experts), counts.data_ptr(),
            None if token_mask is None else token_mask.data_ptr(), workspace.data_ptr(), size, tokens, experts,
            torch.cuda.current_stream(logits.device).cuda_stream), "balance_loss_launch")
    return loss, scale


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, counts, token_mask):
        rows = _rows(logits, "logits")
        loss, scale = _forward(rows, counts, token_mask)
        ctx.save_for_backward(rows, counts, token_mask, scale)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream):
        logits, counts, token_mask, scale = ctx.saved_tensors
        tokens, experts = logits.shape
        grad = torch.empty((tokens, experts), dtype=logits.dtype, device=logits.device)
        if tokens:
            upstream = upstream.contiguous()
            with _on(logits.device):
                abi.check(abi.load().netra_balance_loss_grad_launch(
                    grad.data_ptr(), experts, logits.data_ptr(), _DTYPES[logits.dtype], max(logits.stride(0), experts), counts.data_ptr(),
                    None if token_mask is None else token_mask.data_ptr(), scale.data_ptr(), upstream.data_ptr(), tokens, experts,
                    torch.cuda.current_stream(logits.device).cuda_stream), "balance_loss_grad_launch")
        return grad, None, None


def balance_loss(logits: torch.Tensor, counts: torch.Tensor, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``logits`` [tokens, E] (BF16, FP16 or FP32), ``counts`` int32 [E] -> FP32 scalar ``E * sum_e f_e * P_e``.

    Tokens that ``token_mask`` leaves out are not read and get a zero gradient; with no counted token, or no counts, the
    loss is 0.  A masked expert (logit -inf, or the type's lowest value) has probability 0; a row whose logits are all -inf
    counts as a token and contributes 0.  NaN and +inf in a counted row give NaN."""
    if not logits.is_cuda or logits.dim() != 2 or logits.dtype not in _DTYPES:
        raise ValueError("logits must be a BF16, FP16 or FP32 CUDA matrix [tokens, experts]")
    tokens, experts = logits.shape
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"experts must be 1..{MAX_EXPERTS}")
    if counts.dtype != torch.int32 or counts.device != logits.device or tuple(counts.shape) != (experts,) or not counts.is_contiguous():
        raise ValueError("counts must be a contiguous int32 [experts] tensor on the same device")
    _mask_ptr(token_mask, tokens, logits.device)
    if logits.requires_grad and torch.is_grad_enabled():
        return _BalanceLoss.apply(logits, counts, token_mask)
    return _forward(_rows(logits, "logits"), counts, token_mask)[0]
