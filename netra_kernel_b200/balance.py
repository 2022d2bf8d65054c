"""The router's load and the loss that keeps it even, for fine-tuning the router of a routed-MoE layer.

    counts = expert_counts(topk_ids, 256, token_mask)                 # int32 [256]
    loss = balance_loss(logits, counts, token_mask)                   # FP32 scalar, differentiable with respect to logits

With f = counts / sum counts and P_e the mean softmax probability of expert e over the counted tokens,
``loss = E * sum_e f_e * P_e``: 1 when both are even; up to ``MAX_EXPERTS`` experts.  The counts carry no gradient; a data- or
expert-parallel program adds up the ranks' counts before it calls ``balance_loss``.  Calls enqueue on torch's current stream of the
operands' device and may be captured in a CUDA graph (a backward pass not while an eager graph of one of its leaves, made on
the default stream, is alive: RuntimeError); results do not depend on the order in which blocks run.  There is no CPU
implementation.  Bad operands raise ValueError, operands that carry a forward-mode tangent NotImplementedError, failures of the C
ABI RuntimeError.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import abi

_ext = abi.torch_binding()

MAX_EXPERTS = 1024


def expert_counts(topk_ids: torch.Tensor, num_experts: int, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``topk_ids`` int32 or int64 [tokens, slots] -> int32 [num_experts]: how often each expert was chosen by the tokens that
    ``token_mask`` (bool [tokens]) counts.  Ids outside 0..num_experts-1 are not counted, so the layer's nine-slot ids can be
    passed as they are: slot 8 holds the shared expert's id 256."""
    return _ext.expert_counts(topk_ids, num_experts, token_mask)


def balance_loss(logits: torch.Tensor, counts: torch.Tensor, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``logits`` [tokens, E] (BF16, FP16 or FP32), ``counts`` int32 [E] -> FP32 scalar ``E * sum_e f_e * P_e``.

    Tokens that ``token_mask`` leaves out are not read and get a zero gradient; with no counted token, or no counts, the
    loss is 0.  A masked expert (logit -inf, or the type's lowest value) has probability 0; a row whose logits are all -inf
    counts as a token and contributes 0.  NaN and +inf in a counted row give NaN.  The gradient cannot be differentiated again: a
    second derivative raises RuntimeError."""
    return _ext.balance_loss(logits, counts, token_mask)


def balance_loss_grad(upstream: torch.Tensor, logits: torch.Tensor, counts: torch.Tensor, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``upstream`` (FP32 scalar tensor) times the gradient of ``balance_loss`` with respect to logits, without autograd."""
    return _ext.balance_loss_grad(upstream, logits, counts, token_mask)
