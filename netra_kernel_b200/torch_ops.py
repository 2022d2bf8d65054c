"""``torch.library`` custom ops over the layer's C ABI, for serving stacks that call operators by name
(the role of the reference's SGLang custom-op registration, ``scripts/rocm/integrations/sglang/netra_gfx1151_sglang.py:1121-1311``).

    handle = register_layer(layer)                       # a RoutedMoELayer
    out = torch.ops.netra.moe_layer(hidden, handle)      # router + top-8 inside
    out = torch.ops.netra.moe_apply(hidden, topk_weights, topk_ids, handle)   # the caller's top-k

A handle is a small integer naming a live layer object of this process; ``release_layer`` drops it.
Both ops run on torch's current stream through ``libnetra_sm100.so`` and have fake (meta) kernels, so
they can sit inside traced graphs; there is no CPU implementation.

    y = torch.ops.netra.fp8_linear(x, weight, weight_scale)                    # dense.fp8_linear, with its gradient
    counts = torch.ops.netra.expert_counts(topk_ids, 256, token_mask)          # balance.expert_counts
    loss = torch.ops.netra.balance_loss(logits, counts, token_mask)            # balance.balance_loss, with its gradient

Bring-up modes (the role of the reference's ``SGLANG_NETRA_ENGINE_MODE`` shadow / compare modes,
``docs/compiler/validation.md:187-193``), chosen by the environment variable ``NETRA_ENGINE_MODE`` when a layer is
registered with its row-major weights (``register_layer(layer, shadow_weights=...)``):
``engine`` (default) runs the fused layer only; ``shadow`` also runs the slot-order per-kernel bridges on the layer's
own routing and records the comparison in ``last_comparison(handle)``; ``compare`` raises when the two disagree
beyond the layer tolerances.  Both extra modes synchronise and are meant for bring-up, not for serving.
"""
from __future__ import annotations

import torch

import os
from typing import Optional

_layers: dict[int, object] = {}
_shadow: dict[int, tuple] = {}
_comparisons: dict[int, dict] = {}
_next_handle = 1
MAX_ABS, REL_L2 = 2e-2, 5e-3          # BF16 output tolerances of the layer


def register_layer(layer, shadow_weights=None) -> int:
    """``shadow_weights`` = (w13, w13_scale, w2, w2_scale) in the checkpoint's row-major layout, on the GPU; needed only
    for the shadow / compare modes."""
    global _next_handle
    handle = _next_handle
    _next_handle += 1
    _layers[handle] = layer
    if shadow_weights is not None:
        _shadow[handle] = tuple(shadow_weights)
    return handle


def release_layer(handle: int) -> None:
    _layers.pop(handle, None)
    _shadow.pop(handle, None)
    _comparisons.pop(handle, None)


def last_comparison(handle: int):
    """{"max_abs", "rel_l2"} of the most recent shadow / compare call of this layer, or None."""
    return _comparisons.get(int(handle))


def _mode() -> str:
    mode = os.environ.get("NETRA_ENGINE_MODE", "engine")
    if mode not in ("engine", "shadow", "compare"):
        raise RuntimeError(f"NETRA_ENGINE_MODE must be engine, shadow or compare, not {mode!r}")
    return mode


def _check_against_bridges(handle: int, hidden: torch.Tensor, out: torch.Tensor) -> None:
    """Recompute the expert part with the slot-order bridge kernels from the layer's own routing and quantised rows."""
    from . import moe
    mode = _mode()
    if mode == "engine":
        return
    if handle not in _shadow:
        raise RuntimeError("netra: shadow / compare mode needs register_layer(layer, shadow_weights=...)")
    layer = _layers[handle]
    w13, w13_s, w2, w2_s = _shadow[handle]
    tokens = hidden.shape[0]
    torch.cuda.current_stream().synchronize()
    inter = layer.intermediates(tokens)
    pairs = tokens * 8
    a_fp8 = inter["a_fp8"][pairs:pairs + tokens].contiguous()
    a_scale = inter["a_scale"][pairs:pairs + tokens].contiguous()
    ids9, w9 = inter["topk_ids"].contiguous(), inter["topk_w"].contiguous()
    gate_up = moe.bridge_gate_up(a_fp8, a_scale, w13, w13_s, ids9)
    act, act_s = moe.bridge_silu_mul_quant(gate_up)
    ref = moe.bridge_down_reduce(act, act_s, w2, w2_s, w9, ids9)
    torch.cuda.current_stream().synchronize()
    d = out.float() - ref.float()
    result = {"max_abs": float(d.abs().max()), "rel_l2": float(d.norm() / ref.float().norm().clamp_min(1e-30))}
    _comparisons[handle] = result
    if mode == "compare" and (result["max_abs"] > MAX_ABS or result["rel_l2"] > REL_L2):
        raise RuntimeError(f"netra: fused layer and bridge path disagree: {result}")


def _lookup(handle: int):
    layer = _layers.get(int(handle))
    if layer is None:
        raise RuntimeError(f"netra: no registered layer with handle {handle}")
    return layer


@torch.library.custom_op("netra::moe_layer", mutates_args=(), device_types="cuda")
def moe_layer(hidden: torch.Tensor, handle: int) -> torch.Tensor:
    hidden = hidden.contiguous()
    out = _lookup(handle)(hidden)
    _check_against_bridges(int(handle), hidden, out)
    return out


@moe_layer.register_fake
def _(hidden: torch.Tensor, handle: int) -> torch.Tensor:
    return torch.empty_like(hidden)


@torch.library.custom_op("netra::moe_apply", mutates_args=(), device_types="cuda")
def moe_apply(hidden: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor, handle: int) -> torch.Tensor:
    hidden = hidden.contiguous()
    out = _lookup(handle).apply(hidden, topk_weights.contiguous(), topk_ids.contiguous())
    _check_against_bridges(int(handle), hidden, out)
    return out


@moe_apply.register_fake
def _(hidden: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor, handle: int) -> torch.Tensor:
    return torch.empty_like(hidden)


# The operators beside the layer (dense.py, balance.py) by name, for traced graphs.  Eager callers use the modules, which cost less
# per call.
@torch.library.custom_op("netra::fp8_linear", mutates_args=(), device_types="cuda")
def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor) -> torch.Tensor:
    from . import dense
    return dense.fp8_linear(x, weight, weight_scale)


@fp8_linear.register_fake
def _(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor) -> torch.Tensor:
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.custom_op("netra::fp8_linear_input_grad", mutates_args=(), device_types="cuda")
def fp8_linear_input_grad(grad: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor) -> torch.Tensor:
    from . import dense
    codes, scale = dense.quantize_rows(grad)
    out = dense.block_scaled_matmul(codes, scale, weight, weight_scale, transpose_weight=True, out_dtype=grad.dtype)
    return out.view(*grad.shape[:-1], weight.shape[1])


@fp8_linear_input_grad.register_fake
def _(grad: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor) -> torch.Tensor:
    return grad.new_empty((*grad.shape[:-1], weight.shape[1]))


def _keep_weight(ctx, inputs, output) -> None:
    ctx.save_for_backward(*inputs[1:])


def _linear_backward(ctx, grad):
    from . import abi
    abi.torch_binding().check_captured_backward()
    return torch.ops.netra.fp8_linear_input_grad(grad, *ctx.saved_tensors), None, None


fp8_linear.register_autograd(_linear_backward, setup_context=_keep_weight)


@torch.library.custom_op("netra::expert_counts", mutates_args=(), device_types="cuda")
def expert_counts(topk_ids: torch.Tensor, num_experts: int, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    from . import balance
    return balance.expert_counts(topk_ids, num_experts, token_mask)


@expert_counts.register_fake
def _(topk_ids: torch.Tensor, num_experts: int, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    return topk_ids.new_empty((num_experts,), dtype=torch.int32)


@torch.library.custom_op("netra::balance_loss", mutates_args=(), device_types="cuda")
def balance_loss(logits: torch.Tensor, counts: torch.Tensor, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    from . import balance
    return balance.balance_loss(logits, counts, token_mask)


@balance_loss.register_fake
def _(logits: torch.Tensor, counts: torch.Tensor, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    return logits.new_empty((), dtype=torch.float32)


@torch.library.custom_op("netra::balance_loss_grad", mutates_args=(), device_types="cuda")
def balance_loss_grad(upstream: torch.Tensor, logits: torch.Tensor, counts: torch.Tensor,
                      token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    from . import balance
    return balance.balance_loss_grad(upstream, logits, counts, token_mask)


@balance_loss_grad.register_fake
def _(upstream: torch.Tensor, logits: torch.Tensor, counts: torch.Tensor, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    return logits.new_empty(logits.shape)


def _keep_routing(ctx, inputs, output) -> None:
    logits, counts, ctx.has_mask = inputs[0], inputs[1], inputs[2] is not None
    ctx.save_for_backward(logits, counts, *([inputs[2]] if ctx.has_mask else []))


def _balance_backward(ctx, upstream):
    from . import abi
    abi.torch_binding().check_captured_backward()
    logits, counts, *mask = ctx.saved_tensors
    return torch.ops.netra.balance_loss_grad(upstream, logits, counts, mask[0] if ctx.has_mask else None), None, None


balance_loss.register_autograd(_balance_backward, setup_context=_keep_routing)
