"""Mixture-of-experts layer over GGUF-quantised experts, for a few tokens.

Stands beside GGUFLinearMethod for the expert stacks of a model file. The reference serves them from
plugin/vllm_gguf_plugin/quantization/fused_moe.py on its stock ops (ggml_moe_a8, ggml_moe_a8_vec), with routing, activation and
the weighted sum as kernels of their own; here the layer is one call.

  moe_layer_gguf(x, router_logits, w13, w2, ...)            from the router's logits on
  fused_moe_gguf(x, w13, w2, topk_weights, topk_ids, ...)   from given choices, as an expert-parallel rank calls it
  moe_route(router_logits, top_k, ...)                      the choice alone

Weights are uint8 in GGUF order (not repacked), any of the ten types: w13 [experts, 2 * inter, bytes of `hidden` values] with the
gate rows before the up rows, w2 [experts, hidden, bytes of `inter` values]; gguf_load.load_experts makes them from a file.
Activations are taken in 8 bits, 32 values to a 32-bit scale (the linear path's block_q8_1 has a 16-bit one). No derivative is computed: a call
that would need one is refused.
"""

from __future__ import annotations

import torch

from .. import _gsq_ops

ACTIVATIONS = {"silu": 0, "gelu": 1}
SCORINGS = {"softmax": 0, "sigmoid": 1}


def _direct(x: torch.Tensor) -> bool:
    """A plain CUDA tensor and nobody compiling or intercepting: straight to the native code under the custom ops, which goes back to
    the op where torch.func or a jit trace has to see it."""
    return type(x) is torch.Tensor and x.is_cuda and not torch.compiler.is_compiling() and not torch._C._len_torch_dispatch_stack()


def _code(table: dict, name: str, what: str) -> int:
    if name not in table:
        raise ValueError(f"unsupported {what} {name!r}: expected one of {sorted(table)}")
    return table[name]


def fused_moe_gguf(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor, w13_type: int,
                   w2_type: int, activation: str = "silu") -> torch.Tensor:
    """y [tokens, hidden] = sum over a token's choices of weight * W2[id] (act(gate) * up). topk_ids int32 or int64 [tokens, top_k];
    an id outside [0, experts) is another rank's expert and adds nothing."""
    act = _code(ACTIVATIONS, activation, "activation")
    return (_gsq_ops.moe_experts if _direct(x) else torch.ops._C_gguf.gsq_moe_experts)(x, w13, w2, topk_weights, topk_ids, w13_type, w2_type, act)


def moe_route(router_logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", renormalize: bool = True, bias: torch.Tensor | None = None,
              scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(weights fp32, ids int32), both [tokens, top_k]: the experts of largest score (score + bias [experts] where given), ties to the
    lowest number. An expert whose logit, or score + bias, is -inf or NaN is never chosen; a choice that finds none left has id -1, weight 0.
    Scores are 32-bit: a sigmoid of a logit below -88 is 0, and where all chosen scores are 0 so are the weights."""
    sc = _code(SCORINGS, scoring, "scoring")
    return (_gsq_ops.moe_route if _direct(router_logits) else torch.ops._C_gguf.gsq_moe_route)(router_logits, top_k, sc, renormalize, bias, scale)


def moe_layer_gguf(x: torch.Tensor, router_logits: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, w13_type: int, w2_type: int, top_k: int, *,
                   scoring: str = "softmax", renormalize: bool = True, bias: torch.Tensor | None = None, scale: float = 1.0,
                   activation: str = "silu") -> torch.Tensor:
    """moe_route and fused_moe_gguf in one call: y [tokens, hidden] in x's dtype."""
    act, sc = _code(ACTIVATIONS, activation, "activation"), _code(SCORINGS, scoring, "scoring")
    return (_gsq_ops.moe_layer if _direct(x) else torch.ops._C_gguf.gsq_moe_layer)(x, router_logits, w13, w2, w13_type, w2_type, top_k, sc, renormalize,
                                                                                     bias, scale, act)
