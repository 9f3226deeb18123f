"""Log probabilities of given tokens, with their rank, the entropy of the row and its most probable alternatives: what a server
answers with behind the head's product.

The reference leaves this to vLLM's sampler (log_softmax over the logits, a gather, a comparison and a topk, each over the whole
row); here it is one kernel that reads the logits once. No derivative is computed: a call that would need one is refused.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _gsq_ops
from .quantization.fused_moe import _direct


class TokenLogprobs(NamedTuple):
    """Of each row. A rank of 1 is the most probable token; equal logits rank by index (a sampler that counts all logits >= the token's
    gives a token behind equal ones, frequent in 16 bits, a larger rank)."""
    logprobs: torch.Tensor       # fp32 [rows]: natural log probability of the given token
    ranks: torch.Tensor          # int64 [rows]
    entropy: torch.Tensor        # fp32 [rows], in nats
    top_logprobs: torch.Tensor   # fp32 [rows, top_n], largest first
    top_ids: torch.Tensor        # int64 [rows, top_n]


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, top_n: int = 0) -> TokenLogprobs:
    """logits [rows, vocabulary] fp32, fp16 or bf16, any row stride; token_ids [rows] int32 or int64: negative = no token (log
    probability 0, rank 0), past the vocabulary = NaN, rank 0. top_n 0 .. 32. Masked logits are -inf."""
    return TokenLogprobs(*(_gsq_ops.token_logprobs if _direct(logits) else torch.ops._C_gguf.gsq_token_logprobs)(logits, token_ids, top_n))


def head_logprobs(method, layer: torch.nn.Module, x: torch.Tensor, token_ids: torch.Tensor, top_n: int = 0, *,
                  max_logit_bytes: int = 1 << 28) -> TokenLogprobs:
    """token_logprobs of method.apply(layer, x) (a GGUFLinearMethod and the head's layer), at most `max_logit_bytes` of logits at a
    time: the log probabilities of a long prompt without its logits, [tokens, vocabulary], in memory."""
    rows = x.shape[0]
    if token_ids.dim() != 1 or token_ids.shape[0] != rows:
        raise RuntimeError(f"head_logprobs: token_ids must be [{rows}]")
    # the product has no autograd node: its result would not say that x needs a derivative
    if not torch.compiler.is_compiling():
        _gsq_ops.no_gradient("head_logprobs", x)
    elif x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("head_logprobs: no gradient is computed here; detach the input or call under torch.no_grad()")
    vocab = layer.weight.shape[0]
    step = max(1, max_logit_bytes // max(1, vocab * x.element_size()))
    parts = [token_logprobs(method.apply(layer, x[i:i + step]), token_ids[i:i + step], top_n) for i in range(0, max(rows, 1), step)]
    return parts[0] if len(parts) == 1 else TokenLogprobs(*(torch.cat(p) for p in zip(*parts)))
