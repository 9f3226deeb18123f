"""The experts' layer and the log probabilities behind kernels that let the next one start before they have written their results: the
fused norm, the products' last steps, the kernels themselves. Every chain runs over changing inputs in the same buffers without a
synchronisation, and has to give bit for bit what it gives with one after every step."""

import pytest
import torch

import gsq_b200  # noqa: F401
from gsq_b200 import fused, logprobs, synth
from gsq_b200.quantization import fused_moe, linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {**synth.TYPE_IDS, **synth.LOW_BIT_TYPE_IDS}


def _linear(name, rows, k, seed):
    """A linear of 2048 rows of the type, repeated up to `rows`."""
    layer, method = torch.nn.Module(), linear.GGUFLinearMethod(None)
    method.create_weights(layer, k, [rows], k, rows, torch.bfloat16)
    raw = torch.from_numpy(synth.make_weight(TYPES[name], min(rows, 2048), k, seed)).to(DEV)
    layer.weight.load_shard(raw[torch.arange(rows, device=DEV) % len(raw)].contiguous(), None)
    layer.weight_type.weight_type = TYPES[name]
    method.process_weights_after_loading(layer)
    return layer, method


def _same_without_synchronisation(rounds, step):
    """step(i, sync): one round's outputs, sync() called between its steps."""
    want = []
    for i in range(rounds):
        want.append(step(i, torch.cuda.synchronize))
        torch.cuda.synchronize()
    got = [step(i, lambda: None) for i in range(rounds)]
    assert all(torch.equal(p, q) for w, h in zip(want, got) for p, q in zip(w, h))


# few rows: the small-batch product (repacked and GGUF order), the low-bit and dp4a products; 40, 100: the product whose parts a kernel of its own adds
# up; 300: the two-step product
@pytest.mark.parametrize("name,m", [("IQ3_S", 1), ("IQ3_S", 4), ("Q6_K", 3), ("Q4_K", 1), ("IQ2_S", 2), ("Q2_K", 1), ("IQ1_M", 5), ("IQ4_XS", 12),
                                    ("Q4_K", 40), ("IQ4_XS", 100), ("IQ3_S", 40), ("Q6_K", 300)])
def test_head_then_log_probabilities(name, m):
    vocab, k, rounds = 40000, 1024, 10
    layer, method = _linear(name, vocab, k, 7)
    g = torch.Generator(device=DEV).manual_seed(m)
    xs = [torch.randn(m, k, device=DEV, generator=g).to(torch.bfloat16) for _ in range(rounds)]
    ids = [torch.randint(0, vocab, (m,), device=DEV, generator=g) for _ in range(rounds)]

    def step(i, sync):
        z = method.apply(layer, xs[i])
        sync()
        whole = logprobs.token_logprobs(z, ids[i], 5)
        sync()
        part = logprobs.token_logprobs(z[:, :2000], ids[i] % 2000, 3)      # a warp a row
        sync()
        return (*whole, *part)

    _same_without_synchronisation(rounds, step)


def _stack(name, experts, rows, k, seed):
    """[experts, rows, bytes], rows of 2048 at most repeated; values of about 0.02."""
    raw = torch.from_numpy(synth.make_weight(TYPES[name], min(experts * rows, 2048), k, seed)).to(DEV)
    w = raw[torch.arange(experts * rows, device=DEV) % len(raw)].view(experts, rows, -1).contiguous()
    b = w.view(experts, rows, k // 256, -1)
    for i in {"Q6_K": (208,), "Q4_K": (0, 2)}.get(name, (0,)):
        b[..., i:i + 2] = (b[..., i:i + 2].contiguous().view(torch.float16).float() * 0.01).to(torch.float16).view(torch.uint8)
    return w


# one token to more than one block of the plan makes the choice for, and more than a pass; products on the tensor cores and by dp4a
@pytest.mark.parametrize("m,t13,t2", [(1, "Q4_K", "Q6_K"), (4, "IQ4_XS", "Q4_K"), (9, "IQ2_S", "IQ4_XS"), (16, "Q4_K", "IQ2_S"), (70, "Q6_K", "Q4_K"),
                                      (1040, "Q4_K", "Q4_K")])
def test_layers_of_norm_router_experts(m, t13, t2):
    """Fused norm with its residual in place -> router (a quantised linear) -> experts -> the next layer's norm: each reads what the
    one before it writes after letting it start."""
    hidden, inter, experts, top_k, layers, rounds = 2048, 512, 16, 3, 3, 6
    g = torch.Generator(device=DEV).manual_seed(m)
    gates = [_linear(name, experts, hidden, 20 + i) for i, name in enumerate(("Q6_K", "Q4_K", "IQ3_S"))]
    w13, w2 = _stack(t13, experts, 2 * inter, hidden, 3), _stack(t2, experts, hidden, inter, 4)
    gamma = (1 + 0.1 * torch.randn(hidden, device=DEV, generator=g)).to(torch.bfloat16)
    starts = [torch.randn(m, hidden, device=DEV, generator=g).to(torch.bfloat16) for _ in range(rounds)]
    residual = torch.empty_like(starts[0])

    def step(i, sync):
        x = starts[i]
        residual.zero_()
        for layer, method in gates[:layers]:
            _, y = fused.rmsnorm_quantize_q8_1(x, gamma, 1e-6, residual, want_y=True)
            sync()
            z = method.apply(layer, y)
            sync()
            x = fused_moe.moe_layer_gguf(y, z, w13, w2, TYPES[t13], TYPES[t2], top_k)
            sync()
        _, last = fused.rmsnorm_quantize_q8_1(x, gamma, 1e-6, residual, want_y=True)
        sync()
        return x, last, residual.clone()

    _same_without_synchronisation(rounds, step)
