"""The experts' layer and the log probabilities behind kernels that let the next one start before they have written their results: the
fused norm, the products' last steps, the kernels themselves. Every chain runs over changing inputs in the same buffers without a
synchronisation, and has to give bit for bit what it gives with one after every step."""

import pytest
import torch

import gsq_b200  # noqa: F401
from gsq_b200 import logprobs, synth
from gsq_b200.quantization import linear

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
