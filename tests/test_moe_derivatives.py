"""The mixture-of-experts layer and the log probabilities have no derivative: a call that would need one, in either mode, is refused
before it runs instead of returning a result without it. On CPU tensors, where a clean call ends in "must be CUDA tensors"."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import gsq_b200  # noqa: F401
from gsq_b200 import logprobs
from gsq_b200.quantization import fused_moe

W13, W2 = torch.zeros(4, 512, 288, dtype=torch.uint8), torch.zeros(4, 512, 210, dtype=torch.uint8)
IDS = torch.zeros(3, 2, dtype=torch.int32)
CALLS = {
    "experts, of x": lambda v: fused_moe.fused_moe_gguf(v(3, 512), W13, W2, torch.zeros(3, 2), IDS, 12, 14),
    "experts, of the weights": lambda v: fused_moe.fused_moe_gguf(torch.zeros(3, 512), W13, W2, v(3, 2), IDS, 12, 14),
    "layer, of x": lambda v: fused_moe.moe_layer_gguf(v(3, 512), torch.zeros(3, 4), W13, W2, 12, 14, 2),
    "layer, of the logits": lambda v: fused_moe.moe_layer_gguf(torch.zeros(3, 512), v(3, 4), W13, W2, 12, 14, 2),
    "layer, of the bias": lambda v: fused_moe.moe_layer_gguf(torch.zeros(3, 512), torch.zeros(3, 4), W13, W2, 12, 14, 2, bias=v(4)),
    "route": lambda v: fused_moe.moe_route(v(3, 4), 2),
    "log probabilities": lambda v: logprobs.token_logprobs(v(3, 100), torch.zeros(3, dtype=torch.int64), 5),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_forward_mode(name):
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            CALLS[name](lambda *s: fwd.make_dual(torch.zeros(s), torch.ones(s)))
        with torch.inference_mode(), pytest.raises(RuntimeError, match="must be CUDA"):
            CALLS[name](torch.zeros)
        with pytest.raises(RuntimeError, match="must be CUDA"):
            CALLS[name](torch.zeros)


@pytest.mark.parametrize("name", list(CALLS))
def test_transforms_of_functions(name):
    def f(t):
        out = CALLS[name](lambda *s: t)
        return (out if isinstance(out, torch.Tensor) else out[0]).sum()

    shape = {"experts, of the weights": (3, 2), "layer, of the logits": (3, 4), "layer, of the bias": (4,), "route": (3, 4), "log probabilities": (3, 100)}.get(name, (3, 512))
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.func.grad(f)(torch.zeros(shape))
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(f, (torch.zeros(shape),), (torch.ones(shape),))


class _Head:
    """A linear method whose product, as the native ones, leaves no trace of a derivative."""

    calls = 0

    def apply(self, layer, x):
        self.calls += 1
        return torch.zeros(x.shape[0], layer.weight.shape[0])


def test_head_in_front():
    """The product in front of the log probabilities has no autograd node: its result does not say that x needs a derivative."""
    layer, head, ids = torch.nn.Module(), _Head(), torch.zeros(3, dtype=torch.int64)
    layer.weight = torch.nn.Parameter(torch.zeros(100, 144, dtype=torch.uint8), requires_grad=False)

    def call(x):
        return logprobs.head_logprobs(head, layer, x, ids, 2)

    with pytest.raises(RuntimeError, match="no gradient"):
        call(torch.zeros(3, 256, requires_grad=True))
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.func.grad(lambda x: call(x).logprobs.sum())(torch.zeros(3, 256))
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda x: call(x).logprobs, (torch.zeros(3, 256),), (torch.ones(3, 256),))
    with fwd.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
        call(fwd.make_dual(torch.zeros(3, 256), torch.ones(3, 256)))
    assert head.calls == 0
    with torch.no_grad(), pytest.raises(RuntimeError, match="must be CUDA"):
        call(torch.zeros(3, 256, requires_grad=True))
    assert head.calls == 1


def test_head_in_front_traced():
    layer, head, ids = torch.nn.Module(), _Head(), torch.zeros(3, dtype=torch.int64)
    layer.weight = torch.nn.Parameter(torch.zeros(100, 144, dtype=torch.uint8), requires_grad=False)
    call = torch.compile(lambda x: logprobs.head_logprobs(head, layer, x, ids, 2), backend="eager", fullgraph=True)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        call(torch.zeros(3, 256))
    with pytest.raises(Exception, match="no gradient"):
        call(torch.zeros(3, 256, requires_grad=True))
