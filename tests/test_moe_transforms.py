"""The experts' layer and the log probabilities under torch.func.vmap and torch.jit.trace: what a transform or a trace has to see goes
through the custom ops, also where the entry points call the native code under them. On the CPU up to the refusal that ends a clean call."""

import pytest
import torch

import gsq_b200  # noqa: F401
from gsq_b200 import _gsq_ops, logprobs, synth
from gsq_b200.quantization import fused_moe

W13, W2 = torch.zeros(4, 512, 288, dtype=torch.uint8), torch.zeros(4, 512, 210, dtype=torch.uint8)
NATIVE = {
    "experts": lambda x, z: _gsq_ops.moe_experts(x, W13, W2, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32), 12, 14, 0),
    "layer": lambda x, z: _gsq_ops.moe_layer(x, z, W13, W2, 12, 14, 2, 0, True, None, 1.0, 0),
    "route": lambda x, z: _gsq_ops.moe_route(z, 2, 0, True, None, 1.0),
    "log probabilities": lambda x, z: _gsq_ops.token_logprobs(z, torch.zeros(3, dtype=torch.int64), 2),
}


@pytest.mark.parametrize("name", list(NATIVE))
def test_native_calls_reach_the_op(name):
    seen = []

    class Mode(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    # under vmap the op's own layer comes before the checks, in which a batched tensor has one dimension less
    with Mode(), pytest.raises(RuntimeError, match="must be CUDA"):
        torch.func.vmap(NATIVE[name])(torch.zeros(2, 3, 512), torch.zeros(2, 3, 4))
    assert any("_C_gguf.gsq_" in s for s in seen), seen


def test_native_products_leave_a_transform_to_the_op():
    w = torch.zeros(256, 144, dtype=torch.uint8)
    torch.func.vmap(lambda x: _none(_gsq_ops.linear(x, w, 12, None, False), x))(torch.zeros(2, 3, 256))
    torch.func.vmap(lambda x: _none(_gsq_ops.linear_runs(x, w, [0, 256, 144, 12], False), x))(torch.zeros(2, 3, 256))


def _none(out, x):
    assert out is None
    return x


def _stacks():
    import numpy as np

    w13 = np.stack([synth.make_weight(12, 512, 512, e) for e in range(4)])
    w2 = np.stack([synth.make_weight(14, 512, 256, 9 + e) for e in range(4)])
    return torch.from_numpy(w13).cuda(), torch.from_numpy(w2).cuda()


@pytest.mark.gpu
def test_vmap():
    g = torch.Generator(device="cuda").manual_seed(3)
    w13, w2 = _stacks()
    x, z = torch.randn(3, 5, 512, device="cuda", generator=g), torch.randn(3, 5, 4, device="cuda", generator=g)
    v, ids = torch.randn(3, 5, 9000, device="cuda", generator=g), torch.randint(0, 9000, (3, 5), device="cuda", generator=g)

    def layer(x, z):
        return fused_moe.moe_layer_gguf(x, z, w13, w2, 12, 14, 2)

    def experts(x, z):
        w, i = fused_moe.moe_route(z, 2)
        return fused_moe.fused_moe_gguf(x, w13, w2, w, i, 12, 14)

    for f in (layer, experts):
        assert torch.equal(torch.func.vmap(f)(x, z), torch.stack([f(a, b) for a, b in zip(x, z)]))
        assert torch.equal(torch.func.vmap(f, in_dims=(None, 0))(x[0], z), torch.stack([f(x[0], b) for b in z]))
    got = torch.func.vmap(lambda a, b: tuple(logprobs.token_logprobs(a, b, 4)))(v, ids)
    want = [logprobs.token_logprobs(a, b, 4) for a, b in zip(v, ids)]
    for i, t in enumerate(got):
        assert torch.equal(t, torch.stack([w[i] for w in want]))


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_jit_trace():
    """A trace records the op: on other inputs it computes, rather than give the results of the traced call."""
    g = torch.Generator(device="cuda").manual_seed(4)
    w13, w2 = _stacks()
    new = lambda: (torch.randn(5, 512, device="cuda", generator=g), torch.randn(5, 4, device="cuda", generator=g))  # noqa: E731

    def f(x, z):
        y = fused_moe.moe_layer_gguf(x, z, w13, w2, 12, 14, 2)
        lp, _, _, _, top = logprobs.token_logprobs(y, torch.zeros(5, dtype=torch.int64, device="cuda"), 3)
        return y, lp, top

    traced = torch.jit.trace(f, new(), check_trace=False)
    for _ in range(2):
        args = new()
        assert all(torch.equal(p, q) for p, q in zip(traced(*args), f(*args)))


def _head(vocab=9000, k=512, name="Q6_K"):
    from gsq_b200.quantization import linear

    layer, method = torch.nn.Module(), linear.GGUFLinearMethod(None)
    method.create_weights(layer, k, [vocab], k, vocab, torch.bfloat16)
    layer.weight.load_shard(torch.from_numpy(synth.make_weight(synth.TYPE_IDS[name], vocab, k, 5)).cuda(), None)
    layer.weight_type.weight_type = synth.TYPE_IDS[name]
    method.process_weights_after_loading(layer)
    return layer, method


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_head_under_vmap_trace_and_compile():
    g = torch.Generator(device="cuda").manual_seed(6)
    layer, method = _head()
    w13, w2 = _stacks()
    ids = torch.randint(0, 9000, (5,), device="cuda", generator=g)
    new = lambda: (torch.randn(5, 512, device="cuda", generator=g).to(torch.bfloat16), torch.randn(5, 4, device="cuda", generator=g))  # noqa: E731

    def f(x, z):
        m = fused_moe.moe_layer_gguf(x, z, w13, w2, 12, 14, 2)
        y = x + 1e-3 * m
        return (m, y, *logprobs.head_logprobs(method, layer, y, ids, 3))

    pairs = [new() for _ in range(3)]
    got = torch.func.vmap(f)(torch.stack([x for x, _ in pairs]), torch.stack([z for _, z in pairs]))
    want = [f(*p) for p in pairs]
    for i, t in enumerate(got):
        assert torch.equal(t, torch.stack([w[i] for w in want]))
    traced = torch.jit.trace(f, new(), check_trace=False)
    compiled = torch.compile(f, backend="aot_eager", fullgraph=True)
    for call in (traced, compiled):
        for p, w in zip(pairs, want):
            m, y, *got = call(*p)
            # (y itself may be rounded once there where it is rounded twice here: a trace fuses its two steps)
            assert torch.equal(m, w[0])
            assert all(torch.equal(a, b) for a, b in zip(got, logprobs.head_logprobs(method, layer, y, ids, 3)))
