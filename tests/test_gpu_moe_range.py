"""The mixture-of-experts layer at the ends of its ranges: many tokens (several passes, groups of 16, more groups than are looked up at a
time), many experts, rows from one superblock to longer than the tensor-core kernel takes, types mixed between the products, stacks past
2^31 bytes, a first call under capture. Bounds as in test_gpu_moe.py: oracle/moe.py's, plus half a step of y's type."""

import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import gsq_b200
from gsq_b200 import synth
from gsq_b200.quantization import fused_moe
from oracle import moe
from test_gpu_moe import DEV, HALF_STEP, TYPES, _check, _cuda, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,experts,top_k", [(200, 20, 8), (1024, 6, 2), (1030, 6, 2), (2049, 3, 1)])
def test_many_tokens(m, experts, top_k):
    x, r13, r2, _, w, ids = _inputs(m, experts, top_k, 512, 256, "Q4_K", "Q6_K", torch.bfloat16, 50 + m)
    ids[5], ids[m - 1] = -1, -1
    xd, a, b, wd, idd = _cuda(x, r13, r2, w, ids)
    y = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, 12, 14)
    _check(y, x, r13, r2, "Q4_K", "Q6_K", w, ids)
    assert not y[5].any() and not y[m - 1].any()
    wide = torch.full((m, 530), 7.0, dtype=x.dtype, device=DEV)
    wide[:, 8:520] = xd
    assert torch.equal(fused_moe.fused_moe_gguf(wide[:, 8:520], a, b, wd, idd, 12, 14), y)


@pytest.mark.parametrize("m,experts", [(3, 300), (64, 12), (65, 12), (70, 300), (1030, 260)])
def test_layer_with_many_tokens_or_experts(m, experts):
    x, r13, r2, logits, _, _ = _inputs(m, 4, 3, 256, 256, "Q4_K", "Q4_K", torch.float32, 60 + experts)
    logits = torch.from_numpy(np.random.default_rng(m).standard_normal((m, experts)).astype(np.float32))
    same = np.arange(experts) % 4                 # experts e, e + 4, ... have the same weights
    xd, a, b, ld = _cuda(x, r13[same], r2[same], logits)
    y = fused_moe.moe_layer_gguf(xd, ld, a, b, 12, 12, 3, scoring="sigmoid")
    w, ids = fused_moe.moe_route(ld, 3, scoring="sigmoid")
    assert torch.equal(y, fused_moe.fused_moe_gguf(xd, a, b, w, ids, 12, 12))
    _check(y, x, r13, r2, "Q4_K", "Q4_K", w.cpu().numpy(), ids.cpu().numpy() % 4)


def test_more_groups_than_a_block_looks_up_at_a_time():
    """992 experts with 33 pairs each, and gate / up rows too long for 16 columns of activations: 4960 groups of 8 and 1, 33 or more a
    block. Some tokens against the oracle; all against calls of 33 tokens, in which every pair is a group of its own. Sums in another order
    may round an activated value the other way: one step of 8 bits in 16 norms of a row, 1.5e-3, a row of 32 pairs' together less."""
    m, experts, top_k, hidden = 1023, 992, 32, 8448
    x, r13, r2, _, _, _ = _inputs(m, 4, 1, hidden, 256, "Q4_K", "Q4_K", torch.float32, 70)
    w = np.random.default_rng(7).random((m, top_k)).astype(np.float32) / 32
    ids = (np.arange(m * top_k).reshape(m, top_k) % experts).astype(np.int32)
    a, b = [d[torch.arange(experts, device=DEV) % 4].contiguous() for d in _cuda(r13, r2)]   # e, e + 4, ... have the same weights
    xd, wd, idd = _cuda(x, w, ids)
    y = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, 12, 12)
    for t in range(0, m, 33):
        part = fused_moe.fused_moe_gguf(xd[t:t + 33], a, b, wd[t:t + 33], idd[t:t + 33], 12, 12)
        assert ((part - y[t:t + 33]).norm(dim=1) <= 1.5e-3 * part.norm(dim=1)).all()
    some = np.arange(0, m, 73)
    _check(y[torch.from_numpy(some).to(DEV)], x[some], r13, r2, "Q4_K", "Q4_K", w[some], ids[some] % 4)


@pytest.mark.parametrize("t13,t2", [("Q4_K", "Q4_K"), ("Q6_K", "IQ4_XS")])
def test_many_experts(t13, t2):
    """992 experts with 33 pairs each (groups of 16, 16 and 1), then 1024 experts with one."""
    experts = 1024
    x, r13, r2, _, _, _ = _inputs(1024, 4, 1, 256, 256, t13, t2, torch.float32, 71)
    same = np.arange(experts) % 4
    xd, a, b = _cuda(x, r13[same], r2[same])
    w = np.random.default_rng(7).random((1023, 32)).astype(np.float32) / 32
    ids = (np.arange(1023 * 32).reshape(1023, 32) % 992).astype(np.int32)
    y = fused_moe.fused_moe_gguf(xd[:1023], a, b, *_cuda(w, ids), TYPES[t13], TYPES[t2])
    _check(y, x[:1023], r13, r2, t13, t2, w, ids % 4)
    ids = np.random.default_rng(8).permutation(experts).astype(np.int32)[:, None]
    w = np.ones((1024, 1), np.float32)
    y = fused_moe.fused_moe_gguf(xd, a, b, *_cuda(w, ids), TYPES[t13], TYPES[t2])
    _check(y, x, r13, r2, t13, t2, w, ids % 4)


@pytest.mark.parametrize("n", range(1, 18))
def test_pairs_of_an_expert(n):
    """1 to 17 tokens of one expert beside one token of another: every form of a group."""
    for t13, t2 in (("Q4_K", "Q6_K"), ("IQ3_S", "IQ4_XS")):
        x, r13, r2, _, _, _ = _inputs(n + 1, 2, 1, 512, 512, t13, t2, torch.float32, 80 + n)
        ids = np.zeros((n + 1, 1), np.int32)
        ids[n // 2] = 1
        w = np.ones((n + 1, 1), np.float32)
        xd, a, b, wd, idd = _cuda(x, r13, r2, w, ids)
        _check(fused_moe.fused_moe_gguf(xd, a, b, wd, idd, TYPES[t13], TYPES[t2]), x, r13, r2, t13, t2, w, ids)


# rows in superblocks: each reaches another layout of the activations and rings, or is longer than fits
ROWS = [("Q4_K", 16), ("Q4_K", 17), ("Q4_K", 33), ("Q4_K", 50), ("Q4_K", 60), ("Q6_K", 5), ("Q6_K", 9), ("Q6_K", 21), ("Q6_K", 45), ("IQ4_XS", 17),
        ("IQ4_XS", 23), ("IQ4_XS", 55), ("IQ4_XS", 66), ("IQ3_S", 17), ("IQ3_S", 20), ("IQ3_S", 43), ("IQ3_S", 59)]


@pytest.mark.parametrize("name,blocks", ROWS)
@pytest.mark.parametrize("m,experts", [(3, 4), (21, 2)])
def test_long_rows(name, blocks, m, experts):
    k = 256 * blocks
    for hidden, inter in ((k, 256), (256, k)):
        t13, t2 = (name, "Q4_K") if hidden == k else ("Q4_K", name)
        x, r13, r2, _, w, ids = _inputs(m, experts, 1, hidden, inter, t13, t2, torch.float32, 90 + blocks)
        xd, a, b, wd, idd = _cuda(x, r13, r2, w, ids)
        y = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, TYPES[t13], TYPES[t2]).cpu().numpy().astype(np.float64)
        ref, bound = moe.experts(x.numpy(), r13, r2, TYPES[t13], TYPES[t2], w, ids)
        assert (np.abs(y - ref) <= bound + HALF_STEP[torch.float32] * (np.abs(ref) + bound) + 1e-7).all()
        # the bound's worst case grows with the row (to 0.17 of y's norm here). Were every activated value rounded the other way, a row would be off by a
        # step to the values' norm, 4 / 127 for values that reach four times that; a superblock that is lost takes 1 / sqrt(66) = 0.12
        assert (np.linalg.norm(y - ref, axis=1) <= 0.04 * np.linalg.norm(ref, axis=1)).all()


@pytest.mark.parametrize("low", list(synth.LOW_BIT_TYPE_IDS))
def test_low_bit_types_beside_the_main_ones(low):
    for t13, t2 in (("Q4_K", low), (low, "Q6_K")):
        x, r13, r2, logits, w, ids = _inputs(3, 4, 2, 512, 256, t13, t2, torch.float32, 95)
        xd, a, b, ld, wd, idd = _cuda(x, r13, r2, logits, w, ids)
        y = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, TYPES[t13], TYPES[t2])
        # as in test_gpu_moe.py's test_types, same sizes: truncated sums in front of the activation's rounding, by row norms
        ref, _ = moe.experts(x.numpy(), r13, r2, TYPES[t13], TYPES[t2], w, ids)
        err = np.linalg.norm(y.cpu().numpy() - ref, axis=1) / np.linalg.norm(ref, axis=1)
        assert err.max() <= 2e-4 + 4 * 3 / 127 / 16
        rw, rids = fused_moe.moe_route(ld, 2)
        assert torch.equal(fused_moe.moe_layer_gguf(xd, ld, a, b, TYPES[t13], TYPES[t2], 2), fused_moe.fused_moe_gguf(xd, a, b, rw, rids, TYPES[t13], TYPES[t2]))


def test_stack_past_2_31_bytes():
    m, experts, hidden, inter = 3, 1024, 4096, 512
    x, r13, r2, _, w, _ = _inputs(m, 2, 2, hidden, inter, "Q4_K", "Q4_K", torch.float32, 96)
    w13 = torch.zeros((experts, *r13.shape[1:]), dtype=torch.uint8, device=DEV)
    w2 = torch.zeros((experts, *r2.shape[1:]), dtype=torch.uint8, device=DEV)
    assert w13.numel() > 2 ** 31
    for i, e in enumerate((950, experts - 1)):
        w13[e], w2[e] = torch.from_numpy(r13[i]).to(DEV), torch.from_numpy(r2[i]).to(DEV)
    ids = np.array([[950, 1023], [1023, 950], [1023, 1023]], np.int32)
    xd, wd, idd = _cuda(x, w, ids)
    _check(fused_moe.fused_moe_gguf(xd, w13, w2, wd, idd, 12, 12), x, r13, r2, "Q4_K", "Q4_K", w, (ids == 1023).astype(np.int32))


def test_first_call_of_a_process_may_be_captured():
    code = """
import torch, gsq_b200
from gsq_b200.quantization import fused_moe
from gsq_b200 import logprobs
g = torch.Generator(device="cuda").manual_seed(1)
x = torch.randn(2, 512, device="cuda", generator=g)
w13 = torch.zeros(4, 512, 288, dtype=torch.uint8, device="cuda"); w2 = torch.zeros(4, 512, 210, dtype=torch.uint8, device="cuda")
w13[..., 16:] = 37; w13[..., 1] = 0x20; w13[..., 145] = 0x20; w2[..., :192] = 90; w2[..., 192:208] = 5; w2[..., 209] = 0x20
logits, ids = torch.randn(2, 4, device="cuda", generator=g), torch.tensor([3, 700], device="cuda")
vocab = torch.randn(2, 70000, device="cuda", generator=g)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = fused_moe.moe_layer_gguf(x, logits, w13, w2, 12, 14, 2)
    p = logprobs.token_logprobs(vocab, ids, 5)
graph.replay()
torch.cuda.synchronize()
q = logprobs.token_logprobs(vocab, ids, 5)
assert torch.equal(y, fused_moe.moe_layer_gguf(x, logits, w13, w2, 12, 14, 2)) and bool(y.any()) and bool(y.isfinite().all())
assert all(torch.equal(a, b) for a, b in zip(p, q))
print("same")
"""
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(gsq_b200.__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_experts_of_all_ranks_add_up():
    """Expert-parallel ranks' parts, each from its own stack: the layer's definition, with half a step of bf16 for each part."""
    m, experts, top_k = 9, 8, 3
    x, r13, r2, logits, _, _ = _inputs(m, experts, top_k, 512, 256, "Q4_K", "Q6_K", torch.bfloat16, 97)
    xd, a, b, ld = _cuda(x, r13, r2, logits)
    w, ids = fused_moe.moe_route(ld, top_k)
    parts = []
    for first in range(0, experts, 2):
        here = (ids >= first) & (ids < first + 2)
        part = fused_moe.fused_moe_gguf(xd, a[first:first + 2], b[first:first + 2], w, torch.where(here, ids - first, -1), 12, 14)
        parts.append(part.double().cpu().numpy())
    ref, bound = moe.experts(x.float().numpy(), r13, r2, 12, 14, w.cpu().numpy(), ids.cpu().numpy())
    tol = bound + HALF_STEP[torch.bfloat16] * 1.01 * sum(np.abs(p) for p in parts) + 1e-7
    assert (np.abs(sum(parts) - ref) <= tol).all()


def _two_ops():
    """Inputs and calls of the layer and the log probabilities on the same buffers."""
    from gsq_b200 import logprobs

    x, r13, r2, logits, _, _ = _inputs(9, 12, 3, 1024, 512, "Q4_K", "Q6_K", torch.bfloat16, 98)
    xd, a, b, ld = _cuda(x, r13, r2, logits)
    vocab = torch.randn(9, 30000, device=DEV)
    ids = torch.arange(9, device=DEV) * 3000

    def call():
        y = fused_moe.moe_layer_gguf(xd, ld, a, b, 12, 14, 3)
        return (y, *logprobs.token_logprobs(vocab, ids, 5), *logprobs.token_logprobs(vocab[:, :1000], ids % 1000, 5))

    return (xd, ld, vocab), call


def test_inputs_written_by_the_kernel_before():
    """The kernels start while the one before still runs: what that one writes, in place and into memory that a call before
    has just given back, is what they read."""
    buffers, call = _two_ops()
    g = torch.Generator(device=DEV).manual_seed(5)
    rounds = [[torch.randn(t.shape, device=DEV, generator=g).to(t.dtype) for t in buffers] for _ in range(12)]
    want = []
    for r in rounds:
        for t, v in zip(buffers, r):
            t.copy_(v)
        torch.cuda.synchronize()
        want.append(call())
        torch.cuda.synchronize()
    got = []
    for r in rounds:
        for t, v in zip(buffers, r):
            t.copy_(v)
        call()                                    # (its results' memory is free again for the next)
        got.append(call())
    assert all(torch.equal(p, q) for w, h in zip(want, got) for p, q in zip(w, h))


def test_captured_behind_copies_and_other_streams():
    """In a graph behind a fill, a copy and a join of two streams, and in front of a copy and of another stream's work."""
    buffers, call = _two_ops()
    new = [torch.randn(t.shape, device=DEV).to(t.dtype) for t in buffers]
    for t, v in zip(buffers, new):
        t.copy_(v)
    want = call()
    for t in buffers:
        t.zero_()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        buffers[0].zero_()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            buffers[2].copy_(new[2])
        buffers[0].copy_(new[0])
        buffers[1].copy_(new[1])
        main.wait_stream(side)
        got = call()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            twice = [2 * t for t in got]
        main.wait_stream(side)
        kept = [t.clone() for t in got]
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for w, p, q, r in zip(want, got, twice, kept):
        assert torch.equal(w, p) and torch.equal(2 * w, q) and torch.equal(w, r)
