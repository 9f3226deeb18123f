"""The mixture-of-experts layer (gsq_b200.quantization.fused_moe) against its definition in 64 bits (oracle/moe.py): the choice of
the experts, the products of all ten types, choices that are not here, strides, types, streams, captured calls.

Bounds: the oracle follows the errors of 32-bit sums through the layer, value by value; y's own rounding adds half a step of its type."""

import numpy as np
import pytest
import torch

import gsq_b200  # noqa: F401
from gsq_b200 import synth
from gsq_b200.quantization import fused_moe
from oracle import moe

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {**synth.TYPE_IDS, **synth.LOW_BIT_TYPE_IDS}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _stack(name, experts, rows, k, seed):
    """[experts, rows, bytes] with block scales that keep products near one (fp16 outputs do not overflow)."""
    raw = np.stack([synth.make_weight(TYPES[name], rows, k, seed + 97 * e) for e in range(experts)])
    b = raw.reshape(experts, rows, k // 256, -1)
    at = {"Q6_K": 208, "Q2_K": 80}.get(name, 0)
    if name == "IQ1_M":
        return raw
    for i in ((at, at + 2) if name in ("Q4_K", "Q2_K") else (at,)):
        d = np.ascontiguousarray(b[..., i:i + 2]).view(np.float16).astype(np.float32) * {"Q6_K": 0.01, "Q4_K": 0.02, "IQ4_XS": 0.01, "IQ3_S": 0.2}.get(name, 0.1)
        b[..., i:i + 2] = d.astype(np.float16).view(np.uint8)
    return raw


def _inputs(m, experts, top_k, hidden, inter, t13, t2, dtype, seed):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(synth.make_activation(m, hidden, seed, 1e-3)).to(dtype)
    r13, r2 = _stack(t13, experts, 2 * inter, hidden, seed + 1), _stack(t2, experts, hidden, inter, seed + 2)
    logits = torch.from_numpy(rng.standard_normal((m, experts)).astype(np.float32) * 2)
    ids = np.argsort(-logits.numpy(), 1)[:, :top_k].astype(np.int32)
    w = rng.random((m, top_k)).astype(np.float32)
    return x, r13, r2, logits, w / w.sum(1, keepdims=True), ids


def _check(y, x, r13, r2, t13, t2, w, ids, act="silu"):
    ref, bound = moe.experts(x.float().numpy(), r13, r2, TYPES[t13], TYPES[t2], w, ids, act, truncates=1.0 if t2 in synth.LOW_BIT_TYPE_IDS else 0.0)
    if t13 in synth.LOW_BIT_TYPE_IDS:
        assert t2 in synth.LOW_BIT_TYPE_IDS      # (the bound has no truncation in front of the activation's rounding)
    y = y.float().cpu().numpy().astype(np.float64)
    assert np.isfinite(ref).all() and np.abs(ref).max() > 0
    tol = bound + HALF_STEP[x.dtype] * (np.abs(ref) + bound) + 1e-7
    off = np.abs(y - ref)
    assert (off <= tol).all(), (off.max(), float((off / tol).max()), np.argwhere(off > tol)[:4])
    # what the bound allows is small against the result, or it would not say anything
    assert np.linalg.norm(bound) <= 0.1 * np.linalg.norm(ref)


def _cuda(*ts):
    return [torch.from_numpy(t).to(DEV) if isinstance(t, np.ndarray) else t.to(DEV) for t in ts]


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("m", [1, 3])
def test_types(name, m):
    x, r13, r2, _, w, ids = _inputs(m, 4, 2, 512, 256, name, name, torch.float32, 10 + TYPES[name])
    xd, a, b, wd, idd = _cuda(x, r13, r2, w, ids)
    y = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, TYPES[name], TYPES[name])
    assert y.shape == x.shape and y.dtype == x.dtype
    if name in synth.LOW_BIT_TYPE_IDS:
        # a truncated sum in the gate or up product moves the activated product by more than fp32 does: row norms, with 1e-4 for
        # each of the two products (the truncating divisions are off by 5e-5 of a row's norm at most) and one 8-bit step for each
        # row of 256 values that may round the other way
        ref, _ = moe.experts(x.numpy(), r13, r2, TYPES[name], TYPES[name], w, ids)
        err = np.linalg.norm(y.cpu().numpy() - ref, axis=1) / np.linalg.norm(ref, axis=1)
        assert err.max() <= 2e-4 + 4 * 3 / 127 / 16
    else:
        _check(y, x, r13, r2, name, name, w, ids)


@pytest.mark.parametrize("t13,t2", [("Q4_K", "Q6_K"), ("IQ4_XS", "Q4_K"), ("IQ3_S", "IQ4_XS"), ("Q6_K", "IQ3_S")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,experts,top_k,hidden,inter", [(1, 8, 8, 256, 256), (2, 16, 3, 768, 512), (7, 5, 2, 1280, 256), (9, 3, 1, 256, 768), (33, 9, 4, 512, 256)])
def test_shapes(t13, t2, dtype, m, experts, top_k, hidden, inter):
    x, r13, r2, _, w, ids = _inputs(m, experts, top_k, hidden, inter, t13, t2, dtype, m + hidden)
    xd, a, b, wd, idd = _cuda(x, r13, r2, w, ids)
    act = "gelu" if m == 7 else "silu"
    y = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, TYPES[t13], TYPES[t2], act)
    _check(y, x, r13, r2, t13, t2, w, ids, act)


def test_all_tokens_on_one_expert_and_one_expert_only():
    for experts, m in ((4, 20), (1, 5)):
        x, r13, r2, _, w, _ = _inputs(m, experts, 1, 512, 256, "Q4_K", "Q6_K", torch.bfloat16, 5)
        ids = np.full((m, 1), experts - 1, dtype=np.int32)
        xd, a, b, wd, idd = _cuda(x, r13, r2, w, ids)
        _check(fused_moe.fused_moe_gguf(xd, a, b, wd, idd, 12, 14), x, r13, r2, "Q4_K", "Q6_K", w, ids)


def test_choices_that_are_not_here():
    m, experts, top_k = 6, 5, 4
    x, r13, r2, _, w, ids = _inputs(m, experts, top_k, 512, 256, "Q4_K", "Q4_K", torch.bfloat16, 6)
    ids[0] = -1                                  # a token without experts
    ids[1, 1:] = [-1, 5, 2 ** 31 - 1]            # one left
    ids[2] = [3, 3, 3, -2 ** 31]                 # the same one three times
    w[3, 2] = 0.0
    xd, a, b, wd, idd = _cuda(x, r13, r2, w, ids)
    y = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, 12, 12)
    _check(y, x, r13, r2, "Q4_K", "Q4_K", w, ids)
    assert not y[0].any()
    wide = ids.astype(np.int64)
    wide[1, 2] = 2 ** 32 + 1                     # not expert 1
    assert torch.equal(fused_moe.fused_moe_gguf(xd, a, b, wd, torch.from_numpy(wide).to(DEV), 12, 12), y)
    none = fused_moe.fused_moe_gguf(xd, a, b, wd, torch.full_like(idd, -1), 12, 12)
    assert not none.any()


def test_nan_and_infinity_stay_with_their_token():
    x, r13, r2, _, w, ids = _inputs(5, 6, 2, 512, 256, "Q4_K", "Q6_K", torch.float32, 7)
    xd, a, b, wd, idd = _cuda(x, r13, r2, w, ids)
    good = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, 12, 14)
    bad = xd.clone()
    bad[1, 40], bad[3, 500] = float("nan"), float("inf")
    y = fused_moe.fused_moe_gguf(bad, a, b, wd, idd, 12, 14)
    keep = [0, 2, 4]
    assert torch.equal(y[keep], good[keep])
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[3]).any()
    large = xd.clone()
    large[2] *= 1e37                             # 127 x overflows
    z = fused_moe.fused_moe_gguf(large, a, b, wd, idd, 12, 14)
    assert torch.equal(z[keep[::2]], good[keep[::2]])


def test_zero_rows_and_zero_activations():
    x, r13, r2, _, w, ids = _inputs(3, 4, 2, 512, 256, "Q4_K", "Q6_K", torch.bfloat16, 8)
    xd, a, b, wd, idd = _cuda(x, r13, r2, w, ids)
    xd[1] = 0
    y = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, 12, 14)
    assert not y[1].any() and y[0].any()
    e = fused_moe.fused_moe_gguf(xd[:0], a, b, wd[:0], idd[:0], 12, 14)
    assert e.shape == (0, 512) and e.dtype == x.dtype


def test_strides_and_alignment():
    m = 5
    x, r13, r2, _, w, ids = _inputs(m, 6, 2, 512, 256, "Q4_K", "Q6_K", torch.bfloat16, 9)
    xd, a, b, wd, idd = _cuda(x, r13, r2, w, ids)
    want = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, 12, 14)
    for offset, stride in ((0, 520), (3, 777), (1, 513)):
        buf = torch.zeros(m * stride + 16, dtype=x.dtype, device=DEV)
        view = buf[offset:offset + m * stride].view(m, stride)[:, :512]
        view.copy_(xd)
        assert torch.equal(fused_moe.fused_moe_gguf(view, a, b, wd, idd, 12, 14), want)
    rows = xd[:1].expand(4, -1)                  # one token four times, row stride 0
    y = fused_moe.fused_moe_gguf(rows, a, b, wd[:1].expand(4, -1), idd[:1].expand(4, -1), 12, 14)
    # (not `want`: other tokens beside it make other groups, and so another order of the sums)
    assert torch.equal(y, fused_moe.fused_moe_gguf(rows.contiguous(), a, b, wd[:1].repeat(4, 1), idd[:1].repeat(4, 1), 12, 14))
    y = fused_moe.fused_moe_gguf(xd, a, b, wd.t().contiguous().t(), idd.t().contiguous().t(), 12, 14)   # the other order
    assert torch.equal(y, want)
    y = fused_moe.fused_moe_gguf(xd, a, b, wd.double(), idd.long(), 12, 14)
    assert torch.equal(y, want)


def test_result_into_a_strided_slot_leaves_the_rest():
    from gsq_b200 import lcpp_ops

    x, r13, r2, _, w, ids = _inputs(3, 4, 2, 512, 256, "Q4_K", "Q6_K", torch.float16, 19)
    xd, a, b, wd, idd = _cuda(x, r13, r2, w, ids)
    want = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, 12, 14)
    buf = torch.full((5, 777), 7.0, dtype=torch.float16, device=DEV)
    with lcpp_ops.output_into(buf[1:4, 3:515]):
        got = fused_moe.fused_moe_gguf(xd, a, b, wd, idd, 12, 14)
    assert got.data_ptr() == buf[1:, 3:].data_ptr() and torch.equal(got, want)
    got.fill_(7.0)
    assert (buf == 7.0).all()


# ---------------------------------------------------------------- routing


def _route_check(logits, top_k, **kw):
    w, ids = fused_moe.moe_route(logits.to(DEV), top_k, **{**kw, "bias": kw["bias"].to(DEV) if kw.get("bias") is not None else None})
    rw, rids = moe.route(logits.float().numpy(), top_k, kw.get("scoring", "softmax"), kw.get("renormalize", True),
                         None if kw.get("bias") is None else kw["bias"].numpy(), kw.get("scale", 1.0))
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    assert np.array_equal(ids.cpu().numpy(), rids)
    # softmax: argument, exponential (2^-22), up to 1024 additions in five plus 32 steps, two divisions, one product
    assert np.allclose(w.cpu().numpy(), rw, rtol=64 * 2.0 ** -24 * 4, atol=1e-37)
    return w, ids


@pytest.mark.parametrize("experts", [1, 2, 31, 32, 33, 64, 65, 128, 255, 256, 257, 1024])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route(experts, scoring):
    g = torch.Generator().manual_seed(experts)
    for dtype, m in ((torch.float32, 3), (torch.bfloat16, 70), (torch.float16, 1)):
        logits = (torch.randn(m, experts, generator=g) * 3).to(dtype)      # bf16: many equal ones
        top_k = min(experts, {torch.float32: 8, torch.bfloat16: 32, torch.float16: 1}[dtype])
        _route_check(logits, top_k, scoring=scoring)
        _route_check(logits, top_k, scoring=scoring, renormalize=False, scale=2.5)
        # a bias on a grid far coarser than fp32's errors decides the choice
        bias = torch.arange(experts).float().roll(experts // 3) * 4.0
        _route_check(logits, top_k, scoring=scoring, bias=bias)


def test_route_ties_go_to_the_lowest_number():
    w, ids = _route_check(torch.zeros(2, 100), 8)
    assert ids.tolist() == [list(range(8))] * 2
    z = torch.zeros(1, 100)
    z[0, 50:] = -0.0
    z[0, 97] = 1.0
    _, ids = _route_check(z, 4)
    assert ids.tolist() == [[97, 0, 1, 2]]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_masked_experts(scoring):
    inf, nan = float("inf"), float("nan")
    z = torch.randn(6, 40, generator=torch.Generator().manual_seed(1))
    z[0] = -inf                                   # nothing left
    z[1, :38] = -inf                              # two left, four wanted
    z[2, ::2] = nan
    z[3] = torch.finfo(torch.float32).min         # the type's lowest value is a score like another
    z[4, 7], z[4, 11] = inf, inf                  # two share the weight
    z[5, 1:] = nan
    w, ids = _route_check(z, 4, scoring=scoring)
    assert ids[0].tolist() == [-1] * 4 and not w[0].any()
    assert sorted(ids[1].tolist())[:2] == [-1, -1] and torch.isfinite(w).all()
    _route_check(z, 4, scoring=scoring, renormalize=False, bias=torch.linspace(-40, 40, 40))


def test_layer_is_the_choice_and_the_experts():
    for m, dtype in ((1, torch.bfloat16), (8, torch.float16), (9, torch.bfloat16), (40, torch.float32)):
        x, r13, r2, logits, _, _ = _inputs(m, 12, 3, 512, 256, "IQ4_XS", "Q6_K", dtype, 20 + m)
        bias = torch.linspace(-0.5, 0.5, 12)
        logits[0, :11] = -float("inf")
        xd, a, b, ld, bd = _cuda(x, r13, r2, logits.to(dtype), bias)
        for kw in ({}, {"scoring": "sigmoid", "bias": bd, "scale": 2.5}, {"renormalize": False, "activation": "gelu"}):
            y = fused_moe.moe_layer_gguf(xd, ld, a, b, 23, 14, 3, **kw)
            act = kw.pop("activation", "silu")
            w, ids = fused_moe.moe_route(ld, 3, **kw)
            assert torch.equal(y, fused_moe.fused_moe_gguf(xd, a, b, w, ids, 23, 14, act))
            _check(y, x, r13, r2, "IQ4_XS", "Q6_K", w.cpu().numpy(), ids.cpu().numpy(), act)


# ---------------------------------------------------------------- how it is called


def test_same_bits_every_time_captured_and_on_other_streams():
    x, r13, r2, logits, _, _ = _inputs(12, 16, 4, 1024, 512, "Q4_K", "Q6_K", torch.bfloat16, 30)
    xd, a, b, ld = _cuda(x, r13, r2, logits)
    call = lambda: fused_moe.moe_layer_gguf(xd, ld, a, b, 12, 14, 4)  # noqa: E731
    want = call()
    assert all(torch.equal(call(), want) for _ in range(5))
    graphs = []
    for _ in range(2):                            # two graphs alive at once, replayed in turn and side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = call()
        graphs.append((g, y))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for (g, _), s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for _, y in graphs)
    new = torch.randn_like(xd)
    old = xd.clone()
    xd.copy_(new)
    for g, _ in graphs:
        g.replay()
    assert all(torch.equal(y, call()) for _, y in graphs)
    xd.copy_(old)
    outs = []
    for i in range(8):                            # eager calls that overlap
        with torch.cuda.stream(streams[i % 2]):
            outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in outs)


def test_custom_ops_under_compile_tracing():
    from torch._subclasses.fake_tensor import FakeTensorMode

    x, r13, r2, logits, w, ids = _inputs(2, 4, 2, 512, 256, "Q4_K", "Q6_K", torch.bfloat16, 31)
    ts = _cuda(x, r13, r2, logits, w, ids)
    with FakeTensorMode(allow_non_fake_inputs=False) as mode:
        fx, a, b, ld, wd, idd = [mode.from_tensor(t) for t in ts]
        assert fused_moe.moe_layer_gguf(fx, ld, a, b, 12, 14, 2).shape == (2, 512)
        assert fused_moe.fused_moe_gguf(fx, a, b, wd, idd, 12, 14).dtype == torch.bfloat16
        assert [t.shape for t in fused_moe.moe_route(ld, 2)] == [(2, 2), (2, 2)]


def test_native_and_dispatched_calls_agree():
    x, r13, r2, logits, w, ids = _inputs(4, 4, 2, 512, 256, "Q4_K", "Q6_K", torch.bfloat16, 32)
    xd, a, b, ld, wd, idd = _cuda(x, r13, r2, logits, w, ids)
    assert torch.equal(torch.ops._C_gguf.gsq_moe_experts(xd, a, b, wd, idd, 12, 14, 0), fused_moe.fused_moe_gguf(xd, a, b, wd, idd, 12, 14))
    assert torch.equal(torch.ops._C_gguf.gsq_moe_layer(xd, ld, a, b, 12, 14, 2, 0, True, None, 1.0, 0), fused_moe.moe_layer_gguf(xd, ld, a, b, 12, 14, 2))
