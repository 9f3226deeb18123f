"""Log probabilities of given tokens with rank, entropy and alternatives (gsq_b200.logprobs) against float64 (oracle/moe.py), and a
run of the operators together as a server has them: router, experts, head, log probabilities."""

import numpy as np
import pytest
import torch

import gsq_b200  # noqa: F401
from gsq_b200 import logprobs, synth
from gsq_b200.quantization import fused_moe, linear
from oracle import moe

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _check(x, ids, top_n, got=None):
    got = logprobs.token_logprobs(x.to(DEV) if not x.is_cuda else x, ids.to(DEV), top_n) if got is None else got
    want = moe.logprobs(x.float().cpu().numpy(), ids.cpu().numpy(), top_n)
    m = x.shape[0]
    assert got.logprobs.dtype == got.entropy.dtype == got.top_logprobs.dtype == torch.float32
    assert got.ranks.dtype == got.top_ids.dtype == torch.int64
    assert got.top_ids.shape == got.top_logprobs.shape == (m, top_n)
    assert np.array_equal(got.ranks.cpu().numpy(), want["ranks"])
    assert np.array_equal(got.top_ids.cpu().numpy(), want["top_ids"])

    def near(a, b, tol):
        a = a.cpu().numpy().astype(np.float64)
        fin = np.isfinite(b)
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[np.isinf(b)], b[np.isinf(b)])
        assert np.isfinite(a[fin]).all()
        off = np.abs(a - np.where(fin, b, 0))[fin]
        lim = (tol + 2.0 ** -23 * np.abs(np.where(fin, b, 0)))[fin]
        assert (off <= lim).all(), (off.max(), (off / np.maximum(lim, 1e-30)).max())

    near(got.logprobs, want["logprobs"], want["tol"])
    near(got.entropy, want["entropy"], want["entropy_tol"])
    near(got.top_logprobs, want["top_logprobs"], want["tol"][:, None])
    return got


def _logits(m, v, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, v, generator=g) * spread).to(dtype), torch.randint(0, v, (m,), generator=g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [1, 2, 7, 8, 31, 33, 255, 1000, 1003, 4096, 8191, 16385, 32003, 50001, 151936])
def test_vocabularies(dtype, v):
    for m, top_n in ((1, 20), (3, 32), (5, 1), (2, 0)):
        x, ids = _logits(m, v, dtype, v + m)
        ids[0] = v - 1
        _check(x, ids, top_n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 2, 9, 40, 150, 300, 700])
def test_rows(dtype, m):
    x, ids = _logits(m, 5003, dtype, m)
    _check(x, ids, 5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masks_and_special_values(dtype):
    inf, nan = float("inf"), float("nan")
    x, ids = _logits(14, 3001, dtype, 5)
    x[0] = -inf                                    # nothing left
    x[1, :2995] = -inf                             # fewer left than alternatives
    x[2, ::2] = -inf
    x[3] = torch.finfo(dtype).min                  # the lowest value everywhere: uniform
    x[4, 100:] = torch.finfo(dtype).min
    x[5, 17] = nan
    x[6, 17] = inf
    x[7, 17], x[7, 900], x[7, 5] = inf, nan, -inf
    x[8] = nan
    x[9] = 1.5                                     # all equal
    x[10, :] = 0.0
    x[10, 1::3] = -0.0                             # equal too
    x[11, 2999] = 40.0                             # one token takes it all
    x[12, :] = -inf
    x[12, 2000] = -5.0
    x[13, :1500] = nan                             # half of the order is NaN
    x[13, 1500:] = -inf
    for top_n in (0, 1, 20, 32):
        got = _check(x, ids, top_n)
    assert got.entropy[0] == 0 and got.entropy[12] == 0
    ids[:] = 2000
    got = _check(x, ids, 3)
    assert got.logprobs[12] == 0 and got.ranks[12] == 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("order", ["ascending", "descending", "blocks", "few values", "head heavy", "one thread's columns"])
def test_orders_that_are_hard_for_a_selection(dtype, order):
    v = 40000
    base = torch.arange(v, dtype=torch.float32) / v * 20 - 10
    x = {"ascending": base, "descending": base.flip(0), "blocks": base.view(40, 1000).flip(0).reshape(-1),
         "few values": (base * 0.2).round(), "head heavy": torch.cat([torch.full((5000,), 3.0), base[:v - 5000]]),
         "one thread's columns": torch.where((torch.arange(v) // 8) % 512 == 77, base + 30, base)}[order]
    x = torch.stack([x, x.roll(7), -x]).to(dtype)
    ids = torch.tensor([0, v - 1, v // 2])
    for top_n in (1, 20, 32):
        _check(x, ids, top_n)


def test_tokens_outside_the_vocabulary():
    x, ids = _logits(6, 500, torch.float32, 8)
    ids[:] = torch.tensor([-1, 500, -2 ** 62, 2 ** 62, 2 ** 32 + 3, 499])
    got = _check(x, ids, 4)
    assert got.ranks.tolist()[:5] == [0] * 5 and got.logprobs[0] == 0 and torch.isnan(got.logprobs[1])
    small = logprobs.token_logprobs(x.to(DEV), torch.tensor([-1, 3, 4, 5, 6, 7], dtype=torch.int32, device=DEV), 0)
    assert torch.equal(small.logprobs, logprobs.token_logprobs(x.to(DEV), torch.tensor([-1, 3, 4, 5, 6, 7], device=DEV), 0).logprobs)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    m, v = 6, 4099
    x, ids = _logits(m, v, dtype, 9)
    want = _check(x, ids, 7)
    for offset, stride in ((0, 4104), (1, 4099), (3, 5001), (8, 4112)):
        buf = torch.full((m * stride + 16,), 99.0, dtype=dtype, device=DEV)      # columns past the vocabulary are larger than any logit
        view = buf[offset:offset + m * stride].view(m, stride)[:, :v]
        view.copy_(x)
        got = logprobs.token_logprobs(view, ids.to(DEV), 7)
        assert torch.equal(got.ranks, want.ranks) and torch.equal(got.top_ids, want.top_ids)
        _check(x, ids, 7, got)
    got = logprobs.token_logprobs(x[:1].to(DEV).expand(4, -1), ids[:1].to(DEV).expand(4), 7)
    assert all((t == t[:1]).all() for t in got)
    empty = logprobs.token_logprobs(x[:0].to(DEV), ids[:0].to(DEV), 3)
    assert empty.top_ids.shape == (0, 3) and empty.logprobs.shape == (0,)


def test_rows_past_two_gigabytes():
    """Offsets that pass 32 bits: the last rows of a table of 2^31 + values."""
    v, stride = 1000, 2 ** 21
    m = 1100
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("not enough device memory")
    buf = torch.zeros(m * stride, dtype=torch.float32, device=DEV)
    view = buf.view(m, stride)[:, :v]
    x, ids = _logits(4, v, torch.float32, 10)
    view[-4:] = x.to(DEV)
    ids_all = torch.full((m,), -1, device=DEV)
    ids_all[-4:] = ids.to(DEV)
    got = logprobs.token_logprobs(view, ids_all, 3)
    _check(x, ids, 3, logprobs.TokenLogprobs(*(t[-4:] for t in got)))


def test_same_bits_every_time_captured_and_on_other_streams():
    for m, v in ((1, 151936), (5, 32003), (400, 2000)):
        x, ids = _logits(m, v, torch.bfloat16, m)
        xd, idd = x.to(DEV), ids.to(DEV)
        call = lambda: logprobs.token_logprobs(xd, idd, 20)  # noqa: E731
        want = call()
        same = lambda r: all(torch.equal(p, q) for p, q in zip(r, want))  # noqa: E731
        assert all(same(call()) for _ in range(5))
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                r = call()
            graphs.append((g, r))
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(5):
            for (g, _), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            assert all(same(r) for _, r in graphs)
        outs = []
        for i in range(6):
            with torch.cuda.stream(streams[i % 2]):
                outs.append(call())
        torch.cuda.synchronize()
        assert all(same(r) for r in outs)


def test_custom_op_and_tracing():
    from torch._subclasses.fake_tensor import FakeTensorMode

    x, ids = _logits(3, 1000, torch.float16, 3)
    xd, idd = x.to(DEV), ids.to(DEV)
    got = torch.ops._C_gguf.gsq_token_logprobs(xd, idd, 4)
    assert all(torch.equal(p, q) for p, q in zip(got, logprobs.token_logprobs(xd, idd, 4)))
    with FakeTensorMode() as mode:
        r = logprobs.token_logprobs(mode.from_tensor(xd), mode.from_tensor(idd), 4)
        assert [tuple(t.shape) for t in r] == [(3,), (3,), (3,), (3, 4), (3, 4)]
        assert [t.dtype for t in r] == [t.dtype for t in got]


def _head(name, vocab, k, dtype):
    layer, method = torch.nn.Module(), linear.GGUFLinearMethod(None)
    method.create_weights(layer, k, [vocab], k, vocab, dtype)
    raw = synth.make_weight(synth.TYPE_IDS[name], vocab, k, 77)
    layer.weight.load_shard(torch.from_numpy(raw).to(DEV), None)
    layer.weight_type.weight_type = synth.TYPE_IDS[name]
    method.process_weights_after_loading(layer)
    return layer, method


def test_router_experts_head_log_probabilities():
    """A block's feed-forward half and the answer, as a server runs them: norm-free hidden states -> router (an unquantised linear) ->
    experts + residual -> head -> log probabilities, eagerly, in pieces and in a graph."""
    m, hidden, inter, experts, top_k, vocab, dtype = 6, 512, 256, 8, 2, 2048, torch.bfloat16
    g = torch.Generator().manual_seed(4)
    x = torch.randn(m, hidden, generator=g).to(dtype).to(DEV)
    gate = (torch.randn(experts, hidden, generator=g) * 0.1).to(dtype).to(DEV)
    stack = lambda name, rows, k, s: torch.from_numpy(np.stack([synth.make_weight(synth.TYPE_IDS[name], rows, k, s + e) for e in range(experts)])).to(DEV)  # noqa: E731
    w13, w2 = stack("Q4_K", 2 * inter, hidden, 1), stack("Q6_K", hidden, inter, 50)
    layer, method = _head("Q6_K", vocab, hidden, dtype)
    ids = torch.randint(0, vocab, (m,), generator=g).to(DEV)

    def step():
        logits = linear.fused_mul_mat_gguf(x, gate, 30)
        y = x + 1e-4 * fused_moe.moe_layer_gguf(x, logits, w13, w2, 12, 14, top_k)
        return y, logprobs.head_logprobs(method, layer, y, ids, 5)

    y, got = step()
    z = method.apply(layer, y)
    _check(z, ids, 5, got)
    pieces = logprobs.head_logprobs(method, layer, y[:2], ids[:2], 5, max_logit_bytes=1)          # a row at a time
    assert pieces.top_ids.shape == (2, 5) and torch.allclose(pieces.logprobs, got.logprobs[:2], atol=0.05)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy, gl = step()
    graph.replay()
    torch.cuda.synchronize()
    _check(method.apply(layer, gy), ids, 5, gl)
    with pytest.raises(RuntimeError, match="token_ids"):
        logprobs.head_logprobs(method, layer, y, ids[:3], 5)
