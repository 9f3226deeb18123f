"""Refusals of the mixture-of-experts layer and of the log probabilities: on CPU tensors every check runs and a clean call ends in
"must be CUDA tensors", as for the products; the C entry points refuse bad arguments before they touch the GPU."""

import ctypes as C

import pytest
import torch

import gsq_b200  # noqa: F401
from gsq_b200 import _cabi, logprobs
from gsq_b200.quantization import fused_moe


def _moe(**kw):
    m, e, k, hidden, inter, t13, t2 = 3, 4, 2, 512, 256, 12, 14
    bs = {12: 144, 14: 210, 21: 110, 23: 136, 29: 56}
    a = {"x": torch.zeros(m, hidden, dtype=torch.bfloat16), "w13": torch.zeros(e, 2 * inter, hidden // 256 * bs[t13], dtype=torch.uint8),
         "w2": torch.zeros(e, hidden, inter // 256 * bs[t2], dtype=torch.uint8), "topk_weights": torch.zeros(m, k),
         "topk_ids": torch.zeros(m, k, dtype=torch.int32), "w13_type": t13, "w2_type": t2}
    a.update(kw)
    return fused_moe.fused_moe_gguf(**a)


MOE = {
    "clean": ({}, "must be CUDA tensors"),
    "x 1-D": ({"x": torch.zeros(512)}, "X must be 2-D"),
    "x int": ({"x": torch.zeros(3, 512, dtype=torch.int32)}, "fp32, fp16 or bf16"),
    "x transposed": ({"x": torch.zeros(512, 3, dtype=torch.bfloat16).t()}, "inner stride"),
    "x of another size": ({"x": torch.zeros(3, 768, dtype=torch.bfloat16)}, "W13 rows of"),
    "x not in superblocks": ({"x": torch.zeros(3, 500, dtype=torch.bfloat16)}, "multiples of 256"),
    "w13 2-D": ({"w13": torch.zeros(512, 288, dtype=torch.uint8)}, "W13 and W2 must be"),
    "w13 float": ({"w13": torch.zeros(4, 512, 288)}, "must be uint8"),
    "w13 of other experts": ({"w13": torch.zeros(5, 512, 288, dtype=torch.uint8)}, "same experts"),
    "w13 odd rows": ({"w13": torch.zeros(4, 511, 288, dtype=torch.uint8)}, "multiples of 256"),
    "w13 strided": ({"w13": torch.zeros(4, 512, 576, dtype=torch.uint8)[..., :288]}, "contiguous"),
    "w13 misaligned": ({"w13": torch.zeros(4 * 512 * 288 + 1, dtype=torch.uint8)[1:].view(4, 512, 288)}, "16-byte aligned"),
    "w2 row bytes": ({"w2": torch.zeros(4, 512, 144, dtype=torch.uint8)}, "W2 must be"),
    "w2 rows": ({"w2": torch.zeros(4, 256, 210, dtype=torch.uint8)}, "W2 must be"),
    "type": ({"w13_type": 2}, "unsupported ggml type 2"),
    "type w2": ({"w2_type": 30}, "unsupported ggml type 30"),
    "ids rows": ({"topk_ids": torch.zeros(2, 2, dtype=torch.int32)}, "topk_weights and topk_ids"),
    "ids float": ({"topk_ids": torch.zeros(3, 2)}, "int32 or int64"),
    "weights int": ({"topk_weights": torch.zeros(3, 2, dtype=torch.int32)}, "floating point"),
    "top_k 0": ({"topk_ids": torch.zeros(3, 0, dtype=torch.int32), "topk_weights": torch.zeros(3, 0)}, "top_k=0"),
    "top_k 33": ({"topk_ids": torch.zeros(3, 33, dtype=torch.int32), "topk_weights": torch.zeros(3, 33)}, "top_k=33"),
    "gradient": ({"x": torch.zeros(3, 512, requires_grad=True)}, "no gradient"),
    "gradient of the weights": ({"topk_weights": torch.zeros(3, 2, requires_grad=True)}, "no gradient"),
}


@pytest.mark.parametrize("name", list(MOE))
def test_experts(name):
    kw, message = MOE[name]
    with pytest.raises(RuntimeError, match=message):
        _moe(**kw)
    if "gradient" in name:
        with torch.no_grad(), pytest.raises(RuntimeError, match="must be CUDA"):
            _moe(**kw)
    assert not torch.cuda.is_initialized()


def test_names():
    for kw in ({"activation": "relu"}, ):
        with pytest.raises(ValueError, match="unsupported activation"):
            _moe(**kw)
    with pytest.raises(ValueError, match="unsupported scoring"):
        fused_moe.moe_route(torch.zeros(2, 4), 2, scoring="linear")


ROUTE = {
    "clean": ((torch.zeros(2, 8), 2), {}, "must be CUDA"),
    "1-D": ((torch.zeros(8), 2), {}, "router logits"),
    "int": ((torch.zeros(2, 8, dtype=torch.int32), 2), {}, "fp32, fp16 or bf16"),
    "transposed": ((torch.zeros(8, 2).t(), 2), {}, "inner stride"),
    "top_k 0": ((torch.zeros(2, 8), 0), {}, "top_k=0"),
    "top_k past the experts": ((torch.zeros(2, 8), 9), {}, "top_k=9"),
    "top_k past the limit": ((torch.zeros(2, 64), 33), {}, "top_k=33"),
    "too many experts": ((torch.zeros(2, 1025), 2), {}, "at most 1024 experts"),
    "bias size": ((torch.zeros(2, 8), 2), {"bias": torch.zeros(7)}, "bias must be"),
    "bias type": ((torch.zeros(2, 8), 2), {"bias": torch.zeros(8, dtype=torch.float16)}, "bias must be"),
    "bias strided": ((torch.zeros(2, 8), 2), {"bias": torch.zeros(16)[::2]}, "bias must be"),
    "gradient": ((torch.zeros(2, 8, requires_grad=True), 2), {}, "no gradient"),
}


@pytest.mark.parametrize("name", list(ROUTE))
def test_route(name):
    args, kw, message = ROUTE[name]
    with pytest.raises(RuntimeError, match=message):
        fused_moe.moe_route(*args, **kw)


def test_layer():
    x, w13, w2 = torch.zeros(3, 512), torch.zeros(4, 512, 288, dtype=torch.uint8), torch.zeros(4, 512, 210, dtype=torch.uint8)
    for logits, message in ((torch.zeros(3, 4), "must be CUDA"), (torch.zeros(2, 4), "logits of 2 tokens"), (torch.zeros(3, 5), "router logits must be")):
        with pytest.raises(RuntimeError, match=message):
            fused_moe.moe_layer_gguf(x, logits, w13, w2, 12, 14, 2)


LOGPROBS = {
    "clean": ((torch.zeros(2, 100), torch.zeros(2, dtype=torch.int64), 5), "must be CUDA"),
    "1-D": ((torch.zeros(100), torch.zeros(1, dtype=torch.int64), 5), "logits must be"),
    "no vocabulary": ((torch.zeros(2, 0), torch.zeros(2, dtype=torch.int64), 5), "logits must be"),
    "double": ((torch.zeros(2, 100, dtype=torch.float64), torch.zeros(2, dtype=torch.int64), 5), "fp32, fp16 or bf16"),
    "transposed": ((torch.zeros(100, 2).t(), torch.zeros(2, dtype=torch.int64), 5), "inner stride"),
    "ids rows": ((torch.zeros(2, 100), torch.zeros(3, dtype=torch.int64), 5), "token_ids must be"),
    "ids float": ((torch.zeros(2, 100), torch.zeros(2), 5), "int32 or int64"),
    "top_n -1": ((torch.zeros(2, 100), torch.zeros(2, dtype=torch.int64), -1), "top_n=-1"),
    "top_n 33": ((torch.zeros(2, 100), torch.zeros(2, dtype=torch.int64), 33), "top_n=33"),
    "gradient": ((torch.zeros(2, 100, requires_grad=True), torch.zeros(2, dtype=torch.int64), 5), "no gradient"),
}


@pytest.mark.parametrize("name", list(LOGPROBS))
def test_logprobs(name):
    args, message = LOGPROBS[name]
    with pytest.raises(RuntimeError, match=message):
        logprobs.token_logprobs(*args)


def test_c_entry_points_refuse_before_the_gpu():
    lib, w, one = _cabi.lib, _cabi.Moe(16, 16, 12, 14, 4, 512, 256, 0), C.c_void_p(256)
    ws = lib.gsq_moe_workspace_bytes(3, 512, 256, 2)
    assert ws > 0 and lib.gsq_moe_workspace_bytes(0, 512, 256, 2) == 0

    def experts(m=3, top_k=2, dtype=2, x=one, y=one, weights=one, ids=one, size=ws, space=one, **kw):
        g = _cabi.Moe(16, 16, 12, 14, 4, 512, 256, 0)
        for k, v in kw.items():
            setattr(g, k, v)
        return lib.gsq_moe_experts(C.byref(g), x, dtype, m, 512, weights, ids, 0, top_k, y, 512, space, size, None)

    assert experts(m=0) == _cabi.OK
    bad = [{"w13": None}, {"w2": None}, {"w13": 8}, {"w13_type": 2}, {"w2_type": 30}, {"hidden": 500}, {"inter": 100}, {"inter": 0}, {"activation": 2},
           {"experts": 0}, {"dtype": 99}, {"x": None}, {"y": None}, {"weights": None}, {"ids": None}, {"top_k": 0}, {"m": -1}]
    for kw in bad:
        assert experts(**kw) == _cabi.ERR_UNSUPPORTED, kw
    for kw in ({"experts": 1025}, {"top_k": 33}, {"m": 65537}):
        assert experts(**{"size": 1 << 60, **kw}) == _cabi.ERR_TOO_LARGE, kw
    for kw in ({"space": None}, {"size": ws - 1}, {"space": C.c_void_p(128)}):
        assert experts(**kw) == _cabi.ERR_SCRATCH, kw

    def route(m=3, experts=8, top_k=2, weights=one, ids=one, **kw):
        r = _cabi.MoeRouter(256, 0, 8, 0, 1, None, 1.0)
        for k, v in kw.items():
            setattr(r, k, v)
        return lib.gsq_moe_route(C.byref(r), m, experts, top_k, weights, ids, None)

    assert route(m=0) == _cabi.OK
    for kw in ({"logits": None}, {"dtype": 99}, {"scoring": 2}, {"top_k": 0}, {"top_k": 9}, {"experts": 0}, {"weights": None}, {"ids": None}):
        assert route(**kw) == _cabi.ERR_UNSUPPORTED, kw
    for kw in ({"experts": 1025}, {"experts": 64, "top_k": 33}):
        assert route(**kw) == _cabi.ERR_TOO_LARGE, kw

    def lp(m=2, vocab=10, dtype=0, logits=one, ids=one, top_n=0, out=one, top=None):
        return lib.gsq_token_logprobs(logits, dtype, m, vocab, 10, ids, top_n, out, one, one, top, top, None)

    assert lp(m=0) == _cabi.OK
    for kw in ({"vocab": 0}, {"m": -1}, {"dtype": 3}, {"logits": None}, {"ids": None}, {"out": None}, {"top_n": -1}, {"top_n": 2}):
        assert lp(**kw) == _cabi.ERR_UNSUPPORTED, kw
    for kw in ({"vocab": 1 << 31}, {"top_n": 33}, {"m": 1 << 31}):
        assert lp(**kw) == _cabi.ERR_TOO_LARGE, kw
    del w


def test_empty_calls_on_the_host():
    with pytest.raises(RuntimeError, match="must be CUDA"):
        logprobs.token_logprobs(torch.zeros(0, 10), torch.zeros(0, dtype=torch.int64), 3)


def test_c_entry_points_refuse_pointers_between_elements():
    lib, at = _cabi.lib, C.c_void_p
    g, size = _cabi.Moe(16, 16, 12, 14, 4, 512, 256, 0), lib.gsq_moe_workspace_bytes(3, 512, 256, 2)

    def experts(x=256, y=256, weights=256, ids=256, ids_64=0, dtype=0):
        return lib.gsq_moe_experts(C.byref(g), at(x), dtype, 3, 512, at(weights), at(ids), ids_64, 2, at(y), 512, at(256), size, None)

    for kw in ({"x": 258}, {"x": 257, "dtype": 2}, {"y": 258}, {"y": 257, "dtype": 1}, {"weights": 258}, {"ids": 258}, {"ids": 260, "ids_64": 1}):
        assert experts(**kw) == _cabi.ERR_UNSUPPORTED, kw
    for logits, dtype, bias, weights, ids in ((258, 0, None, 256, 256), (257, 2, None, 256, 256), (256, 0, 258, 256, 256), (256, 0, None, 258, 256), (256, 0, None, 256, 258)):
        r = _cabi.MoeRouter(logits, dtype, 8, 0, 1, bias, 1.0)
        assert lib.gsq_moe_route(C.byref(r), 3, 8, 2, at(weights), at(ids), None) == _cabi.ERR_UNSUPPORTED
    good = [256] * 7
    for i, v in ((0, 257), (1, 260), (2, 258), (3, 260), (4, 258), (5, 258), (6, 260)):
        p = [at(v if i == j else q) for j, q in enumerate(good)]
        assert lib.gsq_token_logprobs(p[0], 2, 2, 100, 100, p[1], 3, p[2], p[3], p[4], p[5], p[6], None) == _cabi.ERR_UNSUPPORTED
