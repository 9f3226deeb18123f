"""Expert stacks of a GGUF file (gguf_load.load_experts): placement of gate, up and down bytes, a rank's share, refusals; on the
GPU, the layer over what was loaded."""

import numpy as np
import pytest
import torch

from gsq_b200 import gguf_load, synth

NAMES = ("blk.0.ffn_gate_exps.weight", "blk.0.ffn_up_exps.weight", "blk.0.ffn_down_exps.weight")
E, HIDDEN, INTER = 5, 768, 256


def _tensors(t13="Q4_K", t2="Q6_K", seed=40):
    stack = lambda t, rows, k, s: np.stack([synth.make_weight(synth.TYPE_IDS[t], rows, k, s + e) for e in range(E)])  # noqa: E731
    return {NAMES[0]: (synth.TYPE_IDS[t13], stack(t13, INTER, HIDDEN, seed)), NAMES[1]: (synth.TYPE_IDS[t13], stack(t13, INTER, HIDDEN, seed + 10)),
            NAMES[2]: (synth.TYPE_IDS[t2], stack(t2, HIDDEN, INTER, seed + 20)), "norm": (0, np.ones(4, np.float32))}


class HostStager:
    """to_device without a device, in copies of two rows."""

    def to_device(self, src, dst):
        for i in range(0, src.shape[0], 2):
            dst[i:i + 2, :src.shape[1]].copy_(torch.from_numpy(np.ascontiguousarray(src[i:i + 2])))


@pytest.mark.parametrize("chunk", [64 << 20, 1000])       # the second: an expert that is larger than a chunk
@pytest.mark.parametrize("part", [None, slice(1, 4), slice(3, None)])
def test_bytes_are_placed(monkeypatch, chunk, part):
    monkeypatch.setattr(gguf_load, "_CHUNK", chunk)
    t = _tensors()
    w13, w2, t13, t2 = gguf_load.load_experts(t, *NAMES, device="cpu", experts=part, stager=HostStager())
    keep = part or slice(None)
    assert (t13, t2) == (12, 14) and w13.is_contiguous() and w2.is_contiguous()
    assert np.array_equal(w13.numpy(), np.concatenate([t[NAMES[0]][1], t[NAMES[1]][1]], 1)[keep])
    assert np.array_equal(w2.numpy(), t[NAMES[2]][1][keep])


def _swap(**kw):
    t = _tensors()
    t.update({NAMES[int(k[1:])]: v for k, v in kw.items()})
    return t


@pytest.mark.parametrize("tensors,kw,message", [
    (_swap(n1=_tensors("IQ4_XS")[NAMES[1]]), {}, "differ in type or shape"),
    (_swap(n1=(12, np.zeros((E, INTER, 288), np.uint8))), {}, "differ in type or shape"),
    (_swap(n2=(14, np.zeros((E, HIDDEN, 420), np.uint8))), {}, "does not fit"),
    (_swap(n2=(14, np.zeros((E + 1, HIDDEN, 210), np.uint8))), {}, "does not fit"),
    (_swap(n2=(14, np.zeros((E, 512, 210), np.uint8))), {}, "does not fit"),
    (_swap(n0=(12, np.zeros((INTER, 432), np.uint8))), {}, "not a stack"),
    (_swap(n0=(2, np.zeros((E, INTER, 432), np.uint8))), {}, "not a stack"),
    (_swap(), {"experts": slice(5, None)}, "takes none"),
    (_swap(), {"experts": slice(0, 5, 2)}, "leaves gaps"),
])
def test_refusals(tensors, kw, message):
    with pytest.raises(ValueError, match=message):
        gguf_load.load_experts(tensors, *NAMES, device="cpu", stager=HostStager(), **kw)


@pytest.mark.gpu
def test_loaded_layer():
    from gsq_b200.quantization import fused_moe
    from oracle import moe

    t = _tensors()
    whole = gguf_load.load_experts(t, *NAMES)
    raw13 = np.concatenate([t[NAMES[0]][1], t[NAMES[1]][1]], 1)
    assert np.array_equal(whole[0].cpu().numpy(), raw13) and np.array_equal(whole[1].cpu().numpy(), t[NAMES[2]][1])
    x = torch.from_numpy(synth.make_activation(6, HIDDEN, 77, 1e-3)).cuda()
    logits = torch.randn(6, E, generator=torch.Generator().manual_seed(3)).cuda()
    y = fused_moe.moe_layer_gguf(x, logits, *whole, 3)
    w, ids = fused_moe.moe_route(logits, 3)
    ref, bound = moe.experts(x.cpu().numpy(), raw13, t[NAMES[2]][1], 12, 14, w.cpu().numpy(), ids.cpu().numpy())
    assert (np.abs(y.cpu().numpy() - ref) <= bound + 2.0 ** -23 * np.abs(ref) + 1e-7).all()
    # two ranks, three experts and two: their parts add up to the layer (three roundings of fp32 sums more)
    parts = []
    for first, last in ((0, 3), (3, E)):
        share = gguf_load.load_experts(t, *NAMES, experts=slice(first, last))
        parts.append(fused_moe.fused_moe_gguf(x, share[0], share[1], w, torch.where(ids >= first, ids - first, -1), *share[2:]))
    assert (np.abs((parts[0] + parts[1]).cpu().numpy() - ref) <= bound + 2.0 ** -22 * (np.abs(ref) + sum(p.abs().cpu().numpy() for p in parts)) + 1e-7).all()
