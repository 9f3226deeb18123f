"""The gated activations where the gates of a whole block are strongly negative: the 8-bit form takes its scale from the block's largest
value, so an activation that is off by a share of its value there is off by that share in the result.

Weights and activations of one magnitude make every gate -g and every up value +-1 (to 4 roundings), so the activated values are
+-act(-g), which 8 bits hold exactly: the result is act(-g) times the down rows' signed sums."""

import math

import numpy as np
import pytest
import torch

import gsq_b200  # noqa: F401
from gsq_b200 import synth
from gsq_b200.quantization import fused_moe
from oracle import moe

pytestmark = pytest.mark.gpu
H, I = 256, 256


def _rows(name, scales):
    """Rows of 256 equal values: scale (fp16) for each row."""
    d = np.asarray(scales, np.float16).reshape(-1, 1).view(np.uint8)
    if name == "Q6_K":                   # quants 33 - 32, sub-scales 1
        w = np.zeros((len(d), 210), np.uint8)
        w[:, :128], w[:, 128:192], w[:, 192:208], w[:, 208:210] = 0x11, 0xAA, 1, d
    else:                                # Q2_K: quants 1, sub-scales 1, no minima
        w = np.zeros((len(d), 84), np.uint8)
        w[:, :16], w[:, 16:80], w[:, 80:82] = 1, 0x55, d
    return w


@pytest.mark.parametrize("name", ["Q6_K", "Q2_K"])     # the tensor-core products, the dp4a ones
@pytest.mark.parametrize("m", [1, 3])
@pytest.mark.parametrize("act,gates", [("gelu", (0.5, 2, 4, 5, 6, 8, 12)), ("silu", (0.5, 4, 20, 60, 87, 87.75, 88, 88.5))])
def test_strongly_negative_gates(name, m, act, gates):
    t = {**synth.TYPE_IDS, **synth.LOW_BIT_TYPE_IDS}[name]
    sign = np.where(np.random.default_rng(1).random(I) < 0.5, -1.0, 1.0)
    w2 = synth.make_weight(14, H, I, 2)
    values = moe.values(w2, 14)
    x = torch.ones(m, H, device="cuda")
    one, ids = torch.ones(m, 1, device="cuda"), torch.zeros(m, 1, dtype=torch.int32, device="cuda")
    for g in gates:
        w13 = np.concatenate([_rows(name, [-g / H] * I), _rows(name, sign / H)])
        assert np.allclose(moe.values(w13, t).sum(1), np.concatenate([[-g] * I, sign]), rtol=1e-12)
        y = fused_moe.fused_moe_gguf(x, torch.from_numpy(w13[None]).cuda(), torch.from_numpy(w2[None]).cuda(), one, ids, t, 14, act)
        a = -g / (1 + math.exp(g)) if act == "silu" else -0.5 * g * math.erfc(g / math.sqrt(2))
        want, size = a * (values @ sign), abs(a) * np.abs(values).sum(1)
        # the gate: 4 roundings, times the activation's own slope, 1 + g^2 at most; gelu's argument: 2 roundings, times g^2; function, products and
        # sums: 8 steps of erfcf or expf (its argument's rounding: g), 16 roundings behind them
        rel = (4 * (1 + g * g if act == "gelu" else 1 + g) + 2 * (g * g if act == "gelu" else g) + 40) * 2.0 ** -24
        off = np.abs(y.cpu().numpy().astype(np.float64) - want)
        assert (off <= rel * size).all(), (g, float((off / size).max()), rel)
