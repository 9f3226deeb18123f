"""Kernels that start while the kernel before them still runs (programmatic launch): what that one writes is not read-only for their
lifetime, so they may not read it on the non-coherent path, however late they wait for it. Weights, which no kernel before writes, may be."""

import os
import re

import pytest

import gsq_b200

CSRC = os.path.join(os.path.dirname(os.path.dirname(gsq_b200.__file__)), "csrc")


def _code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


# files whose kernels read inputs alone (logits, activations, choices), no weights, all of them behind griddepcontrol.wait
@pytest.mark.parametrize("name", ["gsq_logprobs.cu", "gsq_moe.cu", "gsq_quantize.cu", "gsq_planes.cu", "gsq_quant.cuh"])
def test_inputs_are_read_coherently(name):
    code = _code(name)
    assert name == "gsq_quant.cuh" or "griddepcontrol.wait" in code
    assert not re.findall(r"\bldg_stream_\w+|\b__ldg\b|ld\.global\.nc", code)
