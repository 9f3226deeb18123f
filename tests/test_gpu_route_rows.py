"""The choice of the experts at the largest number of tokens that it takes."""

import pytest
import torch

import gsq_b200  # noqa: F401
from gsq_b200.quantization import fused_moe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [2 ** 31 - 1, 2 ** 31 - 5])
def test_tokens_up_to_2_31(m):
    if torch.cuda.mem_get_info()[0] < 32 << 30:
        pytest.skip("not enough device memory")
    logits = torch.zeros(m, 1, dtype=torch.float16, device="cuda")
    logits[-3] = -float("inf")
    w, ids = fused_moe.moe_route(logits, 1, scale=2.0)
    assert w.shape == ids.shape == (m, 1)
    for part_w, part_ids in zip(w.view(-1)[:-5].split(2 ** 28), ids.view(-1)[:-5].split(2 ** 28)):
        assert bool((part_w == 2).all()) and not part_ids.any()
    assert w[-5:, 0].tolist() == [2, 2, 0, 2, 2] and ids[-5:, 0].tolist() == [0, 0, -1, 0, 0]
