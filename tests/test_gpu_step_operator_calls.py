"""Calls of the operators of a verifying step that their documentation allows, beside those of each operator's own tests."""
import math

import pytest
import torch

from tests import test_gpu_attention_shared as shared

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def test_rows_behind_the_batch_are_no_work():
    """One query, room for five thousand: the same bits, the same workspace as with room for one."""
    from sprout_lm_amd import ops
    got, asked = [], []
    for extra in (0, 5000):
        case = shared.Case(BF16, 64, 8, 32, 16, 100, [(1, 7)], extra_rows=extra)
        case.q[1:] = math.nan

        def workspace(n):
            asked.append(n)
            return torch.full((n,), math.nan, device=DEV)
        got.append(case.run(workspace=workspace))
        case.check(got[-1], *case.definition())
    assert torch.equal(got[0], got[1]) and asked[0] == asked[1]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cap", [0.5, 50.0, 1.0e6])
def test_caps_below_and_far_above_the_scores(cap, dtype):
    """A score far below its cap is the score but for its last places (10 times 2^-24 of it at most, less than what the product's own roundings are
    allowed): scores reach some 8 here."""
    shared.check(shared.Case(dtype, 4, 2, 64, 16, 140, [(1, 20), (3, 5)], seed=3), scores="capped", softcap=cap, definition={"cap": cap})
