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
