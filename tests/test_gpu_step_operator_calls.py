"""Calls of the operators of a verifying step that their documentation allows, beside those of each operator's own tests."""
import math

import pytest
import torch

from tests import test_gpu_attention_shared as shared

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def test_many_rows_behind_the_batch():
    """One query, room for five thousand of 64 heads: more than the launches' grids have blocks for along their second axis."""
    case = shared.Case(BF16, 64, 8, 32, 16, 100, [(1, 7)], extra_rows=5000)
    case.q[1:] = math.nan
    got = case.run()
    case.check(got, *case.definition())


def test_a_recorded_call_replayed_with_more_of_outs_rows():
    """Recorded with two queries in eight rows, replayed with seven in the same two tiles."""
    from sprout_lm_amd import ops
    few, many = (shared.Case(BF16, 4, 2, 64, 16, 100, seqs, extra_rows=8 - sum(q for q, _ in seqs), seed=4) for seqs in ([(1, 40), (1, 40)], [(4, 40), (3, 40)]))
    many.fill()
    k, v, tables = many.k.to(DEV), many.v.to(DEV), many.tables.to(DEV)
    batch = ops.AttentionBatch.build([1, 1], [140, 140], DEV)
    q, out = few.q.to(DEV), torch.full((8, 256), 7.0, dtype=BF16, device=DEV)
    room = torch.full((1 << 20,), math.nan, device=DEV)
    call = lambda: ops.attention_shared(q, 256, k, v, tables, batch, 100, out, 4, 2, 64, 0.125, workspace=lambda n: room[:n])
    call()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    for t, now in ((batch.q_start, [0, 4]), (batch.q_len, [4, 3]), (q, many.q)):
        t.copy_(torch.as_tensor(now))
    for _ in range(3):
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        many.check(out[:7].double().cpu(), *many.definition())
        assert (out[7:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("cap", [0.5, 50.0, 1.0e6])
def test_caps_below_and_far_above_the_scores(cap, dtype):
    """A score far below its cap is the score but for its last places (10 times 2^-24 of it at most, less than what the product's own roundings are
    allowed): scores reach some 8 here."""
    shared.check(shared.Case(dtype, 4, 2, 64, 16, 140, [(1, 20), (3, 5)], seed=3), scores="capped", softcap=cap, definition={"cap": cap})
