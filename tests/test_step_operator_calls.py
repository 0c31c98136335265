"""Calls of the operators of a verifying step that have to be refused before anything runs on a GPU, and what their arguments know on the host."""
import pytest
import torch

from sprout_lm_amd import ops


def shared(batch, rows, prefix=100, **options):
    """`attention_shared` of four heads in two groups, with operands that no kernel may see."""
    q = torch.zeros(max(rows, 1), 256)
    ops.attention_shared(q, 256, torch.zeros(9, 2, 16, 64), torch.zeros(9, 2, 64, 16), torch.zeros(batch.n_seqs, 9, dtype=torch.int32), batch, prefix,
                         torch.zeros(rows, 256), 4, 2, 64, 0.1, **options)


def test_queries_that_out_has_no_rows_for():
    for q_lens, rows in (([16], 1), ([16], 15), ([5, 1], 5), ([1, 40, 3], 43)):
        batch = ops.AttentionBatch.build(q_lens, [100 + q for q in q_lens], "cpu")
        assert batch.rows == sum(q_lens)
        with pytest.raises(ops.KernelError, match="rows"):
            shared(batch, rows)
        with pytest.raises(ops.KernelError, match="current GPU"):      # (all is well but for where the operands lie)
            shared(batch, sum(q_lens))
    whole = ops.AttentionBatch.build([2], [102], "cpu")
    unknown = ops.AttentionBatch(whole.q_start, whole.q_len, whole.ctx_len, 1, whole.lists, 0, 102, first_query=100)
    with pytest.raises(ops.KernelError, match="unknown number of rows"):
        shared(unknown, 2)
    assert ops.AttentionBatch.build([0], [7], "cpu").rows == 0
