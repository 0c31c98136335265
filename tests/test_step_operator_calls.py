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


def two_entries():
    """Five tokens from position 0 and three from position 6, and the cache they lie in."""
    from sprout_lm_amd.cache import CacheManager, PagedKVSpec
    from sprout_lm_amd.engine.batch import StepEntry
    cache = CacheManager([PagedKVSpec(1, 16)], block_size=4, num_blocks=8, max_sequences=3)
    a, b = cache.create(), cache.create()
    assert cache.reserve(a, 5) and cache.reserve(b, 9)
    cache.commit(b, 6)
    return cache, [StepEntry(a, [1, 2, 3, 4, 5], [4]), StepEntry(b, [7, 8, 9], [])]


def context(step, cache, **options):
    from sprout_lm_amd.engine.batch import Workspace, context_from
    return context_from(step, [torch.from_numpy(a) for a in step.arrays], len(cache.groups), Workspace("cpu"), torch.float32, **options)


def test_a_recorded_step_does_not_know_where_later_queries_stand(monkeypatch):
    """The step that is recorded stands behind position 6, one that is replayed may stand before it."""
    from sprout_lm_amd.engine import graphs
    from sprout_lm_amd.engine.batch import Workspace, step_arrays
    cache, entries = two_entries()
    step = step_arrays(entries[1:], cache)
    assert context(step, cache).attention.first_query == 6 and context(step, cache).attention.rows == 3
    zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *size, pin_memory=False, **kw: zeros(*size, **kw))      # (without a GPU there is no pinned memory)
    runner = type("Runner", (), dict(cache=cache, device="cpu", dtype=torch.float32, attention_kind=0))()
    recorded = graphs._PortionGraph(runner, step, 16, Workspace("cpu")).ctx
    assert recorded.host == {} and recorded.attention.first_query is None and recorded.attention.rows == 3
    with pytest.raises(ops.KernelError, match="None does not stand behind"):
        shared(recorded.attention, 3, prefix=6)


def test_the_lowest_position_is_looked_for_when_asked():
    """A step's host work does not grow for a number that only `attention_shared` reads; entries without tokens have no query."""
    from sprout_lm_amd.engine.batch import StepEntry, step_arrays
    cache, entries = two_entries()
    step = step_arrays(entries, cache)
    looks = []

    class Watched(dict):
        def __getitem__(self, name):
            looks.append(name)
            return super().__getitem__(name)
    step.host = Watched(step.host)
    ctx = context(step, cache)
    assert looks == []
    assert ctx.attention.first_query == 0 and ctx.attention.first_query == 0 and len(looks) == 1
    empty = StepEntry(cache.create(), [], [])
    assert context(step_arrays([empty, entries[1]], cache), cache).attention.first_query == 6
    assert context(step_arrays([empty], cache), cache).attention.first_query is None


def test_the_sampler_gives_no_token_outside_its_vocabulary(monkeypatch):
    """Rows longer than the vocabulary (a padded head): an id behind it is refused as `Sampler.sample` does, drawn or kept as a draft."""
    from sprout_lm_amd.sampling import NonFiniteLogits, Sampler, SamplingParams
    sampler, tokens = Sampler(torch.device("cpu"), 5), torch.tensor([1, 6, 2], dtype=torch.int32)

    def verify(held, following):
        def answer(logits, tokens, starts, lens, uniform, accepted, next_token, *rest):
            accepted[:], next_token[:] = held, following
        monkeypatch.setattr(ops, "verify_drafts", answer)
        return sampler.verify(torch.zeros(3, 8), tokens, [3], [SamplingParams()], [0])
    assert verify(0, 4) == [[4]]
    for held, following in ((0, 5), (0, -1), (1, 3), (2, 3)):      # drawn: 5; refused by the kernel; the draft 6 kept
        with pytest.raises(NonFiniteLogits):
            verify(held, following)


def test_shared_attention_refuses_sizes_that_no_index_holds():
    from sprout_lm_amd.ops.library import check
    lib = ops.library()
    #       stream dtype q stride k  v  tables max table prefix start len ctx tiles n max_ctx T ws floats out nq nkv hd page pages scale cap sinks
    good = [None, 1, 16, 1 << 30, 16, 16, 16, 9, 16, 100, 16, 16, 16, 16, 2, 110, 2, 16, 1 << 60, 16, 4, 2, 64, 16, 9, 0.1, 0.0, None]
    #       rows of heads; a token's numbers; keys; blocks of 128 rows of many groups
    for changes, match in (({16: 1 << 29}, "indexes"), ({20: 1 << 25, 21: 1 << 25, 3: 2 ** 31 - 1}, "indexes"), ({7: 2 ** 27 - 1, 15: (1 << 30) + 1}, "indexes"),
                           ({16: 1 << 17, 20: 1 << 13, 21: 1 << 13, 9: 64, 14: 1 << 17}, "launch")):
        args = [changes.get(i, a) for i, a in enumerate(good)]
        with pytest.raises(ops.KernelError, match=match):
            check(lib.sp_attention_shared(*args))
        floats = lib.sp_attention_shared_workspace_floats(args[1], args[22], args[20], args[21], args[16], args[14], args[9], args[15])
        assert (floats == 0) == (match == "indexes")


@pytest.mark.parametrize("cap", [float("inf"), float("nan"), 0.0, -1.0])
def test_shared_attention_refuses_caps_that_are_no_number(cap):
    """An infinite cap would make every score infinity times zero."""
    from sprout_lm_amd.ops.library import check
    batch = ops.AttentionBatch.build([1], [101], "cpu")
    with pytest.raises(ops.KernelError, match="positive cap"):
        shared(batch, 1, scores="capped", softcap=cap)
    with pytest.raises(ops.KernelError, match="current GPU"):
        shared(batch, 1, scores="scaled_dot", softcap=cap)      # (no cap is looked at)
    args = [None, 1, 16, 256, 16, 16, 16, 9, 16, 100, 16, 16, 16, 16, 2, 110, 2, 16, 1 << 40, 16, 4, 2, 64, 16, 9, 0.1, cap, None]
    if cap != 0.0:
        with pytest.raises(ops.KernelError, match="cap"):
            check(ops.library().sp_attention_shared(*args))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64, torch.int32])
def test_4_bit_weights_refuse_scales_that_no_kernel_reads(dtype):
    words = torch.zeros(2 * 2 * 256, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="scales"):
        ops.Q4Matrix(20, 130, 32, words, torch.zeros(5, 32).to(dtype))
    for taken in (torch.float32, torch.bfloat16):
        assert ops.Q4Matrix(20, 130, 32, words, torch.zeros(5, 32).to(taken)).group == 32
