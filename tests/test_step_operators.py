"""What the operators of a verifying step refuse without a GPU: sizes and missing operands at the C interface, tensors at the Python face."""
import pytest
import torch

from sprout_lm_amd import ops


def refused(call, *args, match):
    from sprout_lm_amd.ops.library import check
    with pytest.raises(ops.KernelError, match=match):
        check(call(*args))


def test_shared_attention_refuses_at_the_c_interface():
    lib = ops.library()
    #       stream dtype q stride k  v  tables max table prefix start len ctx tiles n max_ctx T ws floats out nq nkv hd page pages scale cap sinks
    good = [None, 1, 16, 256, 16, 16, 16, 9, 16, 100, 16, 16, 16, 16, 2, 110, 2, 16, 1 << 40, 16, 4, 2, 64, 16, 9, 0.1, 0.0, None]
    for at, value, match in ((1, 2, "dtype"), (20, 3, "divide"), (22, 257, "head size"), (22, 0, "head size"), (23, 0, "geometry"), (7, 0, "geometry"), (7, 1 << 28, "geometry"), (16, 1, "rows"), (2, None, "null"),
                             (8, None, "null"), (3, 255, "stride"), (9, 110, "fit"), (15, 145, "fit"), (9, -1, "fit"), (26, -1.0, "cap"), (18, 10, "workspace"),
                             (17, None, "workspace")):
        refused(lib.sp_attention_shared, *good[:at], value, *good[at + 1:], match=match)
    assert lib.sp_attention_shared(*good[:14], 0, *good[15:]) == 0      # no queries: nothing to do
    assert lib.sp_attention_shared_workspace_floats(1, 257, 4, 2, 2, 2, 100, 110) == 0
    assert lib.sp_attention_shared_workspace_floats(1, 64, 4, 2, 2, 2, 100, 110) >= 2 * 2 * 4 * 66


def test_drafts_refuse_at_the_c_interface():
    lib = ops.library()
    #       stream dtype logits rows vocab tokens starts lens sequences uniform temperature drafter drafted rows accepted next workspace floats
    good = [None, 0, 16, 4, 50, 16, 16, 16, 2, 16, 16, 16, 3, 16, 16, 16, 16, 1 << 40]
    for at, value, match in ((1, 2, "dtype"), (3, -1, "sizes"), (4, 0, "sizes"), (4, (1 << 30) + 1, "sizes"), (3, 0, "rows"), (3, 32768, "rows"), (8, 65536, "sequences"), (2, None, "null"), (9, None, "null"),
                             (11, None, "together"), (13, None, "together"), (16, None, "workspace"), (16, 4, "workspace"), (17, 3, "workspace")):
        refused(lib.sp_verify_drafts, *good[:at], value, *good[at + 1:], match=match)
    assert lib.sp_verify_drafts(*good[:8], 0, *good[9:]) == 0
    assert ops.verify_workspace_floats(0, 2, 50) == 0 < ops.verify_workspace_floats(4, 2, 50)


def test_4_bit_products_refuse_at_the_c_interface():
    lib = ops.library()
    #       stream dtype x  words dtype scales dtype bias mode dtype out T  N  K  group workspace floats
    good = [None, 1, 16, 16, 1, 16, 0, None, 0, 1, 16, 2, 20, 64, 32, None, 0]
    for at, value, match in ((1, 2, "dtypes"), (4, 2, "dtypes"), (6, 2, "dtypes"), (8, 1, "stores"), (8, 2, "stores"), (9, 0, "stores"), (11, -1, "groups"), (12, 0, "groups"), (13, 0, "groups"),
                             (14, 16, "groups"), (2, None, "null"), (5, None, "null"), (3, 20, "16 bytes"), (5, 8, "16 bytes"), (11, 1 << 21, "tokens"), (13, (1 << 24) + 1, "tokens")):
        refused(lib.sp_gemm_q4, *good[:at], value, *good[at + 1:], match=match)
    assert lib.sp_gemm_q4(*good[:11], 0, *good[12:]) == 0
    refused(lib.sp_q4_pack, None, 16, 2, 16, 20, 64, 32, 16, 16, match="dtype")
    refused(lib.sp_q4_pack, None, None, 1, 16, 20, 64, 32, 16, 16, match="null")
    refused(lib.sp_q4_quantize, None, 3, 16, 20, 64, 32, 16, 1, 16, match="dtypes")
    refused(lib.sp_q4_quantize, None, 1, 16, 20, 64, 48, 16, 1, 16, match="groups")
    assert lib.sp_q4_words(20, 130) == 2 * 2 * 256 and lib.sp_q4_words(0, 5) == 0


def test_tensors_must_be_on_the_gpu():
    ints, batch = torch.zeros(2, dtype=torch.int32), ops.AttentionBatch.build([1, 1], [101, 104], "cpu")
    with pytest.raises(ops.KernelError, match="current GPU"):
        ops.attention_shared(torch.zeros(2, 256), 256, torch.zeros(9, 2, 16, 64), torch.zeros(9, 2, 64, 16), torch.zeros(2, 9, dtype=torch.int32), batch, 100,
                             torch.zeros(2, 256), 4, 2, 64, 0.1)
    with pytest.raises(ops.KernelError, match="current GPU"):
        ops.verify_drafts(torch.zeros(2, 5), ints, ints, ints, torch.zeros(2), ints, ints, torch.zeros(100))
    with pytest.raises(ops.KernelError, match="current GPU"):
        ops.q4_quantize(torch.zeros(4, 64), 32)
    with pytest.raises(ops.KernelError, match="current GPU"):
        ops.q4_pack(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2), 32)


def test_a_batch_knows_its_first_query():
    assert ops.AttentionBatch.build([1, 3, 0], [101, 104, 7], "cpu").first_query == 100
    assert ops.AttentionBatch.build([0], [7], "cpu").first_query is None


def test_random_numbers_of_a_sequence_are_its_own():
    from sprout_lm_amd.sampling.sampler import uniform_numbers
    both = uniform_numbers([5, 2 ** 63 - 1], [0, 7], [400, 600])
    assert both.dtype == torch.float32 and both.shape == (1000,) and 0 <= float(both.min()) and float(both.max()) < 1
    assert torch.equal(uniform_numbers([2 ** 63 - 1], [7], [600]), both[400:])
    assert not torch.equal(uniform_numbers([5], [1], [400]), both[:400]) and not torch.equal(uniform_numbers([6], [0], [400]), both[:400])
    assert uniform_numbers([], [], []).shape == (0,)
    assert abs(float(uniform_numbers(list(range(100)), [3] * 100, [100] * 100).double().mean()) - 0.5) < 5 * (1 / 12 / 10000) ** 0.5


def test_the_sampler_refuses_rows_that_do_not_fit():
    from sprout_lm_amd.sampling import Sampler, SamplingParams
    sampler, one = Sampler(torch.device("cpu"), 5), [SamplingParams()]
    for logits, tokens, lens, params, counters in ((3, 2, [2], one, [0]), (2, 3, [2], one, [0]), (2, 2, [2, 0], one * 2, [0, 0]), (2, 2, [2], one * 2, [0]), (2, 2, [2], one, [])):
        with pytest.raises(ValueError, match="verify"):
            sampler.verify(torch.zeros(logits, 5), torch.zeros(tokens, dtype=torch.int32), lens, params, counters)


def test_4_bit_weights_know_their_sizes():
    words, scales = torch.zeros(2 * 2 * 256, dtype=torch.int32), torch.zeros(5, 32)
    assert ops.Q4Matrix(20, 130, 32, words, scales).nbytes() == 4096 + 640
    for args in ((20, 130, 16, words, scales), (33, 130, 32, words, scales), (20, 257, 32, words, scales), (20, 130, 64, words, scales), (20, 130, 32, words.float(), scales)):
        with pytest.raises(ops.KernelError):
            ops.Q4Matrix(*args)
