"""Products with 4-bit weights against the definition in 64 bits; how weights are rounded to 4 bits and laid out."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def weights(N, K, group, seed, scale_dtype=BF16):
    """(codes, scales, what they stand for in float64)"""
    g = torch.Generator().manual_seed(seed)
    groups = -(-K // group)
    c = torch.randint(0, 16, (N, K + K % 2), generator=g, dtype=torch.uint8)
    scales = (torch.rand(N, groups, generator=g) + 0.5).mul_(0.05).to(scale_dtype)
    w = (c[:, :K].double() - 8) * scales.double().repeat_interleave(group, 1)[:, :K]
    return c[:, 0::2] | (c[:, 1::2] << 4), scales, w


def product(x, codes, scales, group, K, **options):
    from sprout_lm_amd import ops
    matrix = ops.q4_pack(codes.to(DEV), scales.to(DEV), group, cols=K)
    out = options.pop("out", None)
    if out is None:
        out = torch.full((x.shape[0], matrix.rows), math.nan, dtype=x.dtype, device=DEV)
    ops.gemm_q4(x.to(DEV), matrix, out, **options)
    return out.double().cpu()


def allowed(x, scales, w, group, dtype, want, more=0.0):
    """Within a group: sums of (code - 8) x taken as (16 + code) x less 24 x, 40 |x| at most a number, each of 2 group products (three
    parts each in float32, whose small ones weigh 2^-8) added with a rounding of 2^-24 of the sums so far; then a product and a sum a group; the result's rounding."""
    K = x.shape[1]
    spread = x.double().abs() @ (40.0 * scales.double().abs().repeat_interleave(group, 1)[:, :K]).t()
    chain = 2 * group * (1.02 if x.dtype == F32 else 1) + 2 * scales.shape[1] + 8
    return 2.0 ** -24 * chain * spread + (2.0 ** -8 if dtype == BF16 else 2.0 ** -24) * (want.abs() + more) + 1e-30


SIZES = [(1, 896, 4864, 128), (1, 16, 128, 32), (5, 37, 160, 32), (16, 100, 256, 64), (17, 48, 896, 128), (33, 130, 320, 64), (64, 64, 512, 128), (2, 1, 32, 32),
         (70, 33, 200, 64), (129, 40, 130, 128), (3, 20, 2, 32), (4, 50, 77, 32), (7, 257, 1000, 64), (48, 4100, 384, 128), (1, 3000, 1544, 32), (40, 300, 4736, 64)]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T,N,K,group", SIZES)
def test_against_the_definition(T, N, K, group, dtype):
    codes, scales, w = weights(N, K, group, seed=T + N, scale_dtype=BF16 if T % 2 else F32)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(K)).to(dtype)
    want = x.double() @ w.t()
    got = product(x, codes, scales, group, K)
    assert ((got - want).abs() <= allowed(x, scales, w, group, dtype, want)).all()


# Sizes at which other ways are taken: two and four tiles a wave, K in parts, x through LDS with two to four tiles of tokens, and the same without whole eights of K
WAYS = [(1, 16400, 64, 32), (4, 16390, 136, 64), (16, 7000, 256, 64), (3, 48, 9000, 128), (40, 100, 8200, 32), (17, 4000, 4304, 64), (17, 4000, 4300, 64), (33, 4001, 4304, 128),
        (64, 4000, 4304, 32), (40, 16390, 1040, 128), (60, 16400, 1040, 32), (1, 16400, 1040, 64), (5, 4000, 4304, 32), (80, 16400, 1040, 64)]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T,N,K,group", WAYS)
def test_every_way(T, N, K, group, dtype):
    codes, scales, w = weights(N, K, group, seed=T + N, scale_dtype=F32 if T % 2 else BF16)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(K)).to(dtype)
    want = x.double() @ w.t()
    got = product(x, codes, scales, group, K)
    assert ((got - want).abs() <= allowed(x, scales, w, group, dtype, want)).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_tensors_that_start_anywhere(dtype):
    """x, the result and the workspace at addresses that no 16-byte access takes."""
    from sprout_lm_amd import ops
    T, N, K, group = 20, 48, 9000, 128
    codes, scales, w = weights(N, K, group, seed=3)
    matrix = ops.q4_pack(codes.to(DEV), scales.to(DEV), group)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(3)).to(dtype)
    flat = torch.zeros(T * K + 1, dtype=dtype, device=DEV)
    flat[1:] = x.to(DEV).reshape(-1)
    room = torch.full((T * N + 2,), 7, dtype=dtype, device=DEV)
    need = ops.gemm_q4_workspace_floats(dtype, T, N, K)
    ops.gemm_q4(flat[1:].view(T, K), matrix, room[1:-1].view(T, N), workspace=lambda n: torch.zeros(n + 1, device=DEV)[1:])
    want = x.double() @ w.t()
    assert need > 0 and room[0] == 7 and room[-1] == 7
    assert ((room[1:-1].view(T, N).double().cpu() - want).abs() <= allowed(x, scales, w, group, dtype, want)).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("bias_dtype", [BF16, F32], ids=["bias16", "bias32"])
def test_bias_and_sums(dtype, bias_dtype):
    T, N, K, group = 9, 70, 256, 64
    codes, scales, w = weights(N, K, group, seed=2)
    g = torch.Generator().manual_seed(3)
    x, bias, before = torch.randn(T, K, generator=g).to(dtype), torch.randn(N, generator=g).to(bias_dtype), torch.randn(T, N, generator=g)
    want = x.double() @ w.t() + bias.double()
    got = product(x, codes, scales, group, K, bias=bias.to(DEV))
    tolerance = allowed(x, scales, w, group, dtype, want)
    assert ((got - want).abs() <= tolerance + 2.0 ** -24 * (want - bias.double()).abs()).all()
    got = product(x, codes, scales, group, K, bias=bias.to(DEV), accumulate=True, out=before.to(DEV))
    want = want + before.double()
    assert ((got - want).abs() <= allowed(x, scales, w, group, F32, want, more=2 * (want.abs() + before.double().abs()))).all()


def test_every_code_of_every_place():
    """Rows of one number: the product is that column's weight, its scale times a whole number in float32 (rounded once: 24 bits times 4)."""
    N, K, group = 40, 256, 32
    codes, scales, w = weights(N, K, group, seed=4, scale_dtype=F32)
    got = product(torch.eye(K, dtype=F32), codes, scales, group, K)
    assert torch.equal(got, w.t().float().double())
    assert torch.equal(product(torch.eye(K, dtype=BF16), codes, scales, group, K), w.t().float().bfloat16().double())


def test_numbers_that_are_not_finite():
    """They reach the columns of their own row; rows beside it and the row's other groups' scales do not matter."""
    T, N, K, group = 5, 33, 256, 64
    codes, scales, w = weights(N, K, group, seed=6)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(1)).to(BF16)
    clean = product(x, codes, scales, group, K)
    x[2, 70] = math.nan
    got = product(x, codes, scales, group, K)
    assert got[2].isnan().all() and torch.equal(got[[0, 1, 3, 4]], clean[[0, 1, 3, 4]])
    scales[7, 1] = math.nan
    got = product(x[:2], codes, scales, group, K)
    assert got[:, 7].isnan().all() and torch.equal(got[:, :7], clean[:2, :7]) and torch.equal(got[:, 8:], clean[:2, 8:])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("scale_dtype", [BF16, F32], ids=["scale16", "scale32"])
@pytest.mark.parametrize("N,K,group", [(3, 128, 128), (17, 100, 32), (5, 77, 64), (40, 512, 64), (1, 1, 32)])
def test_weights_are_rounded_as_said(N, K, group, dtype, scale_dtype):
    from sprout_lm_amd import ops
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(K)).to(dtype)
    w[0, :group] = 0
    w[N - 1, K - 1] = 40.0
    codes, scales = (t.cpu() for t in ops.q4_quantize(w.to(DEV), group, scale_dtype))
    groups = -(-K // group)
    padded = torch.zeros(N, groups * group)
    padded[:, :K] = w.float()
    padded = padded.view(N, groups, group).numpy()
    want_scales = torch.from_numpy(np.abs(padded).max(-1) / np.float32(7)).to(scale_dtype)
    assert torch.equal(scales, want_scales)
    s = want_scales.float().numpy()[..., None]
    with np.errstate(invalid="ignore"):
        q = np.where(s == 0, np.float32(0), np.rint(padded / np.where(s == 0, np.float32(1), s)))
    want = torch.from_numpy((np.clip(q, -8, 7) + 8).astype(np.uint8)).view(N, groups * group)[:, :K]
    got = torch.stack([codes & 15, codes >> 4], -1).view(N, -1)[:, :K]
    assert torch.equal(got, want)
    back = (got.double() - 8) * scales.double().repeat_interleave(group, 1)[:, :K]
    # half a step of the group's scale, and the largest numbers a little more where the scale was rounded down
    step = scales.double().repeat_interleave(group, 1)[:, :K]
    assert ((back - w.double()).abs() <= step / 2 * (1 + 2.0 ** -20) + 7 * step * 2.0 ** -8).all()


def test_groups_with_infinities_and_nan():
    from sprout_lm_amd import ops
    w = torch.ones(3, 64)
    w[0, 5], w[1, 40] = math.inf, math.nan
    codes, scales = (t.cpu() for t in ops.q4_quantize(w.to(DEV), 32, F32))
    assert scales[0, 0] == math.inf and scales[1, 1].isnan() and scales[0, 1] == scales[2, 0] == 1 / torch.tensor(7.0)
    assert codes.max() <= 0xff and (codes[2] == 0xff).all()      # seven steps above zero


def test_repeats_bit_for_bit_on_another_stream_and_from_a_graph():
    from sprout_lm_amd import ops
    N, K, group, T = 500, 1024, 64, 20
    codes, scales, w = weights(N, K, group, seed=1)
    matrix = ops.q4_pack(codes.to(DEV), scales.to(DEV), group)
    x = torch.randn(T, K, device=DEV, dtype=BF16)
    first, second = torch.empty(T, N, device=DEV, dtype=BF16), torch.empty(T, N, device=DEV, dtype=BF16)
    ops.gemm_q4(x, matrix, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.gemm_q4(x, matrix, second)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.gemm_q4(x, matrix, second)
    for i in range(3):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        ops.gemm_q4(x, matrix, first)
        assert torch.equal(first, second)


def test_a_matrix_beyond_32_bits():
    """More than 2^32 codes: the last rows are right."""
    from sprout_lm_amd import ops
    N, K, group = 2 ** 20 + 48, 4224, 128
    codes = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=DEV)
    scales = torch.full((N, K // group), 0.01, dtype=BF16, device=DEV)
    matrix = ops.q4_pack(codes, scales, group)
    x = torch.randn(2, K, device=DEV, dtype=F32)
    out = torch.empty(2, N, device=DEV)
    ops.gemm_q4(x, matrix, out)
    last = codes[-100:].cpu()
    w = (torch.stack([last & 15, last >> 4], -1).view(100, K).double() - 8) * float(scales[0, 0])
    want = x.double().cpu() @ w.t()
    assert ((out[:, -100:].double().cpu() - want).abs() <= allowed(x.cpu(), scales[-100:].cpu(), w, group, F32, want)).all()


def test_no_tokens():
    codes, scales, _ = weights(20, 64, 32, seed=1)
    assert product(torch.empty(0, 64, dtype=BF16), codes, scales, 32, 64).shape == (0, 20)


@pytest.mark.parametrize("what", ["group", "codes", "scales", "shape", "out", "sum", "bias", "cpu", "dtype", "cols"])
def test_refusals(what):
    from sprout_lm_amd import ops
    codes, scales, _ = weights(20, 64, 32, seed=1)
    codes, scales = codes.to(DEV), scales.to(DEV)
    matrix = ops.q4_pack(codes, scales, 32)
    x, out = torch.zeros(2, 64, dtype=BF16, device=DEV), torch.zeros(2, 20, dtype=BF16, device=DEV)
    ops.gemm_q4(x, matrix, out)
    calls = {"group": lambda: ops.q4_pack(codes, scales, 16), "codes": lambda: ops.q4_pack(codes.char(), scales, 32),
             "scales": lambda: ops.q4_pack(codes, scales[:, :1].contiguous(), 32), "shape": lambda: ops.gemm_q4(x[:, :32].contiguous(), matrix, out),
             "out": lambda: ops.gemm_q4(x, matrix, out.float()), "sum": lambda: ops.gemm_q4(x, matrix, out, accumulate=True),
             "bias": lambda: ops.gemm_q4(x, matrix, out, bias=torch.zeros(19, device=DEV)), "cpu": lambda: ops.gemm_q4(x.cpu(), matrix, out),
             "dtype": lambda: ops.gemm_q4(x.half(), matrix, out.half()), "cols": lambda: ops.q4_pack(codes, scales, 32, cols=62)}
    with pytest.raises(ops.KernelError):
        calls[what]()
