"""4-bit products of numbers at the ends of what they take."""
import math

import pytest
import torch

from tests.test_gpu_gemm_q4 import allowed, product, weights

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T", [3, 60])
def test_the_largest_numbers(T, group):
    """bfloat16: magnitudes of 2^122 in a group, of one sign, of both, in one number; float32: 2^125 in a group."""
    K, N = 384, 50
    codes, scales, w = weights(N, K, group, seed=5)
    signs = torch.where(torch.rand(T, K, generator=torch.Generator().manual_seed(6)) < 0.5, -1.0, 1.0)
    signs[0] = 1.0
    for dtype, most in ((BF16, 2.0 ** 122), (F32, 2.0 ** 125)):
        x = (signs * (most / group)).to(dtype)
        x[1] = 0
        x[1, 1::group] = most
        want = x.double() @ w.t()
        got = product(x, codes, scales, group, K)
        assert ((got - want).abs() <= allowed(x, scales, w, group, dtype, want)).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T", [4, 60])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, 3.3999e38])
def test_an_infinity_makes_its_tokens_row_nan(bad, T, dtype):
    """Also a float32 number that bfloat16 rounds to one.  Rows beside it do not change."""
    N, K, group = 33, 256, 64
    codes, scales, _ = weights(N, K, group, seed=6)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(1)).to(dtype)
    clean = product(x, codes, scales, group, K)
    x[2, 70] = bad
    got = product(x, codes, scales, group, K)
    keep = [t for t in range(T) if t != 2]
    assert got[2].isnan().all() and torch.equal(got[keep], clean[keep])
