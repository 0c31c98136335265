"""Products with 4-bit weights whose every sum is a whole number that float32 holds: the result is exact, whatever the order of its additions."""
import pytest
import torch

from tests.test_gpu_gemm_q4 import SIZES, WAYS, product, weights

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def parts(x):
    """x as three bfloat16 numbers, each of what the ones before have left."""
    out = []
    for _ in range(3):
        out.append(x.to(BF16).float())
        x = x - out[-1]
    return out


def whole_numbers(T, K, dtype, seed):
    """Rows of whole numbers: float32, two of 18 bits a row that two bfloat16 numbers do not hold; bfloat16, up to 1,000 of 8 bits."""
    g = torch.Generator().manual_seed(seed)
    x = torch.zeros(T, K)
    if dtype == F32:
        m = (2 * torch.randint(2 ** 16, 2 ** 17, (64 * T * 2 + 640,), generator=g) + 1).float()
        m = m[parts(m)[2] != 0][:T * 2].view(T, 2)
        assert (sum(parts(m)) == m).all()
    else:
        m = torch.randint(-255, 256, (T, min(K, 1000)), generator=g).float()
    for row, numbers in zip(x, m * torch.where(torch.rand(m.shape, generator=g) < 0.5, -1.0, 1.0)):
        row[torch.randperm(K, generator=g)[:len(numbers)]] = numbers
    x[0, K - 1] = m[0, 0]
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("T,N,K,group", SIZES + WAYS)
def test_sums_of_whole_numbers_are_exact(T, N, K, group, dtype):
    """In units of a 32nd (a scale is one or two): three float32 numbers below 2^18, or 1,001 bfloat16 ones below 2^8, times 8 (with what is added and taken
    off: 31 and 24) times 2 stay below 2^24, and so does every part and every sum of some of them."""
    codes, scales, _ = weights(N, K, group, seed=T + N)
    scales = (1 + torch.randint(0, 2, scales.shape, generator=torch.Generator().manual_seed(N))).div(32).to(BF16 if T % 2 else F32)
    x = whole_numbers(T, K, dtype, seed=K)
    codes_at = torch.stack([codes & 15, codes >> 4], -1).view(N, -1)[:, :K]
    want = x.double() @ ((codes_at.double() - 8) * scales.double().repeat_interleave(group, 1)[:, :K]).t()
    assert torch.equal(product(x, codes, scales, group, K), want.to(dtype).double())
