"""Adapter products and gradients where single bits, infinities and unused adapters decide."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def long_value(dtype):
    """Three values whose sum of products with `ones` needs 21 (bf16) or 24 bits, more than two values of the type hold:
    v . ones = 1 + a + b, v . less = 1 + a, exact in fp32 in any order."""
    small, least = (2.0 ** -9, 2.0 ** -20) if dtype == torch.bfloat16 else (2.0 ** -12, 2.0 ** -23)
    half = math.sqrt(least) if dtype == torch.bfloat16 else 2.0 ** -11
    return (1.0, small, half), (1.0, 1.0, least / half), least


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r", [2, 8, 16, 40, 256])
@pytest.mark.parametrize("T", [64, 65, 300, 2050])
def test_low_rank_sums_are_held_in_32_bits(gelim, cuda, T, r, dtype):
    """Y = 1024 (S_0 - S_last) with S_0 = 1 + a + b, S_last = 1 + a: exactly 1024 b, as every sum on the way is a
    multiple of b that 24 bits hold.  The same for dX, whose factors change places."""
    K = N = 72
    v, ones, least = long_value(dtype)
    at = [0, 17, 70]
    U, F, G = torch.zeros(T, K), torch.zeros(1, K, r), torch.zeros(1, r, N)
    U[:, at] = torch.tensor(v)
    F[0, at, 0] = torch.tensor(ones)
    F[0, at, r - 1] = torch.tensor(ones[:2] + (0.0,))
    G[0, 0], G[0, r - 1] = 1024.0, -1024.0
    U, F, G, W = (x.to(dtype).to(cuda) for x in (U, F, G, torch.zeros(K, N)))
    assert (gelim.ops.adapter_matmul(U, W, F, G) == 1024 * least).all()
    FT, GT = F.transpose(1, 2), G.transpose(1, 2)
    dX = gelim.ops.adapter_matmul_grad(U, torch.zeros_like(U), W, GT, FT, need=(True, False, False))[0]
    assert (dX == 1024 * least).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r", [1, 16, 40, 256])
@pytest.mark.parametrize("T", [2, 128, 129, 700])
def test_factor_gradients_of_32_bit_sums(gelim, cuda, T, r, dtype):
    """Two rows of opposite sign whose D (or S) differ by their last bit: the gradient is 1024 times that bit."""
    K = N = 72
    v, ones, least = long_value(dtype)
    at = [0, 17, 70]
    low, other, factor = torch.zeros(T, K), torch.zeros(T, N), torch.zeros(1, K, r)
    low[0, at], low[1, at] = torch.tensor(v), torch.tensor(v[:2] + (0.0,))
    other[0], other[1] = 1024.0, -1024.0
    factor[0, at] = torch.tensor(ones)[:, None]
    low, other, factor, W = (x.to(dtype).to(cuda) for x in (low, other, factor, torch.zeros(K, N)))
    zero = torch.zeros_like(factor)
    dB = gelim.ops.adapter_matmul_grad(other, low, W, factor, zero.transpose(1, 2))[2]
    assert (dB == 1024 * least).all()
    dA = gelim.ops.adapter_matmul_grad(low, other, W, zero, factor.transpose(1, 2))[1]
    assert (dA == 1024 * least).all()
