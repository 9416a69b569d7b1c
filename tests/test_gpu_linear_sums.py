"""How exact fp32 results are, at every K and in every form of the dense products.

The tensor cores cut off what a step of 16 of K adds, and what they cut off grows with the sum so far: the error, relative to the sum, grows with the
length of a chain of steps.  Chains end after 768 of K and meet by fp32 additions, so that the error at any K is that of a
chain: sums that only grow have equal relative errors in all chains, random ones errors that add up as the sums do, by squares.  A
quarter more covers the spread of 10^4 and more results.  The additions: K / 768 <= 66 roundings of 2^-25 of the sum on average that do not
lean, sqrt(66) 2^-25 = 2.4e-7.  (One chain of 16384 is off by 1.9e-5, sums that only grow by 8e-5.)"""
import pytest
import torch

from tcbnn_b200 import ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


def operands(M, N, K, dtype, growing, cuda):
    g = torch.Generator(device=cuda)
    g.manual_seed(M + K)
    x, w = torch.randn((M, K), device=cuda, generator=g), torch.randn((N, K), device=cuda, generator=g).mul_(K ** -0.5)
    if growing:
        x, w = x.abs(), w.abs()
    return x.to(dtype), w.to(dtype)


def most(dtype, growing, cuda):
    """From one chain of 768."""
    x, w = operands(200, 500, 768, dtype, growing, cuda)
    ops.set_linear_plan(64, 1)
    try:
        return 1.25 * off(ops.linear(x, w, out_dtype=FP32), x.double() @ w.double().t()) + 2.4e-7
    finally:
        ops.set_linear_plan()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("growing", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 300, 16384), (8, 500, 50000), (40, 400, 9000), (100, 1000, 16384), (300, 700, 4096), (333, 1000, 2049), (1000, 5000, 8192),
                                   (2100, 4000, 16384), (150, 300, 50000), (500, 20000, 3000), (130, 260, 769), (4000, 4000, 1500)])
def test_long_sums(cuda, dtype, growing, M, N, K):
    x, w = operands(M, N, K, dtype, growing, cuda)
    want = x.double() @ w.double().t()
    assert off(ops.linear(x, w, out_dtype=FP32), want) <= most(dtype, growing, cuda)


@pytest.mark.parametrize("cols,splits", [(16, 1), (48, 1), (112, 1), (128, 1), (208, 1), (256, 1), (16, 2), (48, 4), (64, 2), (64, 8), (80, 2), (96, 4), (112, 8), (128, 8), (32, -2), (96, -2), (224, -2), (256, -2)])
@pytest.mark.parametrize("M,N,K", [(1, 128, 4096), (300, 700, 1000), (530, 1300, 2000), (40, 129, 8200), (2000, 5000, 1600), (5000, 1500, 840)])
def test_chains_of_every_plan(cuda, cols, splits, M, N, K):
    """Whole numbers: exact, whichever chain a product falls into; bias, activation and residual once."""
    g = torch.Generator(device=cuda)
    g.manual_seed(cols + M)
    x = torch.randint(-4, 5, (M, K), generator=g, device=cuda).to(BF16)
    w = torch.randint(-4, 5, (N, K), generator=g, device=cuda).to(BF16)
    bias, res = torch.randint(-50, 51, (N,), generator=g, device=cuda).float(), torch.randint(-50, 51, (M, N), generator=g, device=cuda).float()
    want = (x.double() @ w.double().t() + bias.double()).clamp(min=0) + res.double()
    ops.set_linear_plan(cols, splits)
    try:
        for _ in range(2):
            assert torch.equal(ops.linear(x, w, bias, "relu", res, out_dtype=FP32).double(), want)
        assert ops.linear_status() == 0
    finally:
        ops.set_linear_plan()


@pytest.mark.parametrize("growing", [False, True])
@pytest.mark.parametrize("cols,splits", [(64, 1), (256, 1), (32, 2), (64, 4), (256, -2)])
def test_long_sums_of_every_form(cuda, growing, cols, splits):
    M, N, K = 300, 600, 16384
    x, w = operands(M, N, K, BF16, growing, cuda)
    want = x.double() @ w.double().t()
    ops.set_linear_plan(cols, splits)
    try:
        got = ops.linear(x, w, out_dtype=FP32)
    finally:
        ops.set_linear_plan()
    assert off(got, want) <= most(BF16, growing, cuda)
