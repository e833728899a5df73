"""Products of bf16 rows with 4-bit weights at both ends of bf16's range, few rows and many, in 64 bits.

The bound is that of test_w4_precision_gpu: a rounding to bf16 and 2^-23 (k + 4 groups + 200) of the sum of |x| |w|.  The
inputs keep results and their sums inside fp32's normal numbers, so that nothing but this comes in.
"""
import math

import pytest
import torch

import w4_reference as R
from llm_pytorch_inference_b200 import _native as N
from llm_pytorch_inference_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROWS = [1, 4, 8, 9, 40, 64, 130]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def made(seed, n, k, group, scale):
    g = gen(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV, dtype=torch.uint8)
    scales = (scale * torch.exp(0.5 * torch.randn(n, groups, generator=g, device=DEV))).bfloat16()
    zeros = torch.randint(0, 16, (n, groups), generator=g, device=DEV, dtype=torch.uint8)
    w = ops.pack_w4(codes, scales, zeros, group)
    return w, R.values(codes.cpu().long(), scales.cpu().double(), zeros.cpu().long(), group).to(DEV)


def check(got, x, w, group):
    x = x.double()
    exact, size = x @ w.T, x.abs() @ w.abs().T
    k = x.shape[1]
    bound = 2.0 ** -8 * exact.abs() * 1.001 + 2.0 ** -23 * (k + 4 * -(-k // group) + 200) * size
    assert got.isfinite().all()
    assert ((got.double() - exact).abs() <= bound).all()
    assert N.device_status() == 0


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", ROWS)
def test_rows_up_to_the_largest_number(rows, group):
    """15 times the sum of a group's elements is far beyond fp32's range, the results are not."""
    n, k = 150, 512
    w, exact = made(1, n, k, group, 2.0 ** -20)
    x = torch.rand(rows, k, generator=gen(2), device=DEV) * 3.3e38
    for sign in (torch.ones(k, device=DEV), torch.where(torch.rand(k, generator=gen(3), device=DEV) > 0.5, 1.0, -1.0)):
        y = (x * sign).bfloat16()
        assert y.isfinite().all()
        check(ops.linear_w4(y, w), y, exact, group)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("power", [-100, -110, -120, -126])
def test_rows_down_to_the_smallest_normal_number(rows, group, power):
    n, k = 150, 512
    w, exact = made(4, n, k, group, 2.0 ** 100)
    x = (torch.randn(rows, k, generator=gen(5), device=DEV).double() * 2.0 ** power).float().bfloat16()
    x = torch.where(x.abs() < 2.0 ** -126, 0, x)
    check(ops.linear_w4(x, w), x, exact, group)


@pytest.mark.parametrize("rows", ROWS)
def test_rows_of_subnormal_numbers(rows):
    n, k, group = 48, 256, 128
    w, exact = made(6, n, k, group, 2.0 ** 115)
    x = (torch.randint(-127, 128, (rows, k), generator=gen(7), device=DEV).double() * 2.0 ** -133).float().bfloat16()
    check(ops.linear_w4(x, w), x, exact, group)


@pytest.mark.parametrize("rows", [9, 70])
def test_infinities_and_nan_among_many_rows(rows):
    """As before: such a row has no finite result where its weights are not zero, and leaves the others alone."""
    n, k, group = 64, 256, 64
    w, _ = made(8, n, k, group, 0.02)
    x = torch.randn(rows, k, generator=gen(9), device=DEV).bfloat16()
    plain = ops.linear_w4(x, w)
    x[1, 7], x[2, 9], x[3, 11] = math.nan, math.inf, -math.inf
    got = ops.linear_w4(x, w)
    keep = [i for i in range(rows) if i not in (1, 2, 3)]
    assert got[1].isnan().all() and not got[2:4].isfinite().any() and torch.equal(got[keep], plain[keep])
