"""How exact products of bf16 rows with 4-bit weights are where a group of x spans many powers of two, in 64 bits.

The bound: the result is rounded to bf16 once, and sums are held in 32 bits.  In the kernel of few rows a group's sum
of one digit of x is a whole number, exact; what an element's digits stand for is at most 3.03 times the element in sum (at
worst the first is twice as much, the second takes half of that back); each digit's sums are scaled and added in 32 bits, a
rounding a group, and then 16 warps' four sums and 8 blocks' are, 72 roundings: 3.03 (groups + 72) 2^-24 of the sum of |x| |w|.
What the digits leave is added one by one: k 2^-24.  With many rows a group's products are added in the tensor core, at most
a unit of 2^-23 each, and the groups after them.  So both are within 2^-23 (k + 4 groups + 200) of the sum of |x| |w|: elements
that meet a zero weight count for nothing.
"""
import math

import pytest
import torch

import w4_reference as R
from llm_pytorch_inference_b200 import _native as N
from llm_pytorch_inference_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def packed(seed, n, k, group, scale=0.02):
    g = gen(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV, dtype=torch.uint8)
    scales = (scale * torch.exp(0.5 * torch.randn(n, groups, generator=g, device=DEV))).bfloat16()
    zeros = torch.randint(0, 16, (n, groups), generator=g, device=DEV, dtype=torch.uint8)
    return codes, scales, zeros


def made(codes, scales, zeros, group):
    w = ops.pack_w4(codes, scales, zeros, group)
    return w, R.values(codes.cpu().long(), scales.cpu().double(), zeros.cpu().long(), group).to(DEV)


def check(got, x, w, group):
    x = x.double()
    exact, size = x @ w.T, x.abs() @ w.abs().T
    k = x.shape[1]
    bound = 2.0 ** -8 * exact.abs() * 1.001 + 2.0 ** -23 * (k + 4 * -(-k // group) + 200) * size
    off = (got.double() - exact).abs()
    assert (off <= bound).all(), ((off / bound.clamp_min(1e-300)).max().item(), (off - bound).argmax().item())
    assert N.device_status() == 0


@pytest.mark.parametrize("large", [1e3, 1e4, 1e5, 1e6, 1e12, 1e30])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9])
def test_large_elements_that_meet_a_zero_weight(rows, group, large):
    """One column in 32 holds elements far above the others, and the weights there are zero."""
    n, k = 40, 384
    codes, scales, zeros = packed(1, n, k, group)
    at = torch.arange(5, k, 32, device=DEV)
    codes[:, at] = zeros[:, torch.div(at, group, rounding_mode="floor")]
    w, exact = made(codes, scales, zeros, group)
    x = (0.5 * torch.randn(rows, k, generator=gen(2), device=DEV)).bfloat16()
    x[:, at] = (large * (1 + torch.rand(rows, len(at), generator=gen(3), device=DEV))).bfloat16()
    check(ops.linear_w4(x, w), x, exact, group)
    some = x.clone()  # in some rows and groups only
    some[::2, at[::3]] = 0
    check(ops.linear_w4(some, w), some, exact, group)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 6, 8, 16])
@pytest.mark.parametrize("n, k", [(1, 32), (16, 128), (33, 160), (300, 1056), (2100, 512)])
def test_elements_of_every_size(n, k, rows, group):
    """Sizes spread over 2^-60 .. 2^0 within a group; half the weights are zero, with the largest elements among them."""
    codes, scales, zeros = packed(4, n, k, group)
    x = torch.exp2(-60 * torch.rand(rows, k, generator=gen(5), device=DEV)) * (1 + torch.rand(rows, k, generator=gen(6), device=DEV))
    x = (x * torch.where(torch.rand(rows, k, generator=gen(7), device=DEV) > 0.5, 1.0, -1.0)).bfloat16()
    none = torch.rand(n, k, generator=gen(8), device=DEV) > 0.5
    none |= (x.float().abs() > 2.0 ** -25).any(0)[None] & (torch.arange(n, device=DEV) % 2 == 0)[:, None]
    of = torch.div(torch.arange(k, device=DEV), group, rounding_mode="floor")
    codes = torch.where(none, zeros[:, of], codes)
    w, exact = made(codes, scales, zeros, group)
    check(ops.linear_w4(x, w), x, exact, group)


@pytest.mark.parametrize("rows, n, k, group", [
    (1, 4096, 4096, 128), (2, 6144, 4096, 64), (4, 6144, 4096, 128), (5, 512, 12288, 128), (7, 1024, 8192, 128), (8, 24576, 1024, 128),
    (3, 100, 16384, 64), (2, 16, 32768, 128), (8, 33, 20480, 32), (3, 40, 32768, 32), (1, 40000, 256, 128), (5, 48, 2080, 32),
])
def test_rows_as_they_are(rows, n, k, group):
    """Ordinary rows with a few channels of a hundred times the others', and one element of a thousand."""
    codes, scales, zeros = packed(9, n, k, group)
    w, exact = made(codes, scales, zeros, group)
    x = torch.randn(rows, k, generator=gen(10), device=DEV) * (1 + 100 * (torch.rand(k, generator=gen(11), device=DEV) > 0.99))
    x[:, k // 3] = 1000.0
    x = x.bfloat16()
    check(ops.linear_w4(x, w), x, exact, group)


@pytest.mark.parametrize("rows", [1, 3, 8])
def test_rows_of_tiny_and_of_huge_elements(rows):
    """Elements down to 2^-126 by weights whose products are ordinary numbers, and up to 2^127 the same."""
    n, k, group = 48, 256, 64
    spread = torch.randn(rows, k, generator=gen(12), device=DEV)
    for f, scale in ((2.0 ** -104, 2.0 ** 90), (2.0 ** -112, 2.0 ** 100), (2.0 ** -120, 2.0 ** 110), (2.0 ** 124, 2.0 ** -20)):
        codes, scales, zeros = packed(13, n, k, group, scale)
        w, exact = made(codes, scales, zeros, group)
        x = (spread.double() * f).float().bfloat16()
        if f < 1:  # no subnormal numbers here
            x = torch.where(x.abs() < 2.0 ** -126, 0, x)
        check(ops.linear_w4(x, w), x, exact, group)


@pytest.mark.parametrize("rows", [1, 3, 8])
def test_rows_of_subnormal_elements(rows):
    n, k, group = 48, 256, 128
    codes, scales, zeros = packed(14, n, k, group, 2.0 ** 115)
    w, exact = made(codes, scales, zeros, group)
    x = (torch.randint(-127, 128, (rows, k), generator=gen(15), device=DEV).double() * 2.0 ** -133).float().bfloat16()
    check(ops.linear_w4(x, w), x, exact, group)


def test_many_rows_of_large_elements():
    """Large elements of both signs (test_w4_range_gpu goes to the ends of the range)."""
    n, k, group = 40, 256, 128
    codes, scales, zeros = packed(16, n, k, group)
    w, exact = made(codes, scales, zeros, group)
    for rows in (9, 40, 130):
        x = (1e35 * (2 * torch.rand(rows, k, generator=gen(17), device=DEV) - 1)).bfloat16()
        check(ops.linear_w4(x, w), x, exact, group)


@pytest.mark.parametrize("rows", [1, 3, 8])
def test_a_row_gives_the_same_alone_and_with_others(rows):
    """Elements of all sizes: a row's result in the kernel of few rows does not depend on the rows beside it."""
    n, k, group = 200, 768, 128
    w, _ = made(*packed(18, n, k, group), group)
    x = (torch.randn(rows, k, generator=gen(19), device=DEV) * torch.exp2(-40 * torch.rand(rows, k, generator=gen(20), device=DEV))).bfloat16()
    got = ops.linear_w4(x, w)
    order = torch.randperm(rows, generator=gen(21), device=DEV)
    assert torch.equal(ops.linear_w4(x[order].contiguous(), w), got[order])
    assert torch.equal(ops.linear_w4(x, w), got)
    bad = x.clone()
    bad[0, 3] = math.nan
    other = ops.linear_w4(bad, w)
    assert other[0].isnan().all() and torch.equal(other[1:], got[1:])
