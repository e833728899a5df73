"""Quantising groups whose range is a few units of bf16's smallest number: scales that are one or two units."""
import pytest
import torch

import w4_reference as R
from llm_pytorch_inference_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = 2.0 ** -133


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("sign", [-1, 1])
def test_groups_of_one_sign_and_a_few_units(sign, group):
    """Row i: 0 .. i units of one sign.  Where the scale is rounded down, -lo / scale passes 15.5."""
    n, k = 64, 256
    g = torch.Generator(device=DEV).manual_seed(1)
    units = (torch.rand(n, k, generator=g, device=DEV) * torch.arange(1, n + 1, device=DEV)[:, None]).floor()
    units[:, ::group] = torch.arange(n, device=DEV)[:, None].float()
    w = (sign * units.double() * UNIT).float().bfloat16()
    got = ops.quantise_w4(w, group)
    codes, scales, zeros = R.quantise(w, group)
    a, b, c = R.unpack(got.records, n, k, group)
    assert torch.equal(b, scales) and torch.equal(c, zeros) and torch.equal(a, codes)
    exact = R.values(codes, scales, zeros, group)
    assert torch.equal(ops.dequantise_w4(got, torch.float32).cpu().double(), exact)
    again = ops.pack_w4(codes.to(DEV, torch.uint8), scales.to(DEV, torch.bfloat16), zeros.to(DEV, torch.uint8), group)
    assert torch.equal(again.records, got.records)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_groups_of_both_signs_and_a_few_units(group):
    n, k = 64, 256
    g = torch.Generator(device=DEV).manual_seed(2)
    low, high = torch.arange(n, device=DEV), torch.randint(0, 20, (n,), generator=g, device=DEV)
    units = (torch.rand(n, k, generator=g, device=DEV) * (low + high + 1)[:, None]).floor() - low[:, None]
    units[:, ::group] = -low[:, None].float()
    w = (units.double() * UNIT).float().bfloat16()
    got = ops.quantise_w4(w, group)
    codes, scales, zeros = R.quantise(w, group)
    a, b, c = R.unpack(got.records, n, k, group)
    assert torch.equal(b, scales) and torch.equal(c, zeros) and torch.equal(a, codes)


@pytest.mark.parametrize("rows", [2, 12])
def test_products_of_such_weights(rows):
    """Few rows and many read the same weights from them."""
    n, k = 64, 256
    units = -torch.arange(n, device=DEV)[:, None].expand(n, k).clone()
    units[:, 1::2] = torch.div(units[:, 1::2], 2, rounding_mode="trunc")
    w = ops.quantise_w4((units.double() * UNIT).float().bfloat16(), 128)
    g = torch.Generator(device=DEV).manual_seed(3)
    x = (2.0 ** 120 * torch.randint(0, 8, (rows, k), generator=g, device=DEV).float()).bfloat16()
    exact = x.double() @ ops.dequantise_w4(w, torch.float32).double().T
    # all products have one sign: sums in 32 bits are within k + groups units of 2^-23 of the result, rounded once to bf16
    assert ((ops.linear_w4(x, w).double() - exact).abs() <= (2.0 ** -8 + (k + 4 * 2 + 200) * 2.0 ** -23) * 1.001 * exact.abs()).all()
