"""Products with 4-bit weights where x just fits into a cluster's shared memory, and where it just does not."""
import pytest
import torch

import w4_reference as R
from llm_pytorch_inference_b200 import _native as N
from llm_pytorch_inference_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(rows, n, k, group, q8):
    g = torch.Generator(device=DEV).manual_seed(rows + n + k + group)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV, dtype=torch.uint8)
    scales = (0.02 * torch.exp(0.5 * torch.randn(n, groups, generator=g, device=DEV))).bfloat16()
    zeros = torch.randint(0, 16, (n, groups), generator=g, device=DEV, dtype=torch.uint8)
    w = ops.pack_w4(codes, scales, zeros, group)
    w64 = R.values(codes.cpu().long(), scales.cpu().double(), zeros.cpu().long(), group).to(DEV)
    x = torch.randn(rows, k, generator=g, device=DEV)
    x = x.bfloat16()
    x[:, ::97] = 300.0
    x64 = x.double()
    if q8:
        x = ops.quantise_q8(x)
        x64 = x.values.double() * x.scales.double()[:, None]
    got = ops.linear_w4(x, w)
    exact, size = x64 @ w64.T, x64.abs() @ w64.abs().T
    # a rounding to bf16, sums in 32 bits (and a scale's product): test_w4_precision_gpu derives the second term
    bound = 2.0 ** -8 * exact.abs() * 1.001 + 2.0 ** -23 * (k + 4 * groups + 200) * size
    assert ((got.double() - exact).abs() <= bound).all()
    assert N.device_status() == 0


@pytest.mark.parametrize("rows, n, k, group", [
    # 7 and 8 rows: the last that a cluster of 4 holds and the first that it does not, few weight rows and more
    *[(r, n, k, g) for r in (7, 8) for g, k in ((128, 15872), (128, 15904), (64, 15360), (64, 15392), (32, 13824), (32, 13856))
      for n in (40, 2080)],
    # and of a cluster of 8
    *[(8, 48, k, g) for g, k in ((128, 31744), (128, 31776), (64, 30688), (64, 30752), (32, 27648), (32, 27680))],
    # whatever k, up to 6 rows
    *[(r, 70, 32768, g) for r in (1, 2, 3, 4, 5, 6) for g in (32, 64, 128)], (5, 4000, 8224, 32), (8, 600, 5152, 32), (6, 1000, 8192, 32),
])
def test_bf16_rows(rows, n, k, group):
    check(rows, n, k, group, False)


@pytest.mark.parametrize("rows, n, k, group", [
    *[(r, 70, 32768, g) for r in (8, 9, 16, 17) for g in (32, 64, 128)], (16, 3000, 15392, 32), (12, 3000, 20512, 64), (9, 3000, 23584, 128),
])
def test_8_bit_rows(rows, n, k, group):
    check(rows, n, k, group, True)
