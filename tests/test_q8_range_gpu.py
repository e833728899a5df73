"""Norms to 8 bits of rows whose squares, or whose products with the weight, leave fp32's range."""
import pytest
import torch

from llm_pytorch_inference_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("width", [64, 65, 4096, 40000])
def test_squares_beyond_fp32_read_back_as_zeros_as_in_rmsnorm(width):
    x = torch.ones(3, width, device=DEV).bfloat16()
    x[1] = 1e20
    w = torch.full((width,), 0.5, dtype=torch.bfloat16, device=DEV)
    got = ops.rmsnorm_q8(x, w)
    assert got.scales[1] == 0 and (ops.dequantise_q8(got)[1] == 0).all() and (ops.rmsnorm(x, w)[1] == 0).all()
    one = ops.rmsnorm_q8(x[:1], w)
    for i in (0, 2):
        assert torch.equal(got.values[i], one.values[0]) and got.scales[i] == one.scales[0]
    added, total = ops.fused_add_rmsnorm_q8(x.clone(), torch.zeros_like(x), w)
    assert torch.equal(total, x) and torch.equal(added.scales, got.scales) and torch.equal(added.values, got.values)


@pytest.mark.parametrize("width", [64, 65, 4096, 40000])
def test_products_beyond_fp32_read_back_as_nan(width):
    x = torch.ones(3, width, device=DEV).bfloat16()
    w = torch.ones(width, dtype=torch.bfloat16, device=DEV)
    w[width // 2] = 1e30
    x[1, width // 2] = 1e10
    got = ops.rmsnorm_q8(x, w)
    assert got.scales[1].isnan() and ops.dequantise_q8(got)[1].isnan().all()
    assert got.scales[[0, 2]].isfinite().all()
