"""Refusals of 8-bit rows that are none, on the CPU."""
import pytest
import torch

from llm_pytorch_inference_b200 import ops

CODES, SCALES = torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2)


@pytest.mark.parametrize("rows", [
    None, 3, (), (CODES,), (CODES, SCALES, SCALES), (CODES, None), (None, SCALES), ops.Q8Rows(CODES, 1.0), "ab", CODES, CODES[0], CODES[:1],
    torch.zeros(3, 2, 8, dtype=torch.int8), torch.zeros(()),
], ids=lambda rows: type(rows).__name__)
def test_what_is_no_pair_of_tensors_is_refused(rows):
    with pytest.raises(RuntimeError):
        ops.dequantise_q8(rows)


@pytest.mark.parametrize("x", [ops.Q8Rows(None, None), ops.Q8Rows(CODES, None), (CODES, SCALES), None])
def test_linear_refuses_them(x):
    weight = ops.W4Weight(torch.zeros(1, 1088, dtype=torch.uint8), 16, 128, 128)
    with pytest.raises(RuntimeError):
        ops.linear_w4(x, weight)
