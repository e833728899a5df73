"""4-bit weights and 8-bit rows on the CPU: refusals before any kernel, and the layout of the records."""
import pytest
import torch

from llm_pytorch_inference_b200 import _native as N
from llm_pytorch_inference_b200 import ops
import w4_reference as R


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from llm_pytorch_inference_b200.build import build
        build()
    return N.load()


def bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


W = ops.W4Weight(torch.zeros(1, 1088, dtype=torch.uint8), 16, 128, 128)


@pytest.mark.parametrize("call", [
    lambda: ops.quantise_q8(bf16(2, 8)),
    lambda: ops.dequantise_q8(ops.Q8Rows(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2))),
    lambda: ops.rmsnorm_q8(bf16(2, 8), bf16(8)),
    lambda: ops.fused_add_rmsnorm_q8(bf16(2, 8), bf16(2, 8), bf16(8)),
    lambda: ops.swiglu_q8(bf16(2, 8), bf16(2, 8)),
    lambda: ops.geglu_q8(bf16(2, 8), bf16(2, 8)),
    lambda: ops.quantise_w4(bf16(16, 128)),
    lambda: ops.pack_w4(torch.zeros(16, 128, dtype=torch.uint8), bf16(16, 1)),
    lambda: ops.dequantise_w4(W),
    lambda: ops.linear_w4(bf16(2, 128), W),
    lambda: ops.quantise_q8(None),
    lambda: ops.linear_w4(bf16(2, 128), None),
    lambda: ops.linear_w4(bf16(2, 128), (None, 16, 128, 128)),
])
def test_cpu_tensors_and_none_are_refused(call):
    with pytest.raises(RuntimeError):
        call()


@pytest.mark.parametrize("args, words", [
    ((1, 8, 1, 8, None, 1, 1, 8, 96, 48), b"groups of 48"),
    ((1, 8, 1, 8, None, 1, 1, 8, 40, 64), b"40 columns"),
    ((1, 8, 1, 8, None, 1, 1, 8, 32800, 64), b"32800 columns"),
    ((1, 8, 1, 8, None, 1, -1, 8, 64, 64), b"-1 rows"),
    ((1, 8, 1, 8, None, 1, 1 << 19, 8, 64, 64), b"524288 rows"),
    ((1, 8, 1, 8, None, 1, 1, 1 << 25, 64, 64), b"33554432 weight rows"),
    ((None, 8, 16, 64, None, 16, 1, 8, 64, 64), b"null pointer"),
    ((16, 8, 8, 64, None, 16, 1, 8, 64, 64), b"16 bytes"),
    ((16, 8, 16, 68, None, 16, 2, 8, 64, 64), b"16 bytes"),
    ((16, 4, 16, 64, None, 16, 2, 8, 64, 64), b"16 bytes"),
    ((16, 8, 16, 32, None, 16, 2, 8, 64, 64), b"16 bytes"),
])
def test_linear_refusals_of_the_c_abi(lib, args, words):
    assert lib.mvb_linear_w4(*args, None) == 1
    assert words in lib.mvb_last_error()


def test_other_refusals_of_the_c_abi(lib):
    for rc, words in [
        (lambda: lib.mvb_quantise_w4(16, 16, 64, 8, 33, 32, None), b"33 columns"),
        (lambda: lib.mvb_quantise_w4(16, 8, 64, 8, 64, 32, None), b"16 bytes"),
        (lambda: lib.mvb_quantise_w4(16, 16, 60, 8, 64, 32, None), b"16 bytes"),
        (lambda: lib.mvb_pack_w4(16, None, 16, None, 8, 64, 32, None), b"null pointer"),
        (lambda: lib.mvb_dequantise_w4(16, 16, 8, 64, 32, N.F16, None), b"dtype code 1"),
        (lambda: lib.mvb_quantise_q8(1, 1, 1, 8, 2, 0, N.BF16, None), b"rows of 0"),
        (lambda: lib.mvb_quantise_q8(1, 1, 1, 4, 2, 8, N.BF16, None), b"rows 4 apart"),
        (lambda: lib.mvb_rmsnorm_q8(1, 1, 1, 8, None, 2, 8, 1e-6, 0, N.BF16, None), b"null pointer"),
        (lambda: lib.mvb_gated_q8(1, 1, 1, 8, 1, 8, 2, 8, 7, N.BF16, None), b"activation 7"),
        (lambda: lib.mvb_fused_add_rmsnorm_q8(1, 1, 1, 8, 1, 8, 1, 8, 1, 2, 8, 1e-6, 0, N.I32, None), b"dtype code 3"),
        (lambda: lib.mvb_dequantise_q8(1, 1, 8, 1, -2, 8, N.BF16, None), b"-2 rows"),
    ]:
        assert rc() == 1
        assert words in lib.mvb_last_error(), lib.mvb_last_error()


def test_nothing_to_do_is_no_error(lib):
    assert lib.mvb_linear_w4(None, 8, None, 64, None, None, 0, 8, 64, 64, None) == 0
    assert lib.mvb_linear_w4(None, 8, None, 64, None, None, 3, 0, 64, 64, None) == 0
    assert lib.mvb_quantise_w4(None, None, 64, 0, 64, 64, None) == 0
    assert lib.mvb_quantise_q8(None, None, None, 8, 0, 8, N.BF16, None) == 0


@pytest.mark.parametrize("n, k, group", [(1, 32, 32), (17, 96, 64), (130, 160, 128), (300, 1056, 32)])
def test_size_of_the_records(lib, n, k, group):
    assert lib.mvb_w4_bytes(n, k, group) == -(-n // 16) * -(-k // 128) * R.record_bytes(group)


def test_w4_bytes_refuses(lib):
    assert lib.mvb_w4_bytes(8, 64, 16) == -1 and lib.mvb_w4_bytes(8, 31, 64) == -1


@pytest.mark.parametrize("n, k, group", [(16, 128, 128), (40, 256, 64), (150, 160, 32)])
def test_every_code_and_word_has_a_place_of_its_own(n, k, group):
    size = -(-n // 16) * -(-k // 128) * R.record_bytes(group)
    codes, words = set(), {}
    for i in range(n):
        for j in range(k):
            byte, nibble, word = R.place(i, j, n, k, group)
            assert 0 <= byte < size and word + 4 <= size
            codes.add((byte, nibble))
            words.setdefault(word, (i, j // group))
            assert words[word] == (i, j // group)
    assert len(codes) == n * k and not {b for b, _ in codes} & {w + i for w in words for i in range(4)}
