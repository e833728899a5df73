"""Slot assignment and draft verification through ``torch.ops.mini_vllm_ops``."""
import pytest
import torch

from llm_pytorch_inference_b200 import ops, torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("head", [None, 1])
@pytest.mark.parametrize("held", [None, [2, 0, 1]])
@pytest.mark.parametrize("tokens", [0, 30])
def test_assign_slots(head, held, tokens):
    """What ``ops.assign_slots`` gives, in outputs that share no memory: the schema says of none that it aliases another."""
    ctx, new, free = i32([17, 0, 3]), i32([1, 20, 9]) * (tokens > 0), i32([9, 8, 7, 6, 5])
    res = []
    for fn in (torch.ops.mini_vllm_ops.assign_slots, ops.assign_slots):
        table, count = i32([[3, 4, 0], [0, 0, 0], [2, 0, 0]]), None if held is None else i32(held)
        out = fn(table, ctx, new, free, 16, tokens, None if head is None else i32([head]),
                 *([] if held is None else [count]))
        res.append([*out, table] + ([] if held is None else [count]))
    assert len(res[0]) == len(res[1]) and all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(*res))
    at = [t.untyped_storage().data_ptr() for t in res[0] if t.numel()]
    assert len(set(at)) == len(at)


@pytest.mark.parametrize("given", [True, False])
def test_verify_drafts(given):
    g = torch.Generator(device=DEV).manual_seed(3)
    p, q = (torch.rand(4, n, 50, generator=g, device=DEV).softmax(-1) for n in (4, 3))
    tokens = torch.randint(0, 50, (4, 3), generator=g, device=DEV)
    u, lens = torch.rand(4, 4, generator=g, device=DEV), i32([3, 0, 2, 1])
    got = torch.ops.mini_vllm_ops.verify_drafts(p, tokens, u, q if given else None, lens if given else None)
    want = ops.verify_drafts(p, tokens, u, q if given else None, lens if given else None)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
