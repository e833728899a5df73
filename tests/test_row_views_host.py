"""Which tensors are taken for rows a fixed distance apart, and which are copied or refused, on the CPU."""
import itertools

import pytest
import torch

from llm_pytorch_inference_b200 import ops


def reached(t: torch.Tensor, row: int) -> list[int]:
    """Elements of the storage at which rows `row` apart begin."""
    return [t.storage_offset() + i * row for i in range(t.numel() // t.shape[-1])]


def begins(t: torch.Tensor) -> list[int]:
    """Elements of the storage at which the rows of t begin, in their order."""
    return [t.storage_offset() + sum(i * s for i, s in zip(at, t.stride())) for at in
            itertools.product(*(range(n) for n in t.shape[:-1]))]


def expanded_views():
    a = torch.zeros(4, 8)
    yield "inner of three", a[:, None].expand(4, 5, 8)
    yield "outer of three", a[None].expand(3, 4, 8)
    yield "both of three", a[0].expand(4, 5, 8)
    yield "first of four", a.view(2, 2, 8)[None].expand(3, 2, 2, 8)
    yield "second of four", a.view(2, 1, 2, 8).expand(2, 3, 2, 8)
    yield "third of four", a.view(2, 2, 1, 8).expand(2, 2, 3, 8)
    yield "first and third of four", a.view(1, 4, 1, 8).expand(2, 4, 3, 8)
    yield "second and third of four", a[:, None, None].expand(4, 2, 3, 8)
    yield "all of four", a[0].expand(2, 3, 4, 8)
    yield "a dimension of one beside it", a[:, None, None].expand(4, 1, 3, 8)
    yield "of two", a[0].expand(6, 8)
    yield "of rows further apart", torch.zeros(4, 20)[:, None, 4:12].expand(4, 5, 8)


EXPANDED = list(expanded_views())


@pytest.mark.parametrize("name, t", EXPANDED, ids=[name for name, _ in EXPANDED])
def test_broadcast_rows_are_no_view(name, t):
    assert ops._row_view(t) is None
    copy, row = ops._rows_of(t)
    assert copy.is_contiguous() and copy.shape == t.shape and row == 8


def test_broadcast_elements_are_no_view():
    assert ops._row_view(torch.zeros(4, 1).expand(4, 8)) is None
    assert ops._row_view(torch.zeros(2, 3, 1).expand(2, 3, 8)) is None


VIEWS = [
    torch.zeros(4, 8), torch.zeros(4, 20)[:, 3:11], torch.zeros(9, 8)[::2], torch.zeros(1, 20)[:, :8], torch.zeros(6, 20)[:, :8].view(2, 3, 8),
    torch.zeros(2, 3, 20)[..., 5:13], torch.zeros(2, 1, 3, 20)[..., :8], torch.zeros(4, 3, 8)[:, 1:2], torch.zeros(4, 3, 8)[:, 1], torch.zeros(8),
    torch.zeros(20)[4:12], torch.zeros(5, 1).expand(5, 1), torch.zeros(8)[None, None].expand(1, 1, 8),
]


@pytest.mark.parametrize("t", VIEWS, ids=[f"{tuple(t.shape)} {t.stride()}" for t in VIEWS])
def test_rows_a_fixed_distance_apart_are_taken_where_they_are(t):
    view = ops._row_view(t)
    assert view is not None and view[0].data_ptr() == t.data_ptr()
    assert reached(t, view[1]) == begins(t)


@pytest.mark.parametrize("shape", [(2, 3, 8), (2, 2, 3, 8)])
def test_no_view_reaches_other_elements_than_its_rows(shape):
    """Every order of the dimensions, a slice of the first, a dimension more anywhere, broadcast or not."""
    for order, cut, at, wide in itertools.product(itertools.permutations(range(len(shape))), (slice(None), slice(0, 1), slice(1, None)),
                                                  range(len(shape)), (1, 4)):
        t = torch.zeros(shape).permute(order)[cut].unsqueeze(at)
        for first in (1, 5):
            sizes = [first if t.shape[0] == 1 else t.shape[0], *t.shape[1:]]
            sizes[at] = wide if at else sizes[at]
            view = ops._row_view(t.expand(sizes))
            if view is not None:
                assert reached(view[0], view[1]) == begins(view[0]), (sizes, view[0].stride())
                assert sizes[-1] == 1 or view[0].stride(-1) == 1
