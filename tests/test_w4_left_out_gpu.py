"""Elements far below their group's largest, in products of few rows, for every way in which warps and blocks share the work."""
import pytest
import torch

import w4_reference as R
from llm_pytorch_inference_b200 import _native as N
from llm_pytorch_inference_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def made(seed, n, k, group, at):
    """A weight that is zero in the columns `at`, and what it stands for in 64 bits."""
    g = gen(seed)
    groups = -(-k // group)
    zeros = torch.randint(0, 16, (n, groups), generator=g, device=DEV, dtype=torch.uint8)
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV, dtype=torch.uint8)
    codes[:, at] = zeros[:, torch.div(at, group, rounding_mode="floor")]
    scales = (0.02 * torch.exp(0.5 * torch.randn(n, groups, generator=g, device=DEV))).bfloat16()
    return ops.pack_w4(codes, scales, zeros, group), (codes, scales, zeros)


def rows_of(seed, rows, k, at, large):
    x = torch.randn(rows, k, generator=gen(seed), device=DEV).bfloat16()
    x[:, at] = large
    return x


def check(got, x, parts, group):
    codes, scales, zeros = parts
    of = torch.div(torch.arange(codes.shape[1], device=DEV), group, rounding_mode="floor")
    k = codes.shape[1]
    for lo in range(0, codes.shape[0], 16384):
        part = slice(lo, lo + 16384)
        w = scales[part][:, of].double() * (codes[part].double() - zeros[part][:, of].double())
        exact, size = x.double() @ w.T, x.double().abs() @ w.abs().T
        # test_w4_precision_gpu derives it: a rounding to bf16, and sums in 32 bits of what meets weights that are not zero
        bound = 2.0 ** -8 * exact.abs() * 1.001 + 2.0 ** -23 * (k + 4 * -(-k // group) + 200) * size
        assert ((got[:, part].double() - exact).abs() <= bound).all()
    assert N.device_status() == 0


SHAPES = [  # pairs of tiles a block: one to many, in one round of a cluster or several; warps alone or sharing a pair
    (40, 32, 32), (40, 128, 128), (9000, 128, 64), (100000, 256, 128), (4096, 4096, 128), (50000, 4096, 128), (2500, 2176, 32),
    (100, 16384, 64), (30000, 2048, 128),
]


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("n, k, group", SHAPES)
def test_far_elements_in_some_groups_or_in_all(n, k, group, rows):
    one = torch.tensor([k // 2 + 5], device=DEV)
    many = torch.arange(7, k, 100, device=DEV)
    for at, large in ((one, 3e5), (many, 1e8)):
        w, parts = made(n + k, n, k, group, at)
        x = rows_of(rows, rows, k, at, large)
        check(ops.linear_w4(x, w), x, parts, group)
        x[::2, at] = 0  # other rows leave nothing
        check(ops.linear_w4(x, w), x, parts, group)


@pytest.mark.parametrize("rows", [1, 5, 8])
def test_replayed_with_rows_that_leave_some_and_none(rows):
    n, k, group = 3000, 2048, 128
    at = torch.tensor([5, 700], device=DEV)
    w, parts = made(1, n, k, group, at)
    x = rows_of(2, rows, k, at, 1.0)
    ops.linear_w4(x, w)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.linear_w4(x, w))
        graphs.append(graph)
    for seed, large in ((3, 1e6), (4, 0.5), (5, 1e20)):
        x.copy_(rows_of(seed, rows, k, at, large))
        for graph, out in zip(graphs, outs):
            graph.replay()
            check(out, x, parts, group)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], ops.linear_w4(x, w))


def test_on_two_streams_and_with_launches_that_follow_early():
    n, k, group = 4096, 1024, 64
    at = torch.tensor([9], device=DEV)
    w, _ = made(6, n, k, group, at)
    xs = [rows_of(7 + i, r, k, at, 1e6) for i, r in enumerate((1, 4, 6, 8))]
    want = [ops.linear_w4(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    before = N.set_pdl(True)
    try:
        for _ in range(5):
            got = []
            for stream in streams:
                with torch.cuda.stream(stream):
                    for x, y in zip(xs, want):
                        z = x.clone()
                        got.append((ops.linear_w4(z, w), y))
                        z.zero_()  # behind the product, which reads its rows to the end
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in got)
    finally:
        N.set_pdl(before)
    assert N.device_status() == 0
