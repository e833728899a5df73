"""4-bit weights (quantise, pack, read back) and the products with them against their formulas in 64 bits."""
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


def weight_of(seed, n, k):
    g = gen(seed)
    return (0.02 * torch.randn(n, k, generator=g, device=DEV) * torch.exp(torch.randn(n, 1, generator=g, device=DEV))).bfloat16()


def packed(seed, n, k, group):
    """A weight of random codes, scales and zeros, and what it stands for in 64 bits."""
    g = gen(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV, dtype=torch.uint8)
    scales = (0.02 * torch.exp(torch.randn(n, groups, generator=g, device=DEV))).bfloat16()
    zeros = torch.randint(0, 16, (n, groups), generator=g, device=DEV, dtype=torch.uint8)
    w = ops.pack_w4(codes, scales, zeros, group)
    return w, R.values(codes.cpu().long(), scales.cpu().double(), zeros.cpu().long(), group).to(DEV)


def rows_of(seed, rows, k, q8):
    """Rows as linear_w4 takes them, and in 64 bits."""
    g = gen(seed)
    x = torch.randn(rows, k, generator=g, device=DEV) * (1 + 20 * (torch.rand(k, generator=g, device=DEV) > 0.98))
    x = (x * torch.exp(torch.randn(rows, 1, generator=g, device=DEV))).bfloat16()
    if not q8:
        return x, x.double()
    r = ops.quantise_q8(x)
    return r, r.values.double() * r.scales.double()[:, None]


def check(got, x, w, group):
    exact = x @ w.T
    assert got.dtype is torch.bfloat16 and got.shape == exact.shape
    off = (got.double() - exact).abs() - R.linear_bound(x, w, group, exact)
    assert (off <= 0).all(), (off.max().item(), off.argmax().item())


SHAPES = [(1, 32), (15, 96), (16, 128), (33, 160), (128, 128), (130, 256), (300, 1056)]


# ------------------------------------------------------------------------------------- weights
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n, k", SHAPES + [(2049, 64), (24, 4096)])
def test_quantise(n, k, group):
    w = weight_of(n + k, n, k)
    codes, scales, zeros = R.quantise(w, group)
    got = ops.quantise_w4(w, group)
    assert got[1:] == (n, k, group)
    for a, b in zip(R.unpack(got.records, n, k, group), (codes, scales, zeros)):
        assert torch.equal(a, b)
    exact = R.values(codes, scales, zeros, group)
    assert torch.equal(ops.dequantise_w4(got, torch.float32).cpu().double(), exact)
    assert torch.equal(ops.dequantise_w4(got).cpu(), exact.float().bfloat16())
    # what lies behind the last row or column is zero, and packing its codes gives the same bytes
    again = ops.pack_w4(codes.to(DEV, torch.uint8), scales.to(DEV, torch.bfloat16), zeros.to(DEV, torch.uint8), group)
    assert torch.equal(again.records, got.records)


def test_quantise_groups_of_every_kind():
    w = torch.zeros(16, 64, dtype=torch.bfloat16, device=DEV)
    g = gen(1)
    x = torch.randn(16, 64, generator=g, device=DEV)
    w[1] = 0.5                                  # one value
    w[2] = -3.0
    w[3] = x[3].abs().bfloat16()                # no negative
    w[4] = -x[4].abs().bfloat16()
    w[5] = (x[5] * 1e-38).bfloat16()            # scales that are subnormal
    w[6] = (x[6] * 2.0 ** -130).bfloat16()
    w[7] = (x[7] * 1e37).bfloat16()
    w[8] = torch.arange(64, device=DEV).bfloat16() / 2  # borders between codes: scale 2.1, and below 2
    w[9, :32], w[9, 32:] = -7.5, 7.5
    w[10] = torch.arange(64, device=DEV).remainder(31).bfloat16() - 15
    w[11, 0], w[11, 1] = 15.0, 0.5
    w[12, 0], w[12, 1], w[12, 2] = -7.5, 7.5, 0.5
    got = ops.quantise_w4(w, 64)
    codes, scales, zeros = R.quantise(w, 64)
    a, b, c = R.unpack(got.records, 16, 64, 64)
    assert torch.equal(b, scales) and torch.equal(c, zeros) and torch.equal(a, codes)
    bad = w.clone()
    bad[1, 5], bad[2, 0], bad[3, 63], bad[4, 7], bad[4, 8] = math.nan, math.inf, -math.inf, 3.3e38, -3.3e38
    back = ops.dequantise_w4(ops.quantise_w4(bad, 32))
    good = ops.dequantise_w4(ops.quantise_w4(w, 32))
    touched = torch.zeros(16, 2, dtype=torch.bool, device=DEV)
    touched[1, 0] = touched[2, 0] = touched[3, 1] = touched[4, 0] = True
    touched = touched.repeat_interleave(32, 1)
    assert back[touched].isnan().all() and torch.equal(back[~touched], good[~touched])


def test_pack_and_layouts_of_inputs():
    n, k, group = 40, 96, 64
    g = gen(2)
    codes = torch.randint(0, 256, (n, k), generator=g, device=DEV, dtype=torch.uint8)  # the low 4 bits count
    scales = torch.rand(n, 2, generator=g, device=DEV).bfloat16()
    w = ops.pack_w4(codes, scales, None, group)
    a, b, c = R.unpack(w.records, n, k, group)
    assert torch.equal(a, codes.cpu().long() & 15) and torch.equal(b, scales.cpu().double()) and (c == 8).all()
    apart = torch.zeros(n, 2 * k, dtype=torch.uint8, device=DEV)
    apart[:, 1:k + 1] = codes
    assert torch.equal(ops.pack_w4(apart[:, 1:k + 1], scales, None, group).records, w.records)
    big = weight_of(3, n, 3 * k)
    for t in (big[:, 8:8 + k], big[:, 3:3 + k], big.t()[:k].t()):
        assert torch.equal(ops.quantise_w4(t, group).records, ops.quantise_w4(t.contiguous(), group).records)
    none = ops.quantise_w4(big[:0], group)
    assert none.records.shape[0] == 0 and ops.dequantise_w4(none).shape == (0, 3 * k)
    assert ops.linear_w4(rows_of(1, 3, 3 * k, False)[0], none).shape == (3, 0)


# ------------------------------------------------------------------------------------ products
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n, k", SHAPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 6, 8, 16, 17, 33, 64, 65, 150])
def test_linear(rows, n, k, group, q8):
    w, exact = packed(n + k + group, n, k, group)
    x, x64 = rows_of(rows, rows, k, q8)
    check(ops.linear_w4(x, w), x64, exact, group)
    assert N.device_status() == 0


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("rows, n, k, group", [
    (1, 4096, 4096, 128), (4, 6144, 4096, 128), (1, 2048, 1024, 64), (7, 4096, 12288, 128), (16, 9000, 2048, 32),
    (64, 4096, 4096, 128), (64, 6144, 4096, 64), (40, 24576, 1024, 128), (200, 4096, 2048, 32), (1000, 1536, 4096, 128),
    (2, 16, 32768, 128), (20, 16, 32768, 32), (3, 100, 16384, 64), (8, 33, 20480, 32), (64, 8, 32768, 64), (600, 16, 32, 32),
    (1, 40000, 256, 128), (3000, 300, 96, 64),
])
def test_linear_sizes(rows, n, k, group, q8):
    w, exact = packed(7, n, k, group)
    x, x64 = rows_of(8, rows, k, q8)
    check(ops.linear_w4(x, w), x64, exact, group)
    assert N.device_status() == 0


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("rows", [1, 4, 16, 70])
def test_weights_quantised_here_and_symmetric_zeros(rows, q8):
    w = ops.quantise_w4(weight_of(4, 200, 640), 64)
    x, x64 = rows_of(5, rows, 640, q8)
    check(ops.linear_w4(x, w), x64, ops.dequantise_w4(w, torch.float32).double(), 64)
    codes = torch.randint(0, 16, (200, 640), generator=gen(6), device=DEV, dtype=torch.uint8)
    scales = torch.rand(200, 5, generator=gen(7), device=DEV).bfloat16()
    w = ops.pack_w4(codes, scales, group=128)
    exact = R.values(codes.cpu().long(), scales.cpu().double(), torch.full((200, 5), 8), 128).to(DEV)
    check(ops.linear_w4(x, w), x64, exact, 128)


@pytest.mark.parametrize("rows", [1, 5, 16, 64])
def test_elements_far_below_their_groups_largest(rows):
    """2^-k of the largest, k from 0 to 40 within a group: what the three 8-bit rows hold."""
    k = 256
    x = torch.exp2(-torch.arange(k, device=DEV).remainder(41).float()).repeat(rows, 1)
    x = (x * (1 + torch.rand(rows, k, generator=gen(8), device=DEV))).bfloat16()
    w, exact = packed(9, 64, k, 128)
    check(ops.linear_w4(x, w), x.double(), exact, 128)
    only = torch.zeros_like(x)
    only[:, ::37] = x[:, ::37]
    check(ops.linear_w4(only, w), only.double(), exact, 128)
    for f in (1e-30, 1e30, 2.0 ** -100):
        y = (x.float() * f).bfloat16()
        check(ops.linear_w4(y, w), y.double(), exact, 128)
    assert (ops.linear_w4(torch.zeros_like(x), w) == 0).all()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("rows", [3, 16, 64, 100])
def test_a_row_that_is_not_finite_leaves_the_others(rows, q8):
    w, exact = packed(10, 150, 320, 64)
    x, x64 = rows_of(11, rows, 320, q8)
    plain = ops.linear_w4(x, w)
    if q8:
        x.scales[1] = math.nan
    else:
        x[1, 77], x[2, 0] = math.nan, math.inf
    got = ops.linear_w4(x, w)
    assert got[1].isnan().all() and (q8 or not got[2].isfinite().any())
    keep = [i for i in range(rows) if i not in (1, 2)]
    assert torch.equal(got[keep], plain[keep])


def test_a_group_that_is_not_finite_leaves_the_other_rows():
    weight = weight_of(12, 64, 256)
    weight[5, 200] = math.nan
    w = ops.quantise_w4(weight, 64)
    clean = ops.quantise_w4(torch.where(weight.isnan(), 0, weight), 64)
    for rows in (1, 64):
        for q8 in (False, True):
            x, _ = rows_of(13, rows, 256, q8)
            got, plain = ops.linear_w4(x, w), ops.linear_w4(x, clean)
            assert got[:, 5].isnan().all()
            keep = [i for i in range(64) if i != 5]
            assert torch.equal(got[:, keep], plain[:, keep])


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("rows", [1, 4, 12, 64, 130])
def test_the_same_on_every_call_and_for_every_order_of_rows(rows, q8):
    w, _ = packed(14, 1000, 2048, 128)
    x, _ = rows_of(15, rows, 2048, q8)
    first = ops.linear_w4(x, w)
    for _ in range(3):
        assert torch.equal(ops.linear_w4(x, w), first)
    order = torch.randperm(rows, generator=gen(16), device=DEV)
    mixed = ops.Q8Rows(x.values[order].contiguous(), x.scales[order].contiguous()) if q8 else x[order].contiguous()
    assert torch.equal(ops.linear_w4(mixed, w), first[order])


def test_shapes_strides_and_outputs():
    w, exact = packed(17, 100, 256, 64)
    base = torch.randn(12, 600, generator=gen(18), device=DEV).bfloat16()
    for x in (base[:, 8:264], base[:, 3:259], base[:, 264:520], base.t()[:256].t(), base[0, :256], base[:, :512].reshape(3, 4, 2, 256),
              base[:1, 40:296], base[::5, :256]):
        flat = x.reshape(-1, 256)
        got = ops.linear_w4(x, w)
        assert got.shape == (*x.shape[:-1], 100)
        assert torch.equal(got.reshape(-1, 100), ops.linear_w4(flat.contiguous(), w))
    for rows in (3, 12):  # both kernels
        wide = torch.full((rows + 2, 130), 7.0, dtype=torch.bfloat16, device=DEV)
        out = wide[1:rows + 1, 10:110]
        x = base[:rows, :256]
        assert ops.linear_w4(x, w, out=out) is out
        assert torch.equal(out, ops.linear_w4(x.contiguous(), w))
        out.fill_(7.0)
        assert (wide == 7.0).all()
    q = ops.quantise_q8(base)
    part = ops.Q8Rows(q.values[:, 16:272], q.scales)
    assert torch.equal(ops.linear_w4(part, w), ops.linear_w4(ops.Q8Rows(part.values.contiguous(), q.scales), w))
    odd = ops.Q8Rows(q.values[:, 5:261], q.scales)
    assert torch.equal(ops.linear_w4(odd, w), ops.linear_w4(ops.Q8Rows(odd.values.contiguous(), q.scales), w))
    assert ops.linear_w4(base[:0, :256], w).shape == (0, 100)
    assert ops.linear_w4(ops.quantise_q8(base[:, :256].view(2, 6, 256)), w).shape == (2, 6, 100)


def test_refusals():
    w, _ = packed(19, 32, 128, 128)
    x = rows_of(20, 4, 128, False)[0]
    q = ops.quantise_q8(x)
    for call in (
        lambda: ops.linear_w4(x.float(), w),
        lambda: ops.linear_w4(x[:, :96], w),
        lambda: ops.linear_w4(x.cpu(), w),
        lambda: ops.linear_w4(ops.Q8Rows(q.values, q.scales[:3]), w),
        lambda: ops.linear_w4(ops.Q8Rows(q.values.cpu(), q.scales), w),
        lambda: ops.linear_w4((q.values, q.scales), w),
        lambda: ops.linear_w4(x, w._replace(n=33)),
        lambda: ops.linear_w4(x, w._replace(group=64)),
        lambda: ops.linear_w4(x, w._replace(k=160)),
        lambda: ops.linear_w4(x, w._replace(records=w.records[:, :1024])),
        lambda: ops.linear_w4(x, w, out=torch.empty(4, 33, dtype=x.dtype, device=DEV)),
        lambda: ops.linear_w4(x, w, out=torch.empty(32, 4, dtype=x.dtype, device=DEV).t()),
        lambda: ops.linear_w4(x, w, out=torch.empty(4, 32, device=DEV)),
        lambda: ops.linear_w4(torch.zeros(1, 32800, dtype=x.dtype, device=DEV),
                              ops.quantise_w4(torch.zeros(1, 32800, dtype=x.dtype, device=DEV), 32)),
        lambda: ops.quantise_w4(x.float()),
        lambda: ops.quantise_w4(x, 16),
        lambda: ops.quantise_w4(x[:, :40]),
        lambda: ops.quantise_w4(x[0]),
        lambda: ops.pack_w4(q.values, torch.zeros(4, 1, dtype=x.dtype, device=DEV)),
        lambda: ops.pack_w4(q.values.view(torch.uint8), torch.zeros(4, 2, dtype=x.dtype, device=DEV)),
        lambda: ops.dequantise_w4(w, torch.float16),
        lambda: ops.dequantise_w4(w._replace(records=None)),
    ):
        with pytest.raises(RuntimeError):
            call()


# ----------------------------------------------------------------------- streams, graphs, devices
@pytest.mark.parametrize("rows", [1, 64])
def test_two_streams_at_once(rows):
    w, _ = packed(21, 4096, 1024, 128)
    v, _ = packed(22, 3000, 1024, 64)
    x, _ = rows_of(23, rows, 1024, False)
    q, _ = rows_of(24, rows, 1024, True)
    one, two = ops.linear_w4(x, w), ops.linear_w4(q, v)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(a):
            got_a = [ops.linear_w4(x, w) for _ in range(4)]
        with torch.cuda.stream(b):
            got_b = [ops.linear_w4(q, v) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(t, one) for t in got_a) and all(torch.equal(t, two) for t in got_b)


@pytest.mark.parametrize("rows", [1, 5, 64])
def test_two_graphs_of_a_layer_replayed_on_new_rows(rows):
    """The linear layers of a decoder layer as they follow one another, against the same calls one by one."""
    hidden, inter = 512, 1024
    qkv, _ = packed(25, 768, hidden, 128)
    gate_up, _ = packed(26, 2 * inter, hidden, 64)
    down, _ = packed(27, hidden, inter, 128)
    w = torch.randn(hidden, generator=gen(28), device=DEV).bfloat16()
    x, res = rows_of(29, rows, hidden, False)[0], rows_of(30, rows, hidden, False)[0]
    start = res.clone()

    def layer():
        h, _ = ops.fused_add_rmsnorm_q8(res, x, w)
        a = ops.linear_w4(h, qkv)
        gate, up = ops.linear_w4(h, gate_up).chunk(2, -1)
        return a, ops.linear_w4(ops.swiglu_q8(gate, up), down)

    layer()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer())
        graphs.append(g)
    for seed in (31, 32):
        x.copy_(rows_of(seed, rows, hidden, False)[0])
        for g, out in zip(graphs, outs):
            res.copy_(start)
            g.replay()
            got = [t.clone() for t in out]
            res.copy_(start)
            for a, b in zip(got, layer()):
                assert torch.equal(a, b)


def test_a_layer_against_its_formulas():
    """Norm, product, activation and product, each from what the one before gave, in 64 bits."""
    hidden, inter, rows = 512, 768, 9
    gate_up, gu64 = packed(33, 2 * inter, hidden, 128)
    down, down64 = packed(34, hidden, inter, 32)
    w = torch.randn(hidden, generator=gen(35), device=DEV).bfloat16()
    x, res = rows_of(36, rows, hidden, False)[0], rows_of(37, rows, hidden, False)[0]
    h, total = ops.fused_add_rmsnorm_q8(res.clone(), x, w)
    y, inv = R.normed((res.float() + x.float()).bfloat16().double(), w.double(), 1e-6, False)
    codes, scale = R.q8(y)
    assert torch.equal(h.values.double(), codes.round())
    h64 = codes.round() * (scale * inv)[:, None]
    # a scale is off by 2^-18 of itself at most (w4_reference), far below the bound's 2^-8
    gu = ops.linear_w4(h, gate_up)
    exact = h64 @ gu64.T
    assert ((gu.double() - exact).abs() <= R.linear_bound(h64, gu64, 128, exact) + 2.0 ** -18 * exact.abs()).all()
    a = ops.swiglu_q8(*gu.chunk(2, -1))
    back = a.values.double() * a.scales.double()[:, None]
    y = R.gated(gu.double()[:, :inter], gu.double()[:, inter:], False)
    assert ((back - y).abs() <= y.abs().amax(-1, keepdim=True) * (0.5 / 127 + 4e-5)).all()
    out = ops.linear_w4(a, down)
    check(out, back, down64, 32)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("bits", [8, 16])
def test_fused_mlp_w4(act, bits):
    torch.manual_seed(0)
    mlp = ops.FusedMLP(256, 384, act).to(DEV, torch.bfloat16)
    small = ops.FusedMLPW4(mlp, group=64, rows=bits)
    x = rows_of(38, 11, 256, False)[0]
    with torch.no_grad():
        got = small(x)
        gate_up = ops.W4Weight(small.gate_up, 768, 256, 64)
        down = ops.W4Weight(small.down, 256, 384, 64)
        rows = ops.quantise_q8(x) if bits == 8 else x
        gu = ops.linear_w4(rows, gate_up)
        if bits == 8:
            want = ops.linear_w4((ops.swiglu_q8 if act == "silu" else ops.geglu_q8)(*gu.chunk(2, -1)), down)
            assert torch.equal(small(rows), got)
        else:
            want = ops.linear_w4(ops.fused_mlp_forward(gu, 384, 0 if act == "silu" else 1), down)
    assert torch.equal(got, want)
    again = ops.FusedMLPW4(ops.FusedMLP(256, 384, act).to(DEV, torch.bfloat16), group=64, rows=bits)
    again.load_state_dict(small.state_dict())
    assert torch.equal(again(x), got)
    with pytest.raises(ValueError):
        ops.FusedMLPW4(mlp, rows=4)


def test_namespace():
    import llm_pytorch_inference_b200.torch_ops as T
    space = getattr(torch.ops, T.NAMESPACE)
    weight = weight_of(39, 48, 128)
    w = ops.quantise_w4(weight, 32)
    assert torch.equal(space.quantise_w4(weight, 32), w.records)
    assert torch.equal(space.dequantise_w4(w.records, 48, 128, 32), ops.dequantise_w4(w))
    x = rows_of(40, 3, 128, False)[0]
    q = ops.quantise_q8(x)
    assert torch.equal(space.linear_w4(x, None, w.records, 48, 128, 32), ops.linear_w4(x, w))
    assert torch.equal(space.linear_w4(q.values, q.scales, w.records, 48, 128, 32), ops.linear_w4(q, w))
    codes = torch.randint(0, 16, (48, 128), generator=gen(41), device=DEV, dtype=torch.uint8)
    scales = torch.rand(48, 1, device=DEV).bfloat16()
    assert torch.equal(space.pack_w4(codes, scales, None, 128), ops.pack_w4(codes, scales).records)


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one():
    w, _ = packed(42, 64, 256, 128)
    x, _ = rows_of(43, 4, 256, False)
    want = ops.linear_w4(x, w)
    there = ops.W4Weight(w.records.to("cuda:1"), *w[1:])
    assert torch.equal(ops.linear_w4(x.to("cuda:1"), there).to(DEV), want)
    with pytest.raises(RuntimeError):
        ops.linear_w4(x, there)


def test_launches_that_follow_one_another_early():
    """With programmatic dependent launch on: each kernel waits for the rows of the one before."""
    w, _ = packed(44, 512, 512, 128)
    x, _ = rows_of(45, 3, 512, False)
    big, _ = rows_of(46, 64, 512, False)

    def chain(t):
        for _ in range(6):
            t = ops.linear_w4(ops.quantise_q8(t), w)
            t = ops.dequantise_q8(ops.quantise_q8(t))
        return t

    want = chain(x), chain(big)
    before = N.set_pdl(True)
    try:
        for _ in range(5):
            assert torch.equal(chain(x), want[0]) and torch.equal(chain(big), want[1])
    finally:
        N.set_pdl(before)
    assert N.device_status() == 0


def test_products_right_after_their_weight_is_made():
    """A product asks for records before it waits for the kernel before it, which here makes them."""
    before = N.set_pdl(True)
    try:
        for seed in range(6):
            weight, (x, _) = weight_of(50 + seed, 2048, 1024), rows_of(60 + seed, 3, 1024, False)
            many = x.repeat(30, 1)
            torch.cuda.synchronize()
            got = ops.linear_w4(x, ops.quantise_w4(weight))
            got_many = ops.linear_w4(many, ops.quantise_w4(weight, 32))
            codes = torch.randint(0, 16, (2048, 1024), generator=gen(70 + seed), device=DEV, dtype=torch.uint8)
            scales = torch.rand(2048, 8, generator=gen(80 + seed), device=DEV).bfloat16()
            got_packed = ops.linear_w4(x, ops.pack_w4(codes, scales))
            torch.cuda.synchronize()
            for weight_of_it, rows, y in ((ops.quantise_w4(weight), x, got), (ops.quantise_w4(weight, 32), many, got_many),
                                          (ops.pack_w4(codes, scales), x, got_packed)):
                torch.cuda.synchronize()
                assert torch.equal(y, ops.linear_w4(rows, weight_of_it))
    finally:
        N.set_pdl(before)


def test_an_extent_beyond_fp32():
    """hi - lo infinite in fp32: the group reads back as NaN, its neighbours as what they are."""
    weight = weight_of(52, 32, 128)
    weight[3, 5], weight[3, 9] = 3e38, -3e38
    back = ops.dequantise_w4(ops.quantise_w4(weight, 32))
    assert back[3, :32].isnan().all()
    back[3, :32] = 0
    rest = weight.clone()
    rest[3, :32] = 0
    assert torch.equal(back, ops.dequantise_w4(ops.quantise_w4(rest, 32)))


@pytest.mark.parametrize("q8", [False, True])
def test_offsets_beyond_32_bits(q8):
    """Records of 2.6 GB, results of 3.0e9 elements: the last rows are those of a weight of their own."""
    n, k = 300000, 16384
    weight = torch.zeros(n, k, dtype=torch.bfloat16, device=DEV)
    weight[-48:] = weight_of(53, 48, k)
    own = ops.quantise_w4(weight[-48:])
    w = ops.quantise_w4(weight)
    assert torch.equal(ops.dequantise_w4(w)[-48:], ops.dequantise_w4(own))
    del weight
    for rows in (2, 40):
        x, x64 = rows_of(54, rows, k, q8)
        y = ops.linear_w4(x, w)
        assert (y[:, :-48] == 0).all()
        check(y[:, -48:], x64, ops.dequantise_w4(own, torch.float32).double(), 128)
    del w
    small, exact = packed(55, 150000, 64, 64)
    x, x64 = rows_of(56, 20000, 64, q8)
    y = ops.linear_w4(x, small)
    check(y[-3:], x64[-3:], exact, 64)
    check(y[:, -3:], x64, exact[-3:], 64)


@pytest.mark.parametrize("rows, n, k, group, q8", [
    (5, 40, 12288, 128, False), (6, 40, 12288, 128, False), (8, 600, 8192, 64, False), (8, 600, 8224, 32, False),
    (16, 100, 32768, 128, True), (17, 2400, 1024, 64, True), (65, 2000, 1024, 32, False), (128, 2500, 544, 128, True),
    (129, 130, 4096, 64, False), (300, 1000, 4096, 32, True), (64, 24576, 256, 64, False), (30, 24576, 288, 32, True),
    (640, 4096, 512, 128, False), (1100, 136, 2048, 64, True),
])
def test_either_side_of_every_choice_of_kernel(rows, n, k, group, q8):
    """Few rows and more by rows and k, one or two halves of weight rows, 32, 64 or 128 rows of x, columns split or not."""
    w, exact = packed(rows + n, n, k, group)
    x, x64 = rows_of(rows, rows, k, q8)
    check(ops.linear_w4(x, w), x64, exact, group)
    assert N.device_status() == 0
