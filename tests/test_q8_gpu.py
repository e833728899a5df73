"""Rows in 8 bits (quantise_q8, the norms, the gated activations) against their formulas in 64 bits."""
import math

import pytest
import torch

import w4_reference as R
from llm_pytorch_inference_b200 import _native as N
from llm_pytorch_inference_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rows_of(seed, *shape, dtype=torch.bfloat16, wide=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(*shape, generator=g, device=DEV)
    if wide:
        x = x * torch.exp(torch.randn(*shape[:-1], 1, generator=g, device=DEV))
    return x.to(dtype)


def check(rows, y, scale, exact, rel):
    """Codes of y (64 bits): the nearest whole numbers to 127 y / amax where `exact` (ties to even), else off by what y
    may be, `rel` (a number, or one a row) of amax, and so may amax; scales within what 32 bits give."""
    values, scales = rows
    assert values.dtype is torch.int8 and scales.dtype is torch.float32
    assert values.shape == y.shape and scales.shape == y.shape[:-1] and values.is_contiguous()
    want, _ = R.q8(y)
    rel = torch.as_tensor(rel, dtype=torch.float64, device=DEV)
    if exact:
        assert torch.equal(values.double(), want.round())
    else:
        # y and amax are off by rel, and the quotient is rounded to 2^-24 of itself twice
        assert ((values.double() - want).abs() <= 0.5 + 127 * (2 * rel[..., None] + 2.0 ** -23)).all()
    # the sum of squares, a thread's share after the other; its root halves that; then a few roundings
    off = 2.0 ** -24 * (y.shape[-1] / 256 + 64) + 2 * rel
    assert ((scales.double() - scale).abs() <= off * scale).all()


def gated_off(gate, up, y, gelu):
    """How far y may be off, relative to its row's amax.  The quotient and the exponential are off by 6 + 1.2 |z| units of
    2^-24, and z, for gelu, by 3 of its own; |z| < 104 where fp32 has a number for e^z: 131 and 443 units.  Below 2^-126
    fp32's numbers are 2^-149 apart: e^z, its product with the gate and the result are each off by half of that."""
    apart = 2.0 ** -149 * (gate.double().abs() * up.double().abs() + up.double().abs() + 1).amax(-1)
    amax = y.abs().amax(-1)
    return (443 if gelu else 131) * 2.0 ** -24 + apart / torch.where(amax > 0, amax, 1.0)


WIDTHS = [1, 7, 8, 32, 64, 520, 2048, 2179, 4096, 14336, 33000]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows", [1, 3, 700])
def test_quantise_q8(rows, width):
    x = rows_of(rows + width, rows, width)
    got = ops.quantise_q8(x)
    check(got, x.double(), R.q8(x.double())[1], True, 0.0)
    back = ops.dequantise_q8(got)
    exact = got.values.double() * got.scales.double()[:, None]
    assert ((back.double() - exact).abs() <= HALF[torch.bfloat16] * 1.001 * exact.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("width", [8, 9, 4096])
def test_other_types(dtype, width):
    x, r, w = rows_of(1, 37, width, dtype=dtype), rows_of(2, 37, width, dtype=dtype), rows_of(3, width, dtype=dtype, wide=False)
    check(ops.quantise_q8(x), x.double(), R.q8(x.double())[1], False, 0.0)
    y, inv = R.normed(x.double(), w.double(), 1e-5, False)
    check(ops.rmsnorm_q8(x, w, 1e-5), y, R.q8(y)[1] * inv, False, 2.0 ** -24)
    h = (r.double() + x.double()).float().to(dtype) if dtype is torch.float32 else (r.float() + x.float()).to(dtype)
    got, total = ops.fused_add_rmsnorm_q8(r.clone(), x, w, 1e-5, plus_one=True)
    assert torch.equal(total, h)
    y, inv = R.normed(h.double(), w.double(), 1e-5, True)
    check(got, y, R.q8(y)[1] * inv, False, 2.0 ** -23)
    y = R.gated(x.double(), r.double(), False)
    check(ops.swiglu_q8(x, r), y, R.q8(y)[1], False, gated_off(x, r, y, False))
    for to in (torch.float32, torch.float16, torch.bfloat16):
        q = ops.quantise_q8(rows_of(4, 37, width, dtype=dtype))
        exact = q.values.double() * q.scales.double()[:, None]
        # in 32 bits first, then to the type; below its normal numbers a fixed step
        off = (HALF[to] + 2.0 ** -24) * exact.abs() * 1.001 + (2.0 ** -25 if to is torch.float16 else 0)
        assert ((ops.dequantise_q8(q, to).double() - exact).abs() <= off).all()


@pytest.mark.parametrize("plus_one", [False, True])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows", [1, 64, 700])
def test_norms(rows, width, plus_one):
    x, r = rows_of(width, rows, width), rows_of(width + 1, rows, width)
    w = rows_of(width + 2, width, wide=False)
    rel = 2.0 ** -23 if plus_one else 0.0  # 1 + w, and its product, are rounded to 32 bits
    y, inv = R.normed(x.double(), w.double(), 1e-6, plus_one)
    check(ops.rmsnorm_q8(x, w, 1e-6, plus_one), y, R.q8(y)[1] * inv, not plus_one, rel)
    h = (r.float() + x.float()).bfloat16()
    y, inv = R.normed(h.double(), w.double(), 1e-6, plus_one)
    out = torch.empty_like(r)
    before = r.clone()
    got, total = ops.fused_add_rmsnorm_q8(r, x, w, 1e-6, plus_one, residual_out=out)
    assert total is out and torch.equal(out, h) and torch.equal(r, before)
    check(got, y, R.q8(y)[1] * inv, not plus_one, rel)
    again, total = ops.fused_add_rmsnorm_q8(r, x, w, 1e-6, plus_one)
    assert total is r and torch.equal(r, h)
    assert torch.equal(again.values, got.values) and torch.equal(again.scales, got.scales)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("width", [1, 8, 100, 768, 12288, 14336, 40000])
@pytest.mark.parametrize("rows", [1, 5, 400])
def test_gated(rows, width, act):
    both = rows_of(width, rows, 2 * width)
    gate, up = both.chunk(2, -1)
    f = ops.swiglu_q8 if act == "silu" else ops.geglu_q8
    y = R.gated(gate.double(), up.double(), act == "gelu")
    check(f(gate, up), y, R.q8(y)[1], False, gated_off(gate, up, y, act == "gelu"))
    apart = f(gate.contiguous(), up.contiguous())
    assert torch.equal(f(gate, up).values, apart.values)


@pytest.mark.parametrize("width", [8, 9, 4096])
def test_rows_that_are_zero_tiny_huge_or_not_finite(width):
    x = rows_of(5, 9, width, wide=False)
    x[0] = 0
    x[1] *= 1e-38
    x[2] *= 2.0 ** -133  # subnormal
    x[3] = x[3] / x[3].abs().max() * 3e38
    x[4, width // 2] = math.inf
    x[5, width - 1] = math.nan
    x[6, 0] = -math.inf
    x[7] = -0.0
    got = ops.quantise_q8(x)
    fine = [1, 2, 3, 8]
    check(ops.Q8Rows(got.values[fine].contiguous(), got.scales[fine].where(got.scales[fine] > 2.0 ** -120, 1.0)),
          x[fine].double(), R.q8(x[fine].double())[1].where(got.scales[fine] > 2.0 ** -120, 1.0), True, 0.0)
    for i in (0, 7):
        assert got.scales[i] == 0 and (got.values[i] == 0).all()
    for i in (4, 5, 6):
        assert got.scales[i].isnan() and (got.values[i] == 0).all()
        assert ops.dequantise_q8(got)[i].isnan().all()
    w = torch.ones(width, dtype=torch.bfloat16, device=DEV)
    one, _ = ops.fused_add_rmsnorm_q8(x.clone(), torch.zeros_like(x), w)
    assert torch.equal(one.scales.isnan().nonzero().flatten().cpu(), torch.tensor([4, 5, 6]))
    assert one.scales[0] == 0
    two = ops.swiglu_q8(x, torch.ones_like(x))
    assert two.scales[4].isnan() and two.scales[5].isnan() and not two.scales[[0, 1, 2, 3, 7, 8]].isnan().any()


def test_strides_shapes_and_alignment():
    base = rows_of(6, 40, 300)
    x = base[:, 8:264]                     # rows apart
    odd = base[:, 3:259]                   # and not on 16 bytes
    for t in (x, odd, base.t()[:40], base[:, :256].view(5, 8, 256), base[::2, :64], base[:1, 5:6], base[3]):
        got = ops.quantise_q8(t)
        want = ops.quantise_q8(t.contiguous().clone())
        assert got.values.shape == t.shape and got.scales.shape == t.shape[:-1]
        assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales)
    w = rows_of(7, 256, wide=False)
    wide = torch.zeros(40, 300, dtype=torch.bfloat16, device=DEV)
    res = wide[:, 8:264]
    res.copy_(rows_of(8, 40, 256))
    plain, _ = ops.fused_add_rmsnorm_q8(res.contiguous(), x.contiguous(), w)
    total = (res.float() + x.float()).bfloat16()
    got, out = ops.fused_add_rmsnorm_q8(res, x, w)
    assert torch.equal(got.values, plain.values) and torch.equal(out, total) and torch.equal(res, total)
    assert (wide[:, :8] == 0).all() and (wide[:, 264:] == 0).all()
    # the sum into the input
    x2 = x.contiguous()
    r2 = rows_of(8, 40, 256)
    got, _ = ops.fused_add_rmsnorm_q8(r2, x2, w, residual_out=x2)
    assert torch.equal(got.values, plain.values) and torch.equal(x2, total)
    q = ops.quantise_q8(base)
    part = ops.Q8Rows(q.values[::3, 16:272], q.scales[::3])
    assert torch.equal(ops.dequantise_q8(part), ops.dequantise_q8(ops.Q8Rows(part.values.contiguous(), part.scales.contiguous())))
    for empty in (x[:0], torch.empty(3, 0, 8, dtype=torch.bfloat16, device=DEV)):
        got = ops.quantise_q8(empty)
        assert got.values.shape == empty.shape and got.scales.shape == empty.shape[:-1]
        assert ops.dequantise_q8(got).shape == empty.shape


def test_refusals():
    x, w = rows_of(9, 4, 64), rows_of(10, 64, wide=False)
    for call in (
        lambda: ops.quantise_q8(x.int()),
        lambda: ops.quantise_q8(torch.zeros((), device=DEV)),
        lambda: ops.quantise_q8(x[:, :0]),
        lambda: ops.rmsnorm_q8(x, w[:63]),
        lambda: ops.rmsnorm_q8(x, w.cpu()),
        lambda: ops.fused_add_rmsnorm_q8(x[:3], x, w),
        lambda: ops.fused_add_rmsnorm_q8(x.float(), x, w),
        lambda: ops.fused_add_rmsnorm_q8(x, x, w, residual_out=torch.empty(64, 4, dtype=x.dtype, device=DEV).t()),
        lambda: ops.swiglu_q8(x, x[:, :32]),
        lambda: ops.swiglu_q8(x, x.cpu()),
        lambda: ops.geglu_q8(x, None),
        lambda: ops.dequantise_q8(ops.Q8Rows(x, torch.zeros(4, device=DEV))),
        lambda: ops.dequantise_q8(ops.Q8Rows(x.to(torch.int8), torch.zeros(3, device=DEV))),
        lambda: ops.dequantise_q8(ops.quantise_q8(x), torch.int8),
        lambda: ops.dequantise_q8((None, None)),
    ):
        with pytest.raises(RuntimeError):
            call()
    before = x.clone()
    assert torch.equal(x, before)


def test_graph_stream_and_namespace():
    x, r, w = rows_of(11, 33, 512), rows_of(12, 33, 512), rows_of(13, 512, wide=False)
    out = torch.empty_like(r)

    def step():
        rows, total = ops.fused_add_rmsnorm_q8(r, x, w, residual_out=out)
        return rows, ops.dequantise_q8(rows)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, back = step()
    x.copy_(rows_of(14, 33, 512))
    graph.replay()
    fresh, values = step()
    assert torch.equal(held.values, fresh.values) and torch.equal(back, values)
    assert not torch.equal(held.values, first[0].values)
    import llm_pytorch_inference_b200.torch_ops as T
    space = getattr(torch.ops, T.NAMESPACE)
    a, b = space.fused_add_rmsnorm_q8(r.clone(), x, w, 1e-6, False)
    assert torch.equal(a, fresh.values) and torch.equal(b, fresh.scales)
    assert torch.equal(space.dequantise_q8(a, b), values)
    for act, f in ((N.ACT_SILU, ops.swiglu_q8), (N.ACT_GELU_TANH, ops.geglu_q8)):
        assert torch.equal(space.gated_q8(x, r, act)[0], f(x, r).values)
    assert torch.equal(space.quantise_q8(x)[0], ops.quantise_q8(x).values)
    assert torch.equal(space.rmsnorm_q8(x, w, 1e-6, True)[1], ops.rmsnorm_q8(x, w, 1e-6, True).scales)
    assert N.device_status() == 0


def test_offsets_beyond_32_bits():
    """2.3e9 elements: the last rows are what they are by themselves."""
    x = torch.zeros(140000, 16384, dtype=torch.bfloat16, device=DEV)
    x[-5:] = rows_of(90, 5, 16384)
    last = x[-5:].clone()
    weight = rows_of(91, 16384, wide=False)
    for call in (ops.quantise_q8, lambda t: ops.rmsnorm_q8(t, weight), lambda t: ops.swiglu_q8(t, t),
                 lambda t: ops.fused_add_rmsnorm_q8(t, t, weight, residual_out=torch.empty_like(t))[0]):
        got, want = call(x), call(last)
        assert torch.equal(got.values[-5:], want.values)
        torch.testing.assert_close(got.scales[-5:], want.scales, rtol=2 ** -20, atol=0)  # squares are shared out otherwise
        assert not got.scales[:-5].any() and not got.values[:-5].any()
        back = ops.dequantise_q8(got)
        assert torch.equal(back[-5:], ops.dequantise_q8(ops.Q8Rows(got.values[-5:], got.scales[-5:])))
        assert not back[:-5].any()


@pytest.mark.parametrize("rows, width", [(1, 8191), (400, 8193), (2, 16385), (600, 4099), (3, 32767), (1, 32769), (310, 32773),
                                         (5, 8192), (2, 16384), (700, 16392)])
def test_rows_that_do_not_begin_on_16_bytes(rows, width):
    """Single elements, 8, 16 or 32 a thread, or worked out twice: what the aligned copy gives where there is one."""
    g = torch.Generator(device=DEV).manual_seed(width)
    base = torch.randn(2 * rows * width + 16, generator=g, device=DEV).bfloat16()
    x, z = base[1:1 + rows * width].view(rows, width), base[3 + rows * width:3 + 2 * rows * width].view(rows, width)
    weight = (1 + 0.2 * torch.randn(width + 1, generator=g, device=DEV)).bfloat16()[1:]
    h = (x.float() + z.float()).bfloat16()
    y = h.double() * weight.double()
    rstd = 1 / (h.double().square().mean(-1) + 1e-6).sqrt()
    got, residual = ops.fused_add_rmsnorm_q8(x.clone(), z, weight)
    assert torch.equal(residual, h)
    check(got, y, R.q8(y)[1] * rstd, True, 0.0)
    plain = ops.quantise_q8(x)
    check(plain, x.double(), R.q8(x.double())[1], True, 0.0)
    assert torch.equal(ops.dequantise_q8(plain), (plain.values.float() * plain.scales[:, None]).bfloat16())
    act = x.double() * torch.sigmoid(x.double()) * z.double()
    check(ops.swiglu_q8(x, z), act, R.q8(act)[1], False, gated_off(x, z, act, False))
