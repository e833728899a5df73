"""Rows in 8 bits and products of rows that are broadcast: what their copies give, and nothing behind them written."""
import pytest
import torch

from llm_pytorch_inference_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
WIDTH = 64


def views(seed):
    """[name, view] of rows, some dimensions of which are broadcast."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    a = torch.randn(4, WIDTH, generator=g, device=DEV).bfloat16()
    wide = torch.randn(4, 3 * WIDTH, generator=g, device=DEV).bfloat16()
    return [("inner", a[:, None].expand(4, 5, WIDTH)), ("outer", a[None].expand(3, 4, WIDTH)), ("both", a[0].expand(4, 5, WIDTH)),
            ("second of four", a.view(2, 1, 2, WIDTH).expand(2, 3, 2, WIDTH)),
            ("third of four", a.view(2, 2, 1, WIDTH).expand(2, 2, 3, WIDTH)), ("all of four", a[0].expand(2, 3, 4, WIDTH)),
            ("many of one", a[0].expand(7, 9, WIDTH)), ("of rows apart", wide[:, None, 8:8 + WIDTH].expand(4, 5, WIDTH)),
            ("of two", a[0].expand(6, WIDTH))]


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


CASES = ["inner", "outer", "both", "second of four", "third of four", "all of four", "many of one", "of rows apart", "of two"]


@pytest.mark.parametrize("name", CASES)
def test_inputs(name):
    x, z = dict(views(1))[name], dict(views(2))[name]
    xc, zc = x.contiguous(), z.contiguous()
    w = torch.randn(WIDTH, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).bfloat16()
    assert same(ops.quantise_q8(x), ops.quantise_q8(xc))
    assert same(ops.rmsnorm_q8(x, w), ops.rmsnorm_q8(xc, w))
    for f in (ops.swiglu_q8, ops.geglu_q8):
        assert same(f(x, z), f(xc, zc)) and same(f(x, zc), f(xc, zc)) and same(f(xc, z), f(xc, zc))
    out, want = torch.empty_like(xc), torch.empty_like(xc)
    assert same(ops.fused_add_rmsnorm_q8(z, x, w, residual_out=out)[0], ops.fused_add_rmsnorm_q8(zc, xc, w, residual_out=want)[0])
    assert torch.equal(out, want)
    q = ops.Q8Rows(_codes(x), z[..., 0].float())
    qc = ops.Q8Rows(q.values.contiguous(), q.scales.contiguous())
    assert torch.equal(ops.dequantise_q8(q), ops.dequantise_q8(qc))
    weight = ops.quantise_w4(torch.randn(48, WIDTH, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).bfloat16(), 32)
    assert torch.equal(ops.linear_w4(x, weight), ops.linear_w4(xc, weight))
    assert torch.equal(ops.linear_w4(q, weight), ops.linear_w4(qc, weight))


def _codes(x):
    """int8 codes laid out as x is: broadcast where it is."""
    base = x[tuple(slice(0, 1) if s == 0 else slice(None) for s in x.stride())]
    return base.float().mul(20).clamp(-127, 127).to(torch.int8).expand(x.shape)


@pytest.mark.parametrize("name", CASES)
def test_a_broadcast_sum_is_refused_and_nothing_is_written(name):
    shape = dict(views(1))[name].shape
    x = torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV).bfloat16()
    w = torch.ones(WIDTH, dtype=torch.bfloat16, device=DEV)
    target = dict(views(2))[name]
    before = target.clone()
    for call in (lambda: ops.fused_add_rmsnorm_q8(target, x, w),
                 lambda: ops.fused_add_rmsnorm_q8(x.clone(), x, w, residual_out=target)):
        with pytest.raises(RuntimeError, match="contiguous and evenly apart"):
            call()
    assert torch.equal(target, before)
