"""Attention over the 4-bit pool where magnitudes differ: channels of q, groups and tokens of V, each output against a
bound of its own."""
import math

import pytest
import torch

import kv4_reference as ref
from llm_pytorch_inference_b200 import _native as N
from llm_pytorch_inference_b200 import ops
from llm_pytorch_inference_b200.kv_cache import kv4_pool

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
# (query tokens, query heads, KV heads): up to 4, 8, 16 and 24 query rows of a KV head, and two chunks of them
ROWS = [(1, 4, 2), (1, 8, 2), (2, 6, 2), (3, 10, 2), (6, 8, 2), (7, 10, 2)]


@pytest.fixture(autouse=True)
def _status_clean():
    N.device_status(clear=True)
    yield
    assert N.device_status(clear=True) == 0, "a kernel reported a device-side error"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def case(q, k, v, scale):
    """One sequence: q [T, Hq, D], k and v [n, Hkv, D] in a pool of shuffled blocks."""
    n, heads, D = k.shape
    blocks = (n + 15) // 16
    order = torch.randperm(blocks, generator=gen(n), device=DEV)
    pool = kv4_pool(blocks, 16, 1, heads, D)
    at = torch.arange(n, device=DEV)
    ops.kv4_write(k.to(BF), v.to(BF), pool, 0, order[at // 16] * 16 + at % 16)
    return q.to(BF)[None], pool, 0, order.int()[None], torch.tensor([n], dtype=torch.int32, device=DEV), scale


def check(c, **kw):
    want, tol = ref.attention_each(*c, **kw)
    got = ops.paged_attention_decode_kv4(*c, **kw).double()
    assert bool(got.isfinite().all())
    over = (got - want).abs() - tol
    assert float(over.max()) <= 0, (float(((got - want).abs() / tol.clamp_min(1e-300)).max()),
                                    float((got - want).abs().max()))
    return want, tol


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,Hq,Hkv", ROWS)
def test_ordinary(D, T, Hq, Hkv):
    g = gen(D + T)
    c = case(normal(g, T, Hq, D), normal(g, 700, Hkv, D), normal(g, 700, Hkv, D) + 0.5, 1 / math.sqrt(D))
    check(c)
    check(c, softcap=20.0, window=333)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("T,Hq,Hkv", ROWS)
@pytest.mark.parametrize("big", [100.0, 1e4, 1e7])
def test_q_with_one_large_channel(D, T, Hq, Hkv, big):
    """A channel of q far above the others, over keys that say nothing there: the scores come from the small channels,
    which have to keep all their bits.  Half a step of 16 bits of the largest would be big / 65024 a channel."""
    g = gen(int(math.log10(big)) + D + T)
    n = 40
    q, k = normal(g, T, Hq, D), normal(g, n, Hkv, D)
    q[..., 70] = big
    k[..., 64:128] = 0.0
    c = case(q, k, normal(g, n, Hkv, D), 4 / math.sqrt(D))
    want, tol = check(c)
    coarse = (c[0].double() / (big / 32512)).round() * (big / 32512)     # q in 16 bits of the largest
    lost, _ = ref.attention_each(coarse, *c[1:])
    if big > 1000:                                                       # the bound tells it apart
        assert float(((lost - want).abs() > tol).double().mean()) > 0.2


@pytest.mark.parametrize("T,Hq,Hkv", ROWS)
def test_q_with_a_large_channel_over_keys_alike(T, Hq, Hkv):
    """As attention sinks and biased keys have it: one channel of q and k is large and the same for every key."""
    g = gen(T + Hq)
    D, n = 128, 2000
    q, k = normal(g, T, Hq, D), normal(g, n, Hkv, D)
    q[..., 5], k[..., 5] = 100.0, 3.0
    check(case(q, k, normal(g, n, Hkv, D), 1 / math.sqrt(D)))


@pytest.mark.parametrize("T,Hq,Hkv", ROWS)
@pytest.mark.parametrize("power", [-110, -60, 60, 100])
def test_q_and_k_of_any_magnitude(T, Hq, Hkv, power):
    """Queries tiny over huge keys and the other way round, with ordinary scores."""
    g = gen(power + 200)
    D, n = 128, 300
    f = 2.0 ** power
    check(case(normal(g, T, Hq, D) / f, normal(g, n, Hkv, D) * f, normal(g, n, Hkv, D), 0.09))


# ------------------------------------------------------------------ values of different magnitude
def telling(c, want, tol, groups=slice(None)):
    """The bound is one that zeros, and the groups' minima in place of the values, do not keep."""
    q, pool, layer, tables, ctx, scale = c
    plain = pool.clone()
    D = pool.shape[-1] // 18
    plain[..., 8 * D:16 * D] = 0                                         # the codes of V
    least, _ = ref.attention_each(q, plain, layer, tables, ctx, scale)
    for other in (torch.zeros_like(want), least):
        out = ((other - want).abs() > tol).unflatten(-1, (-1, 64))[..., groups, :]
        assert float(out.double().mean()) > 0.75


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("T,Hq,Hkv", ROWS)
@pytest.mark.parametrize("power", [-100, -30, -18, -14, 14, 40])
def test_groups_of_different_magnitude(D, T, Hq, Hkv, power):
    """One group of V 2^power of the others: each keeps its own bits."""
    g = gen(D + T + power + 500)
    n = 900
    v = normal(g, n, Hkv, D)
    v[..., 64:128] *= 2.0 ** power
    c = case(normal(g, T, Hq, D), normal(g, n, Hkv, D), v, 1 / math.sqrt(D))
    telling(c, *check(c))


@pytest.mark.parametrize("T,Hq,Hkv", ROWS)
@pytest.mark.parametrize("at", [0, 7, 450, 899])
@pytest.mark.parametrize("power", [10, 20, 40, 100])
def test_a_large_value_without_weight(T, Hq, Hkv, at, power):
    """One token's values 2^power of the others', which nobody attends to: those after it and before it keep their bits."""
    g = gen(at + T + power)
    D, n = 128, 900
    q, k, v = normal(g, T, Hq, D), normal(g, n, Hkv, D), normal(g, n, Hkv, D)
    q[..., 3], k[..., 3], v[at] = 8.0, 0.5, v[at] * 2.0 ** power
    k[at, :, 3] = -(power + 40) * math.log(2) * math.sqrt(D) / 8.0       # a weight of some 2^-(power + 40)
    if at > n - T:                                                       # a drafted token that the first ones do not see
        k[at, :, 3] *= 1.5
    c = case(q, k, v, 1 / math.sqrt(D))
    telling(c, *check(c))


@pytest.mark.parametrize("T,Hq,Hkv", ROWS)
@pytest.mark.parametrize("at", [0, 450, 850])
@pytest.mark.parametrize("power", [6, 14, 30, 60])
def test_rows_that_disagree_on_a_large_value(T, Hq, Hkv, at, power):
    """Half of the heads attend to the token with the large values, the others not at all: each row its own bits."""
    g = gen(at + T + power + 7)
    D, n = 128, 900
    q, k, v = normal(g, T, Hq, D), normal(g, n, Hkv, D), normal(g, n, Hkv, D)
    v[at:at + 2] *= 2.0 ** power
    k[..., 3], k[at:at + 2, :, 3] = 0.0, (power + 40) * math.log(2) * math.sqrt(D) / 8.0
    q[:, ::2, 3], q[:, 1::2, 3] = 8.0, -8.0
    c = case(q, k, v, 1 / math.sqrt(D))
    want, tol = check(c)
    telling((c[0][:, :, 1::2], *c[1:]) if Hq // Hkv % 2 == 0 else c, *((want[:, :, 1::2], tol[:, :, 1::2]) if
                                                                     Hq // Hkv % 2 == 0 else (want, tol)))


@pytest.mark.parametrize("T,Hq,Hkv", ROWS)
@pytest.mark.parametrize("n", [128, 1000])
@pytest.mark.parametrize("rise,fall", [(20, 18), (60, 40), (60, 50), (-60, -40), (5, 30)])
def test_values_that_fall_while_scores_rise(T, Hq, Hkv, n, rise, fall):
    """Scores that rise by 2^rise in steps while the values fall by 2^fall, and the other way round: references and
    scalings change again and again, together and against each other."""
    g = gen(n + T + rise)
    D = 128
    q, k, v = normal(g, T, Hq, D), normal(g, n, Hkv, D), normal(g, n, Hkv, D)
    step = (torch.arange(n, device=DEV) * 8 // n).double() / 7
    q[..., 3] = 8.0
    k[..., 3] = ((step - 0.5) * rise * math.log(2) * math.sqrt(D) / 8.0)[:, None].float()
    v *= torch.exp2((0.5 - step) * fall)[:, None, None].float()
    c = case(q, k, v, 1 / math.sqrt(D))
    telling(c, *check(c))
    check(c, window=n // 3)


@pytest.mark.parametrize("T,Hq,Hkv", ROWS)
def test_values_towards_the_ends_of_bf16(T, Hq, Hkv):
    """Groups of 1e32 and of 1e-34, and tokens of 1e30 and 1e-30 in one group.  (A group of +-3e38 spans more than fp32
    holds and reads back as NaN, and sums of 200 weights of up to 2^6 times a value of 3e34 or more leave fp32.)"""
    g = gen(T)
    D, n = 256, 200
    v = normal(g, n, Hkv, D).clamp(-3, 3)
    v[..., :64] *= 1e32
    v[..., 64:128] *= 1e-34
    v[::2, :, 128:192] *= 1e30
    v[1::2, :, 128:192] *= 1e-30
    c = case(normal(g, T, Hq, D), normal(g, n, Hkv, D), v, 1 / math.sqrt(D))
    telling(c, *check(c), groups=slice(0, 2))


@pytest.mark.parametrize("T,Hq,Hkv", ROWS)
def test_groups_without_a_spread(T, Hq, Hkv):
    """Constant values for a while in one group, throughout in the other (scale 0), then ordinary and tiny ones."""
    g = gen(T + 1)
    D, n = 128, 640
    v = normal(g, n, Hkv, D)
    v[..., 64:] = 0.75
    v[:300, :, :64] = -0.25
    v[400:, :, :64] *= 2.0 ** -20
    check(case(normal(g, T, Hq, D), normal(g, n, Hkv, D), v, 1 / math.sqrt(D)))


# ------------------------------------------------------------------ the largest counts that are accepted
@pytest.mark.parametrize("T,Hq,Hkv,n", [(1024, 4, 2, 1024), (1024, 2, 1, 40), (1024, 3, 1, 1300), (1, 4096, 8, 100),
                                        (1, 4096, 4096, 50), (2, 4096, 1, 200), (49, 4, 4, 300), (50, 10, 2, 77)])
def test_many_query_rows(T, Hq, Hkv, n):
    """1,024 query tokens, 4,096 query heads, chunks of rows that do not divide evenly."""
    g = gen(T + Hq + n)
    D = 64
    check(case(normal(g, T, Hq, D), normal(g, n, Hkv, D), normal(g, n, Hkv, D), 1 / math.sqrt(D)))
    check(case(normal(g, T, Hq, D), normal(g, n, Hkv, D), normal(g, n, Hkv, D), 1 / math.sqrt(D)), window=30)


def test_more_query_rows_are_refused():
    z = torch.zeros(1, 1025, 1, 64, dtype=BF, device=DEV)
    pool, table, n = kv4_pool(1, 16, 1, 1, 64), torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(
        1, dtype=torch.int32, device=DEV)
    for q in (z, z[:, :1].expand(1, 1, 4097, 64)):
        with pytest.raises(RuntimeError):
            ops.paged_attention_decode_kv4(q, pool, 0, table, n, 1.0)
