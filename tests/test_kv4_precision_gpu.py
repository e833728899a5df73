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
