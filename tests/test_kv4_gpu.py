"""The 4-bit KV cache on the GPU: writing, reading and attention against plain implementations in 64 bits."""
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


@pytest.fixture(autouse=True)
def _status_clean():
    N.device_status(clear=True)
    yield
    assert N.device_status(clear=True) == 0, "a kernel reported a device-side error"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV).to(BF)


# ----------------------------------------------------------------------- write / read
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("tokens,heads,bs", [(1, 1, 16), (7, 3, 16), (33, 8, 32), (130, 5, 64), (1000, 2, 16)])
def test_written_bytes_and_values(D, tokens, heads, bs):
    """Every byte of the pool as the layout says, blocks that no slot names untouched; reading gives the
    stored values, correctly rounded."""
    g = gen(tokens * D + heads)
    P = (tokens + bs - 1) // bs + 2
    slots = torch.randperm(P * bs, generator=g, device=DEV)[:tokens]
    k, v = normal(g, tokens, heads, D), normal(g, tokens, heads, D) * 3 + 1
    pool = torch.randint(0, 256, (2, P, heads, bs // 16, 18 * D), generator=g, device=DEV, dtype=torch.uint8)
    # a byte holds two codes of one token, so untouched tokens keep theirs whole
    want = pool.cpu().clone()
    n = min(tokens, 40)                       # the byte-by-byte reference is slow
    ref.pack(want, 1, k[:n].cpu(), v[:n].cpu(), slots[:n].tolist(), bs)
    ops.kv4_write(k[:n], v[:n], pool, 1, slots[:n])
    assert torch.equal(pool.cpu(), want)
    ops.kv4_write(k, v, pool, 1, slots)
    gk, gv = ops.kv4_read(pool, 1, slots)
    for x, got in ((k, gk), (v, gv)):
        exact = ref.stored(x.cpu())
        assert torch.equal(got.cpu(), exact.float().to(BF))


def test_write_odd_strides_and_views():
    """K and V as columns of a fused projection (16-byte aligned or not), transposed, and expanded."""
    g = gen(5)
    pool = kv4_pool(4, 16, 1, 2, 128)
    slots = torch.arange(3, 40, device=DEV)
    fused = normal(g, 37, 1030)
    for lo in (0, 8, 3):                       # offset 3 is not 16-byte aligned
        k = fused[:, lo:lo + 256].unflatten(1, (2, 128))
        v = fused[:, 512 + lo:768 + lo].unflatten(1, (2, 128))
        ops.kv4_write(k, v, pool, 0, slots)
        gk, gv = ops.kv4_read(pool, 0, slots)
        assert torch.equal(gk.cpu(), ref.stored(k.cpu()).float().to(BF))
        assert torch.equal(gv.cpu(), ref.stored(v.cpu()).float().to(BF))
    t = normal(g, 2, 37, 128).transpose(0, 1)
    e = normal(g, 37, 1, 128).expand(37, 2, 128)
    ops.kv4_write(t, e, pool, 0, slots.repeat_interleave(2)[::2])
    gk, gv = ops.kv4_read(pool, 0, slots)
    assert torch.equal(gk.cpu(), ref.stored(t.cpu()).float().to(BF))
    assert torch.equal(gv.cpu(), ref.stored(e.cpu()).float().to(BF))


def test_write_dense_rows_under_any_stride():
    """A dimension of one may have any stride: one token out of a wide row, one head of an odd pitch."""
    g = gen(6)
    slots = torch.tensor([17, 5], device=DEV)
    for tokens, heads in ((1, 2), (1, 1), (2, 1)):
        base = normal(g, 4 * 128)
        sizes, dense = (tokens, heads, 128), (heads * 128, 128)
        strides = [s if n > 1 else 257 for n, s in zip(sizes, dense)] + [1]
        k, v = base.as_strided(sizes, strides), base.as_strided(sizes, strides, 256)
        assert k.is_contiguous() and 257 in k.stride()
        pool = kv4_pool(2, 16, 1, heads, 128)
        ops.kv4_write(k, v, pool, 0, slots[:tokens])
        gk, gv = ops.kv4_read(pool, 0, slots[:tokens])
        assert torch.equal(gk.cpu(), ref.stored(k.cpu()).float().to(BF))
        assert torch.equal(gv.cpu(), ref.stored(v.cpu()).float().to(BF))


@pytest.mark.parametrize("tokens,heads,D", [(8300, 8, 64), (4100, 8, 128), (2049, 12, 256), (8200, 6, 64), (4100, 5, 128),
                                            (2500, 12, 128)])
def test_long_writes_and_reads_are_those_of_short_ones(tokens, heads, D):
    """A lane takes up to four heads of a long call: the same bytes and values as token by token runs of a few."""
    g = gen(tokens + heads)
    k, v = normal(g, tokens, heads, D), normal(g, tokens, heads, D) * 5 - 2
    k[5:40:7] = 3.0                                   # groups of one value
    v[6:60:9, 1] *= 1e-38                             # subnormal scales
    k[100, 2, 7], v[101, 3, 60], k[102, 0, 0] = float("nan"), float("inf"), float("-inf")
    k[103, 1, :2] = torch.tensor([3e38, -3e38], device=DEV).to(BF)
    bs = 32
    pools = [kv4_pool(tokens // bs + 2, bs, 2, heads, D) for _ in range(2)]
    slots = torch.randperm(pools[0].shape[1] * bs, generator=g, device=DEV)[:tokens]
    slots[50:60] = -1
    ops.kv4_write(k, v, pools[0], 1, slots)
    for i in range(0, tokens, 200):
        ops.kv4_write(k[i:i + 200], v[i:i + 200], pools[1], 1, slots[i:i + 200])
    assert torch.equal(pools[0], pools[1])
    gk, gv = ops.kv4_read(pools[0], 1, slots)
    for i in range(0, tokens, 200):
        pk, pv = ops.kv4_read(pools[0], 1, slots[i:i + 200])
        assert torch.equal(gk[i:i + 200].view(torch.int16), pk.view(torch.int16))
        assert torch.equal(gv[i:i + 200].view(torch.int16), pv.view(torch.int16))
    live = slots >= 0
    for x, got in ((k, gk), (v, gv)):
        assert torch.equal(got[:200][live[:200]].cpu().isnan(), ref.stored(x[:200][live[:200]].cpu()).isnan())
        some = torch.arange(104, 200, device=DEV)
        assert torch.equal(got[some].cpu(), ref.stored(x[some].cpu()).float().to(BF))


def test_write_extreme_values():
    """Constant groups, ties between two codes, tiny and huge values, and NaN and infinity in one group only."""
    pool = kv4_pool(2, 16, 1, 1, 128)
    x = torch.zeros(10, 1, 128, device=DEV)
    x[0] = 3.25                                                     # one value: scale 0
    x[1, 0, :64] = torch.arange(64, device=DEV) * 0.25             # ties: 15 steps of 1.0625
    x[1, 0, 64:] = torch.arange(64, device=DEV) % 31 * 0.5          # steps of 1, every other value halfway
    x[2] = torch.linspace(-1e-38, 1e-38, 128, device=DEV)
    x[3] = torch.linspace(-1e38, 1e38, 128, device=DEV)
    x[4] = 1.0
    x[4, 0, 5] = float("nan")
    x[5] = 2.0
    x[5, 0, 70] = float("inf")
    x[6] = -2.0
    x[6, 0, 1] = -float("inf")
    x[7] = torch.linspace(-3.3e38, 3.3e38, 128, device=DEV)        # past fp32's range between: not finite
    x[9] = torch.linspace(-3.3e38, 3.3e38, 128, device=DEV, dtype=torch.float64)   # each group spans less than fp32 holds
    x[8, 0, :64] = torch.where(torch.arange(64, device=DEV) % 2 == 0, 3.3e38, -3.3e38)   # this one more
    x = x.to(BF)
    slots = torch.arange(10, device=DEV)
    ops.kv4_write(x, x.flip(0), pool, 0, slots)
    k, v = ops.kv4_read(pool, 0, slots)
    assert torch.equal(k[:4].cpu(), ref.stored(x[:4].cpu()).float().to(BF))
    assert bool(k[7].isnan().all()) and not bool(x[7].isfinite().all())
    assert bool(k[9].isfinite().all()) and torch.equal(k[9].cpu(), ref.stored(x[9:10].cpu())[0].float().to(BF))
    for t, bad in ((4, 0), (5, 1), (6, 0), (8, 0)):
        group = slice(64 * bad, 64 * bad + 64)
        other = slice(64 - 64 * bad, 128 - 64 * bad)
        assert bool(k[t, 0, group].isnan().all()) and torch.equal(k[t, 0, other], x[t, 0, other])
    assert torch.equal(k.flip(0).nan_to_num(), v.nan_to_num())


def test_slots_outside_the_pool():
    """Negative slots are skipped and read as zeros; slots past the pool too, and are reported."""
    g = gen(8)
    pool = kv4_pool(3, 16, 2, 1, 64)
    k, v = normal(g, 5, 1, 64), normal(g, 5, 1, 64)
    slots = torch.tensor([0, -1, 47, -(1 << 40), 20], device=DEV)
    ops.kv4_write(k, v, pool, 0, slots)
    assert not bool(pool[1].any())
    gk, gv = ops.kv4_read(pool, 0, slots)
    assert not bool(gk[[1, 3]].any()) and not bool(gv[[1, 3]].any())
    assert torch.equal(gk[[0, 2, 4]].cpu(), ref.stored(k[[0, 2, 4]].cpu()).float().to(BF))
    before = pool.clone()
    for slot in (48, 1 << 33, (1 << 62) + 5):
        ops.kv4_write(k[:1], v[:1], pool, 1, torch.tensor([slot], device=DEV))
        assert N.device_status(clear=True) == N.DEV_BAD_BLOCK
        assert not bool(ops.kv4_read(pool, 1, torch.tensor([slot], device=DEV))[0].any())
        assert N.device_status(clear=True) == N.DEV_BAD_BLOCK
    assert torch.equal(pool, before)
    ops.kv4_write(k[:0], v[:0], pool, 0, slots[:0])
    assert ops.kv4_read(pool, 0, slots[:0])[0].shape == (0, 1, 64)


# -------------------------------------------------------------------------- attention
def attend_case(seed, lens, T, Hq, Hkv, D, bs=16, spare=2, wide=0, qscale=1.0, unused=255):
    """A pool of quantised keys and values whose unused tokens hold NaN pairs (bytes of 255; 127: pairs of
    3.4e38), and shuffled tables whose unused entries are invalid."""
    g = gen(seed)
    held = [(n + bs - 1) // bs for n in lens]
    P = sum(held) + spare
    order = torch.randperm(P, generator=g, device=DEV)
    pool = torch.full((2, P, Hkv, bs // 16, 18 * D), unused, dtype=torch.uint8, device=DEV)
    mb = max(held + [1]) + wide
    table = torch.full((len(lens), mb), -7, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(lens):
        blocks = order[at:at + held[b]]
        at += held[b]
        table[b, :held[b]] = blocks.int()
        if n:
            pos = torch.arange(n, device=DEV)
            slots = blocks[pos // bs] * bs + pos % bs
            ops.kv4_write(normal(g, n, Hkv, D) * 1.5, normal(g, n, Hkv, D) + 0.5, pool, 1, slots)
    q = (torch.randn(len(lens), T, Hq, D, generator=g, device=DEV) * qscale).to(BF)
    return dict(q=q, pool=pool, table=table, ctx=torch.tensor(lens, dtype=torch.int32, device=DEV),
                scale=1 / math.sqrt(D))


def check(c, got, **kw):
    want, tol = ref.attention(c["q"], c["pool"], 1, c["table"], c["ctx"], c["scale"], **kw)
    got = got.reshape(want.shape)
    assert bool(got.isfinite().all())
    over = (got.double() - want).abs() - tol
    assert float(over.max()) <= 0, (float(over.max()), float((got.double() - want).abs().max()))


def attend(c, **kw):
    return ops.paged_attention_decode_kv4(c["q"], c["pool"], 1, c["table"], c["ctx"], c["scale"], **kw)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (32, 8), (3, 1), (35, 5), (16, 1), (40, 2)])
def test_attention_head_layouts(D, Hq, Hkv):
    c = attend_case(Hq * D + Hkv, [1, 17, 130, 700], 1, Hq, Hkv, D)
    check(c, attend(c))


@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [127], [128], [129], [255], [256], [257], [2048], [5000],
                                  [1, 4097], [3000, 1, 2, 700, 64]])
@pytest.mark.parametrize("bs", [16, 64])
def test_attention_lengths(lens, bs):
    c = attend_case(sum(lens) + bs, lens, 1, 8, 2, 128, bs=bs, wide=3)
    check(c, attend(c))


@pytest.mark.parametrize("unused", [0, 127, 128, 255])
def test_attention_unused_tokens_hold_anything(unused):
    """The tokens behind a sequence in its last page and before its window: zeros, NaN, the largest and lowest pairs."""
    c = attend_case(40 + unused, [5, 20, 300, 1000], 1, 8, 2, 128, bs=64, unused=unused)
    check(c, attend(c))
    c = attend_case(41 + unused, [5, 20, 300, 1000], 3, 8, 2, 128, bs=64, unused=unused)
    check(c, attend(c))
    slot = int(c["table"][3, 0]) * 64
    c["pool"][1, slot // 64] = unused                     # the first block lies before the window
    check(c, attend(c, window=900), window=900)


@pytest.mark.parametrize("T", [1, 2, 3, 5, 8, 16, 33])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 128), (32, 8, 128), (12, 2, 64), (8, 4, 256)])
def test_attention_several_query_tokens(T, Hq, Hkv, D):
    """Drafted tokens: query i sees the keys up to itself; sequences shorter than the queries leave some
    without any key."""
    c = attend_case(T * D + Hq, [T, T + 15, 300, 1, max(T - 1, 1), 1025], T, Hq, Hkv, D)
    out = attend(c)
    check(c, out)
    for b, n in enumerate(c["ctx"].tolist()):
        if n < T:
            assert not bool(out[b, :T - n].any())


@pytest.mark.parametrize("window", [1, 5, 16, 17, 100, 128, 129, 1000, 5000, 1 << 40])
@pytest.mark.parametrize("T,D", [(1, 128), (4, 128), (2, 256)])
def test_attention_window(window, T, D):
    c = attend_case(window % 1000 + T, [4, 40, 333, 1600], T, 8, 4, D, bs=32)
    check(c, attend(c, window=window), window=window)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("cap", [5.0, 50.0])
def test_attention_softcap(D, cap):
    c = attend_case(int(cap) + D, [1, 90, 1300], 2, 8, 4, D, qscale=4.0)
    check(c, attend(c, softcap=cap), softcap=cap)
    check(c, attend(c, softcap=cap, window=77), softcap=cap, window=77)


def test_attention_empty_sequences_and_padding():
    """A length of zero gives zeros, whatever its table row says; three- and four-dimensional q agree."""
    c = attend_case(3, [0, 33, 0], 1, 8, 2, 128)
    out = attend(c)
    check(c, out)
    assert not bool(out[0].any()) and not bool(out[2].any())
    flat = ops.paged_attention_decode_kv4(c["q"][:, 0], c["pool"], 1, c["table"], c["ctx"], c["scale"])
    assert torch.equal(flat, out[:, 0])
    dst = torch.full_like(out, 7.0)
    assert attend(c, out=dst) is dst and torch.equal(dst, out)
    assert attend(dict(c, q=c["q"][:0], table=c["table"][:0], ctx=c["ctx"][:0])).shape == (0, 1, 8, 128)


def test_attention_large_and_small_scores():
    """Scores of one token far above the others, queries of any magnitude, keys and values tiny or huge."""
    c = attend_case(21, [700], 2, 8, 2, 128, qscale=40.0)
    check(c, attend(c))
    for f in (2.0 ** -60, 2.0 ** 60):
        g = gen(31)
        n = 300
        pool = kv4_pool(32, 16, 2, 2, 128)
        slots = torch.arange(n, device=DEV)
        ops.kv4_write((normal(g, n, 2, 128).float() * f).to(BF), (normal(g, n, 2, 128).float() * f).to(BF), pool, 1, slots)
        c = dict(q=(normal(g, 1, 1, 8, 128).float() / f).to(BF), pool=pool,
                 table=torch.arange(32, dtype=torch.int32, device=DEV)[None],
                 ctx=torch.tensor([n], dtype=torch.int32, device=DEV), scale=0.09)
        check(c, attend(c))


def test_attention_values_of_mixed_magnitude():
    """Value scales that differ by powers of two between tokens, the largest late, early or masked by the window."""
    g = gen(77)
    n = 900
    pool = kv4_pool(64, 16, 2, 2, 128)
    slots = torch.arange(n, device=DEV)
    for at in (0, 450, 899):
        mag = torch.ones(n, 1, 1, device=DEV)
        mag[at] = 1e6
        ops.kv4_write(normal(g, n, 2, 128), (normal(g, n, 2, 128).float() * mag).to(BF), pool, 1, slots)
        c = dict(q=normal(g, 1, 1, 8, 128), pool=pool, table=torch.arange(64, dtype=torch.int32, device=DEV)[None],
                 ctx=torch.tensor([n], dtype=torch.int32, device=DEV), scale=0.09)
        check(c, attend(c))
        if at < 700:
            check(c, attend(c, window=200), window=200)


@pytest.mark.parametrize("later", [1.0, 1e-6, 1e6])
@pytest.mark.parametrize("T,Hq,Hkv,D", [(1, 8, 2, 128), (1, 16, 2, 256), (5, 8, 2, 128)])
def test_attention_constant_values_first(later, T, Hq, Hkv, D):
    """Values without a spread (scale 0) for a while, then ordinary, tiny or large ones, and scores that rise late, so
    that the references and the scaling of the weights change after sums have begun."""
    g = gen(int(math.log10(later)) + 50 + D)
    n = 640
    pool = kv4_pool(40, 16, 2, Hkv, D)
    slots = torch.arange(n, device=DEV)
    k, v = normal(g, n, Hkv, D), normal(g, n, Hkv, D).float() * later
    v[:100] = 0.25
    v[300:310] *= 1e-3
    q = normal(g, 1, T, Hq, D)
    # keys along the first query head's direction, ever longer
    d = q[0, 0].view(Hkv, Hq // Hkv, D)[:, 0].float()
    k = (k.float() * 0.3 + torch.arange(n, device=DEV)[:, None, None] / n * 3 * d / d.norm(dim=-1, keepdim=True)).to(BF)
    ops.kv4_write(k, v.to(BF), pool, 1, slots)
    c = dict(q=q, pool=pool, table=torch.arange(40, dtype=torch.int32, device=DEV)[None],
             ctx=torch.tensor([n], dtype=torch.int32, device=DEV), scale=2 / math.sqrt(D))
    check(c, attend(c))
    # one worker's 128 tokens: constant values up to 32, scores some 20 powers of two higher from 112 on
    v[:32], v[32:128] = 0.25, normal(g, 96, Hkv, D).float() * later
    k[:112], k[112:128] = k[:112] * 0.1, (4 * d / d.norm(dim=-1, keepdim=True) + 0.1 * k[112:128].float()).to(BF)
    ops.kv4_write(k, v.to(BF), pool, 1, slots)
    c = dict(c, ctx=torch.tensor([128], dtype=torch.int32, device=DEV), table=c["table"][:, :8])
    check(c, attend(c))


def test_attention_nan_value_stays_with_those_that_see_it():
    """A drafted token whose V is NaN reaches the queries that see it and no other."""
    c = attend_case(9, [200, 200], 3, 8, 2, 128)
    slot = int(c["table"][0, 199 // 16]) * 16 + 199 % 16
    bad = torch.full((1, 2, 128), float("nan"), dtype=BF, device=DEV)
    ops.kv4_write(bad, bad, c["pool"], 1, torch.tensor([slot], device=DEV))
    out = attend(c)
    assert bool(out[0, 2].isnan().all()) and bool(out[0, :2].isfinite().all()) and bool(out[1].isfinite().all())
    want, tol = ref.attention(c["q"][:, :2], c["pool"], 1, c["table"], c["ctx"] - 1, c["scale"])
    assert float(((out[:, :2].double() - want).abs() - tol).max()) <= 0


def test_attention_bad_blocks_and_lengths_are_reported():
    """A block outside the pool counts as masked and a context past its table is cut; both are reported."""
    c = attend_case(10, [100, 60], 1, 8, 2, 128)
    good = attend(c)
    for bad in (-1, c["pool"].shape[1], 2 ** 31 - 1, -2 ** 31):
        t = c["table"].clone()
        t[0, 2] = bad
        out = attend(dict(c, table=t))
        assert N.device_status(clear=True) == N.DEV_BAD_BLOCK
        assert torch.equal(out[1], good[1]) and bool(out.isfinite().all())
        keep = [i for i in range(100) if i // 16 != 2]
        k, v = ref.unpack(c["pool"], 1, c["table"][0, :7].long())
        z = torch.einsum("hrd,nhd->hrn", c["q"][0, 0].double().unflatten(0, (2, 4)), k[keep]) * c["scale"]
        want = torch.einsum("hrn,nhd->hrd", z.softmax(-1), v[keep]).flatten(0, 1)
        assert float((out[0, 0].double() - want).abs().max()) < 2.0 ** -7
    cut = attend(dict(c, ctx=torch.tensor([113, -3], dtype=torch.int32, device=DEV), table=c["table"][:, :3]))
    assert N.device_status(clear=True) == N.DEV_BAD_POSITION
    assert torch.equal(cut[1], torch.zeros_like(cut[1]))
    short = attend(dict(c, ctx=torch.tensor([48, 0], dtype=torch.int32, device=DEV)))
    assert torch.equal(cut[0], short[0])


def test_attention_strides_and_table_views():
    """q as columns of a fused projection, a table that is a slice of a wider one, a table in column order."""
    c = attend_case(12, [300, 20, 77], 2, 8, 2, 128, wide=5)
    want = attend(c)
    wide = torch.zeros(3, 2, 8 * 128 + 64, dtype=BF, device=DEV)
    for lo in (0, 8, 5):
        view = wide[..., lo:lo + 1024]
        view.copy_(c["q"].flatten(2))
        assert torch.equal(attend(dict(c, q=view.unflatten(2, (8, 128)))), want)
    need = 300 // 16 + 1
    assert torch.equal(attend(dict(c, table=c["table"][:, :need])), want)
    assert torch.equal(attend(dict(c, table=c["table"].t().contiguous().t())), want)
    one = attend(dict(c, q=c["q"][:1], table=c["table"][:1], ctx=c["ctx"][:1]))
    check(dict(c, q=c["q"][:1], table=c["table"][:1], ctx=c["ctx"][:1]), one)


@pytest.mark.parametrize("batch,D,T", [(700, 64, 1), (1500, 128, 1), (33, 128, 1), (32, 128, 5), (257, 256, 2)])
def test_attention_many_sequences(batch, D, T):
    """More sequences than lanes, than warps; all short, and with a few long ones among them."""
    lens = [(37 * i) % 190 for i in range(batch)]
    c = attend_case(batch, lens, T, 4, 2, D)
    check(c, attend(c))
    for i in (0, batch // 2, batch - 1):
        lens[i] = 3000 + i
    c = attend_case(batch + 1, lens, T, 4, 2, D)
    check(c, attend(c))


@pytest.mark.parametrize("lens", [[128] * 40, [100, 7, 128, 1, 0]])
def test_attention_short_tables(lens):
    """Tables of at most 128 tokens, whose items are not split; the same sequences under a wider table."""
    for T, Hq, Hkv, D in ((1, 32, 8, 128), (3, 8, 4, 256), (2, 6, 6, 64), (9, 8, 2, 128)):
        c = attend_case(len(lens) + T, lens, T, Hq, Hkv, D, bs=32)
        out = attend(c)
        check(c, out)
        wide = torch.cat([c["table"], torch.full_like(c["table"], -1)], 1)
        check(c, attend(dict(c, table=wide)))


def test_attention_sequences_that_share_blocks():
    """A common prefix held once: the same blocks in several tables, and twice in one."""
    c = attend_case(23, [700, 700, 700], 1, 8, 2, 128)
    c["table"][1, :20] = c["table"][0, :20]
    c["table"][2, 30:40] = c["table"][2, :10]
    check(c, attend(c))


def test_attention_is_deterministic_and_stream_safe():
    """The same bits on every call, from two streams at once, and from two captured graphs replayed together."""
    c = attend_case(15, [3000, 2000, 1, 900], 1, 32, 8, 128)
    d = attend_case(16, [10, 4000], 3, 8, 2, 128)
    want_c, want_d = attend(c), attend(d)
    for _ in range(3):
        assert torch.equal(attend(c), want_c)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s, x in zip(streams, (c, d)):
            with torch.cuda.stream(s):
                outs.append(attend(x))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, [want_c, want_d] * 10))
    graphs, held = [], []
    for x in (c, d):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(attend(x))
        graphs.append(g)
    for _ in range(5):
        for o in held:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], want_c) and torch.equal(held[1], want_d)


def test_attention_workspace_argument():
    c = attend_case(17, [3000], 1, 32, 8, 128)
    need = N.lib().mvb_paged_attention_decode_kv4_workspace_bytes(1, 1, 32, 8, 128, 0)
    ws = torch.randint(0, 256, (max(need, 1),), dtype=torch.uint8, device=DEV)
    assert torch.equal(attend(c, workspace=ws), attend(c))
    for bad in (ws[:-1], ws[1:], ws[:0], ws[::2], ws.int()):
        with pytest.raises(RuntimeError):
            attend(c, workspace=bad)
    short = attend_case(18, [3, 128], 1, 32, 8, 128)            # at most 128 tokens: none is needed
    assert torch.equal(attend(short, workspace=ws[:0]), attend(short))


def test_attention_under_programmatic_launch():
    """With programmatic dependent launch on, as the engine runs its steps: write, then attend, many times."""
    c = attend_case(18, [500, 40], 1, 8, 2, 128)
    want = attend(c)
    slots = torch.tensor([int(c["table"][0, 3]) * 16 + 5], device=DEV)
    k, v = ops.kv4_read(c["pool"], 1, slots)
    old = N.set_pdl(True)
    try:
        outs = []
        for i in range(20):
            x = (k.float() + i).to(BF)
            ops.kv4_write(x, x, c["pool"], 1, slots)
            outs.append(attend(c))
            ops.kv4_write(k, v, c["pool"], 1, slots)
            outs.append(attend(c))
        torch.cuda.synchronize()
    finally:
        N.set_pdl(old)
    last = outs[1]
    assert all(torch.equal(o, last) for o in outs[1::2])
    for i in (0, 7, 19):
        x = (k.float() + i).to(BF)
        ops.kv4_write(x, x, c["pool"], 1, slots)
        assert torch.equal(attend(c), outs[2 * i])
    assert torch.equal(want[1], last[1])


def test_long_cache_offsets_pass_32_bits():
    """A pool of more than 4 GiB: blocks at both ends of it."""
    D, H, bs = 128, 8, 16
    P = (1 << 32) // (H * 18 * D) + 200
    pool = torch.zeros(1, P, H, 1, 18 * D, dtype=torch.uint8, device=DEV)
    g = gen(19)
    blocks = torch.tensor([P - 1, 0, P - 2, P // 2], device=DEV)
    pos = torch.arange(64, device=DEV)
    slots = blocks[pos // bs] * bs + pos % bs
    k, v = normal(g, 64, H, D), normal(g, 64, H, D)
    ops.kv4_write(k, v, pool, 0, slots)
    gk, _ = ops.kv4_read(pool, 0, slots)
    assert torch.equal(gk.cpu(), ref.stored(k.cpu()).float().to(BF))
    q = normal(g, 1, 1, 16, D)
    got = ops.paged_attention_decode_kv4(q, pool, 0, blocks.int()[None], torch.tensor([64], dtype=torch.int32, device=DEV),
                                         0.09)
    want, tol = ref.attention(q, pool, 0, blocks.int()[None], torch.tensor([64]), 0.09)
    assert float(((got.double() - want).abs() - tol).max()) <= 0


def test_wrong_arguments_are_refused():
    c = attend_case(20, [40], 1, 8, 2, 128)
    bad = [dict(c, q=c["q"].half()), dict(c, q=c["q"][..., :64]), dict(c, q=c["q"][:, :, :5]), dict(c, ctx=c["ctx"].long()),
           dict(c, table=c["table"].long()), dict(c, table=c["table"].repeat(2, 1)), dict(c, pool=c["pool"].view(torch.int8)),
           dict(c, pool=c["pool"][..., :-18 * 64]), dict(c, ctx=c["ctx"].cpu()), dict(c, pool=c["pool"][0])]
    for x in bad:
        with pytest.raises(RuntimeError):
            attend(x)
    for kw in (dict(window=-1), dict(softcap=-1.0), dict(out=c["q"][0]), dict(out=c["q"].float())):
        with pytest.raises(RuntimeError):
            attend(c, **kw)
    with pytest.raises(RuntimeError):
        ops.paged_attention_decode_kv4(c["q"], c["pool"], 2, c["table"], c["ctx"], 1.0)
    x, s = torch.zeros(3, 2, 128, dtype=BF, device=DEV), torch.arange(3, device=DEV)
    for k, v, sl, layer in ((x[:2], x, s, 0), (x, x[:, :1], s, 0), (x.float(), x, s, 0), (x, x, s.int(), 0), (x, x, s, 2),
                            (x, x, s[None], 0), (x, x, s.cpu(), 0)):
        with pytest.raises(RuntimeError):
            ops.kv4_write(k, v, c["pool"], layer, sl)


def test_torch_ops_namespace():
    from llm_pytorch_inference_b200 import torch_ops  # noqa: F401
    c = attend_case(22, [40, 7], 1, 8, 2, 128)
    slots = torch.tensor([0, 5], device=DEV)
    m = torch.ops.mini_vllm_ops
    k, v = m.kv4_read(c["pool"], 1, slots)
    m.kv4_write(k, v, c["pool"], 0, slots)
    got = m.paged_attention_decode_kv4(c["q"], c["pool"], 1, c["table"], c["ctx"], c["scale"], 0.0, 0)
    assert torch.equal(got, attend(c))
