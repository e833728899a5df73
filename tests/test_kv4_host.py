"""The 4-bit KV cache, slot assignment and draft verification on the CPU: what the entry points refuse
before any launch, the pool's geometry, and the tests' own reference against its definition."""
import pytest
import torch

import kv4_reference as ref
from llm_pytorch_inference_b200 import _native as N
from llm_pytorch_inference_b200 import kv_cache, ops

A = 4096   # stands for an aligned device pointer: no call below gets as far as using one


def refused(rc, text):
    assert rc == 1 and text in N.lib().mvb_last_error().decode(), N.lib().mvb_last_error()


def test_pool_geometry():
    p = kv_cache.kv4_pool(5, 32, 2, 3, 128, device="cpu")
    assert p.shape == (2, 5, 3, 2, 18 * 128) and p.dtype == torch.uint8
    assert p[:, 0].numel() == kv_cache.kv4_block_bytes(32, 3, 128, 2)
    assert kv_cache.kv4_block_bytes(16, 8, 128, 36) * 32 == 9 * kv_cache.block_bytes(16, 8, 128, 36, 2)
    for bad in [(5, 24, 2, 3, 128), (5, 0, 2, 3, 128), (5, 16, 2, 3, 96), (0, 16, 2, 3, 128), (5, 16, 0, 3, 128)]:
        with pytest.raises(ValueError):
            kv_cache.kv4_pool(*bad, device="cpu")


@pytest.mark.parametrize("change, text", [
    (dict(kv4=None), "null pointer"), (dict(k=None), "null pointer"), (dict(slots=None), "null pointer"),
    (dict(kv4=A + 8), "16-byte aligned"), (dict(k=A + 2), "16-byte aligned"), (dict(ks=1028), "16-byte aligned"),
    (dict(hs=130), "16-byte aligned"), (dict(D=96), "head_dim 96"), (dict(H=0), "0 KV heads"),
    (dict(layer=2), "layer 2 of 2"), (dict(layer=-1), "layer -1"), (dict(bs=24), "block_size 24"),
    (dict(bs=0), "block_size 0"), (dict(P=0), "0 blocks"), (dict(P=1 << 40), "blocks"), (dict(n=-1), "-1 tokens"),
    (dict(n=1 << 40), "tokens"),
])
def test_kv4_write_and_read_refuse(change, text):
    a = dict(kv4=A, k=A, ks=1024, hs=128, slots=A, n=4, H=8, D=128, L=2, layer=1, P=7, bs=16)
    a.update(change)
    tail = (a["slots"], a["n"], a["H"], a["D"], a["L"], a["layer"], a["P"], a["bs"], None)
    refused(N.lib().mvb_kv4_write(a["kv4"], a["k"], a["ks"], a["hs"], a["k"], a["ks"], a["hs"], *tail), text)
    if not {"ks", "hs"} & set(change):
        refused(N.lib().mvb_kv4_read(a["k"], a["k"], a["kv4"], *tail), text)


@pytest.mark.parametrize("change, text", [
    (dict(out=None), "null pointer"), (dict(q=None), "null pointer"), (dict(kv4=None), "null pointer"),
    (dict(bt=None), "null pointer"), (dict(ctx=None), "null pointer"), (dict(B=-1), "batch"),
    (dict(T=0), "0 query tokens"), (dict(T=1 << 20), "query tokens"), (dict(hq=33), "33 query heads"),
    (dict(hkv=0), "query heads"), (dict(D=80), "head_dim 80"), (dict(layer=5), "layer 5 of 2"),
    (dict(bs=8), "block_size 8"), (dict(P=0), "0 blocks"), (dict(mb=0), "0 blocks a sequence"),
    (dict(mb=1 << 40, ts=1 << 40), "blocks a sequence"), (dict(ts=3), "table_stride 3"),
    (dict(qs=4095), "16-byte aligned"), (dict(qs=4088), "rows at least a token apart"),
    (dict(os=2048), "rows at least a token apart"), (dict(q=A + 4), "16-byte aligned"),
    (dict(window=-1), "window"), (dict(cap=-1.0), "softcap"), (dict(scale=float("nan")), "scale"),
    (dict(cap=float("nan")), "softcap"), (dict(cap=float("inf")), "softcap"), (dict(scale=float("inf")), "scale"),
    (dict(cap=1e-40), "softcap"), (dict(B=65537), "batch 65537"), (dict(hq=8192, qs=1 << 20, os=1 << 20), "8192 query heads"),
])
def test_kv4_attention_refuses(change, text):
    a = dict(out=A, os=4096, q=A, qs=4096, kv4=A, bt=A, ts=9, mb=9, ctx=A, B=2, T=1, hq=32, hkv=8, D=128, L=2, layer=0,
             P=20, bs=16, scale=0.1, cap=0.0, window=0)
    a.update(change)
    refused(N.lib().mvb_paged_attention_decode_kv4(
        a["out"], a["os"], a["q"], a["qs"], a["kv4"], a["bt"], a["ts"], a["mb"], a["ctx"], a["B"], a["T"], a["hq"],
        a["hkv"], a["D"], a["L"], a["layer"], a["P"], a["bs"], a["scale"], a["cap"], a["window"], A, 1 << 40, None), text)


@pytest.mark.parametrize("change, text", [
    (dict(start=None), "null pointer"), (dict(granted=None), "null pointer"), (dict(ctx=None), "null pointer"),
    (dict(bt=None), "block_tables"), (dict(batch=1 << 21), "batch 2097152"), (dict(batch=-1), "batch -1"),
    (dict(ts=3), "table_stride 3"), (dict(free=None), "free list"), (dict(nf=-1), "free list"),
    (dict(bs=0), "block_size 0"), (dict(mb=1 << 30, ts=1 << 30), "blocks a sequence"), (dict(n=-1), "num_tokens"),
    (dict(slots=None), "num_tokens"), (dict(head=A + 4), "free_head_out may not be free_head"),
])
def test_assign_slots_refuses(change, text):
    a = dict(slots=A, pos=A, start=A, granted=A, head_out=A + 4, bt=A, ts=8, mb=8, ctx=A, new=A, free=A, nf=10,
             head=None, batch=3, bs=16, n=12, ws=None, ws_bytes=0)
    a.update(change)
    refused(N.lib().mvb_assign_slots(*a.values(), None), text)


@pytest.mark.parametrize("change, text", [
    (dict(granted=None), "null pointer"), (dict(bs=0), "block_size 0"), (dict(held=A + 64), "held_blocks"),
    (dict(held=A + 96), "held_blocks"),
])
def test_assign_slots_ex_refuses(change, text):
    a = dict(slots=A, pos=A, start=A, granted=A, head_out=A + 4, bt=A, ts=8, mb=8, ctx=A + 64, new=A + 96, held=A + 128,
             free=A, nf=10, head=None, batch=3, bs=16, n=12, ws=None, ws_bytes=0)
    a.update(change)
    refused(N.lib().mvb_assign_slots_ex(*a.values(), None), text)


def test_reference_slots_with_counts():
    """Where lengths only grow, counting the blocks changes nothing; after a step back they are used again."""
    a, b, held = [[-1] * 4], [[-1] * 4], [0]
    for n, add, head in ((0, 5, 0), (5, 4, 2), (9, 1, 3)):
        assert ref.assign(a, [n], [add], [7, 8, 9], 4, add, head) == ref.assign_held(b, [n], [add], held, [7, 8, 9], 4, add,
                                                                                     head)
    assert a == b == [[7, 8, 9, -1]] and held == [3]
    assert ref.assign_held(b, [3], [6], held, [7, 8, 9], 4, 6, 3)[::4] == ([31, 32, 33, 34, 35, 36], 3)


@pytest.mark.parametrize("change, text", [
    (dict(out=None), "null pointer"), (dict(p=None), "null pointer"), (dict(u=None), "null pointer"),
    (dict(tok=None), "null pointer"), (dict(ps=99), "rows of 99"), (dict(qs=99), "rows of 100 and 99"),
    (dict(batch=-1), "batch -1"), (dict(K=-1), "-1 drafts"), (dict(K=5000), "5000 drafts"), (dict(V=0), "vocab 0"),
    (dict(V=1 << 25, ps=1 << 25, qs=1 << 25), "vocab"),
])
def test_verify_drafts_refuses(change, text):
    a = dict(out=A, acc=A, p=A, ps=100, q=A, qs=100, tok=A, u=A, lens=None, batch=2, K=3, V=100)
    a.update(change)
    refused(N.lib().mvb_verify_drafts(*a.values(), None), text)


def test_cpu_tensors_are_refused():
    kv4 = kv_cache.kv4_pool(2, 16, 1, 1, 64, device="cpu")
    x, i32 = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    calls = [lambda: ops.kv4_write(x, x, kv4, 0, torch.zeros(1, dtype=torch.int64)),
             lambda: ops.kv4_read(kv4, 0, torch.zeros(1, dtype=torch.int64)),
             lambda: ops.paged_attention_decode_kv4(x, kv4, 0, i32[None], i32, 1.0),
             lambda: ops.assign_slots(i32[None], i32, i32, i32, 16, 1),
             lambda: ops.verify_drafts(torch.ones(1, 2, 4), torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 2))]
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_reference_pool_round_trip():
    """pack / unpack agree on the layout, and a stored value is within half a step of its input."""
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(5, 2, 128, generator=g).bfloat16() for _ in range(2))
    pool = kv_cache.kv4_pool(3, 32, 1, 2, 128, device="cpu")
    slots = [64, 3, 17, -1, 95]
    ref.pack(pool, 0, k, v, slots, 32)
    kk, vv = ref.unpack(pool, 0, torch.arange(3))
    for x, got in ((k, kk), (v, vv)):
        _, scale, _ = ref.quantise(x)
        for t, s in enumerate(slots):
            if s >= 0:
                assert torch.equal(got[s], ref.stored(x)[t])
                # half a step, and 15 steps fall short of the maximum by at most 15 roundings of the scale
                off = (got[s] - x[t].double()).abs().unflatten(-1, (-1, 64)).amax(-1)
                assert bool((off <= scale[t] * (0.5 + 15 * 2.0 ** -8)).all())


def test_reference_slots_follow_the_block_manager():
    mgr = kv_cache.KVCacheManager(12, 4, 1, 1, 8, allocate_pool=False, free_order=list(range(11, -1, -1)))
    tables = [[0] * 6 for _ in range(3)]
    got = ref.assign(tables, [0, 0, 0], [5, 8, 1], list(range(11, -1, -1)), 4, 14)
    for seq, n in enumerate([5, 8, 1]):
        blocks = mgr.allocate(seq, n)
        assert tables[seq][:len(blocks)] == blocks
    assert got[0][:5] == [b * 4 + o for b, o in (mgr.slot(0, i) for i in range(5))] and got[4] == 12 - mgr.num_free_blocks
