"""Slot assignment and draft verification on the GPU, and a speculative step of the 4-bit cache as a whole."""
import math
import random

import pytest
import torch

import kv4_reference as ref
from llm_pytorch_inference_b200 import _native as N
from llm_pytorch_inference_b200 import ops
from llm_pytorch_inference_b200.kv_cache import KVCacheManager, kv4_pool

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _status_clean():
    N.device_status(clear=True)
    yield
    assert N.device_status(clear=True) == 0, "a kernel reported a device-side error"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------ slots
def run_slots(tables, ctx, new, free, bs, n, head=None):
    t = i32(tables) if tables and tables[0] else torch.zeros(len(ctx), 0, dtype=torch.int32, device=DEV)
    plan = ops.assign_slots(t, i32(ctx), i32(new), i32(free), bs, n, free_head=None if head is None else i32([head]))
    want_t = [list(r) for r in tables]
    slots, pos, start, granted, taken = ref.assign(want_t, ctx, new, free, bs, n, head or 0)
    assert plan.slots.tolist() == slots
    assert plan.positions.tolist() == pos
    assert plan.seq_start.tolist() == start
    assert plan.granted.tolist() == granted
    assert plan.free_head.tolist() == [taken]
    if tables and tables[0]:
        assert t.tolist() == want_t
    return plan


@pytest.mark.parametrize("batch,most,bs", [(1, 1, 16), (1, 5000, 16), (3, 1, 16), (64, 1, 16), (65, 9, 4), (511, 3, 16),
                                           (512, 40, 32), (513, 40, 7), (1500, 100, 16), (8192, 2, 16), (2, 0, 16),
                                           (8193, 3, 16), (12288, 1, 4), (50001, 2, 16)])
def test_slots(batch, most, bs):
    """Ragged lengths, zero-token sequences, tables with room to spare, against the sequences one by one."""
    r = random.Random(batch * 1000 + most)
    ctx = [r.randint(0, 60) for _ in range(batch)]
    new = [r.randint(0, most) for _ in range(batch)]
    width = max(-(-(c + n) // bs) for c, n in zip(ctx, new)) + 2
    ids = list(range(batch * width + 50))
    r.shuffle(ids)
    tables = [[ids.pop() if i < -(-c // bs) else -3 for i in range(width)] for c in ctx]
    run_slots(tables, ctx, new, ids, bs, sum(new))
    run_slots(tables, ctx, new, ids, bs, sum(new) + 37)         # padding behind the last token
    run_slots(tables, ctx, new, ids, bs, sum(new), head=5)


@pytest.mark.parametrize("batch", [5119, 5120, 6100, 6111, 6120, 6143, 6144, 8191])
def test_slots_around_the_default_shared_memory(batch):
    """Lengths held in shared memory up to and past 48 KB, the kernel's own arrays beside them."""
    run_slots([[b, -1] for b in range(batch)], [b % 17 for b in range(batch)], [b % 3 for b in range(batch)],
              list(range(batch, 3 * batch)), 16, 3 * batch)


@pytest.mark.parametrize("seed", range(6))
def test_slots_that_do_not_fit(seed):
    """Short of blocks, of table entries, or of room in the outputs: refused one by one, later ones served."""
    r = random.Random(seed)
    batch, bs, width = 200, 8, 5
    ctx = [r.randint(0, 24) for _ in range(batch)]
    new = [r.randint(0, 30) for _ in range(batch)]
    tables = [[r.randint(0, 999) for _ in range(width)] for _ in range(batch)]
    for free in (0, 1, 40, 150, 1000):
        run_slots(tables, ctx, new, list(range(1000, 1000 + free)), bs, sum(new))
        run_slots(tables, ctx, new, list(range(1000, 1000 + free)), bs, sum(new) // 2)
        run_slots(tables, ctx, new, list(range(1000, 1000 + free)), bs, sum(new), head=free // 2)
    if seed < 2:                                                      # a batch cut into pieces
        batch = 9000 + 4000 * seed
        ctx, new = [r.randint(-1, 24) for _ in range(batch)], [r.randint(0, 12) for _ in range(batch)]
        tables = [[r.randint(0, 999) for _ in range(4)] for _ in range(batch)]
        for free in (0, 1, 700, 3000, 20000):
            run_slots(tables, ctx, new, list(range(1000, 1000 + free)), bs, sum(new), head=1)
            run_slots(tables, ctx, new, list(range(1000, 1000 + free)), bs, sum(new) // 2)
        assert N.device_status(clear=True) == N.DEV_BAD_POSITION
        return
    run_slots(tables, ctx, new, [1, 2, 3], bs, sum(new), head=9)      # a head past the list: nothing left
    run_slots([[] for _ in ctx], ctx, new, [1, 2, 3], bs, sum(new))   # no table entries at all


def test_slots_of_a_large_batch_need_a_workspace():
    x = torch.zeros(9001, dtype=torch.int32, device=DEV)
    p = x.data_ptr()
    need = N.lib().mvb_assign_slots_workspace_bytes(9000)
    assert need > 0 and N.lib().mvb_assign_slots_workspace_bytes(8192) == 0
    for ws, size in ((None, need), (p, need - 1), (p + 4, need)):
        rc = N.lib().mvb_assign_slots(p, p, p, p, p + 8, p, 1, 1, p, p, p, 5, None, 9000, 16, 0, ws, size, N.stream_handle())
        assert rc == 1 and b"workspace" in N.lib().mvb_last_error()


def test_slots_negative_lengths_are_refused():
    run_slots([[1, 2], [3, 4], [5, 6]], [4, -1, 3], [2, 2, -5], [7, 8, 9], 4, 6)
    assert N.device_status(clear=True) == N.DEV_BAD_POSITION


def test_slots_empty_batch_and_strided_tables():
    plan = ops.assign_slots(torch.zeros(0, 4, dtype=torch.int32, device=DEV), i32([]), i32([]), i32([1]), 16, 3)
    assert plan.slots.tolist() == [-1] * 3 and plan.seq_start.tolist() == [0] and plan.free_head.tolist() == [0]
    wide = torch.full((3, 9), 77, dtype=torch.int32, device=DEV)
    plan = ops.assign_slots(wide[:, 2:6], i32([0, 5, 16]), i32([17, 1, 16]), i32([4, 5, 6, 7]), 16, 34)
    assert wide.tolist() == [[77, 77, 4, 5, 77, 77, 77, 77, 77], [77] * 9, [77, 77, 77, 6, 77, 77, 77, 77, 77]]
    assert plan.slots.tolist() == [*range(64, 80), 80, 77 * 16 + 5, *range(96, 112)]
    for bad in (wide.t()[:4], wide[:1].expand(3, 9), wide.long()):
        with pytest.raises(RuntimeError):
            ops.assign_slots(bad, i32([0] * bad.shape[0]), i32([1] * bad.shape[0]), i32([4, 5, 6, 7]), 16, 3)


def test_slots_chain_follows_the_block_manager():
    """Many steps of ragged growth with the head kept on the GPU, captured once and replayed: the block
    manager's tables, slots and free list."""
    bs, B, P, width = 16, 9, 400, 30
    order = list(range(P))
    random.Random(1).shuffle(order)
    mgr = KVCacheManager(P, bs, 1, 1, 8, allocate_pool=False, free_order=order)
    free = i32(order)
    table = torch.zeros(B, width, dtype=torch.int32, device=DEV)
    ctx, new, head = i32([0] * B), i32([0] * B), i32([0])
    ops.assign_slots(table, ctx, new, free, bs, 64, free_head=head)           # warm-up: nothing to place
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan = ops.assign_slots(table, ctx, new, free, bs, 64, free_head=head)
        ctx += new
        head.copy_(plan.free_head)
    r = random.Random(2)
    for b in range(B):
        mgr.allocate(b, 0)
    for step in range(12):
        add = [r.randint(0, 7) for _ in range(B)]
        new.copy_(i32(add))
        g.replay()
        want = []
        for b, n in enumerate(add):
            for _ in range(n):
                assert mgr.append_token(b)
                block, off = mgr.slot(b, mgr.seq_num_tokens[b] - 1)
                want.append(block * bs + off)
        assert plan.slots.tolist() == want + [-1] * (64 - len(want))
    for b in range(B):
        blocks = mgr.get_block_table(b)
        assert table[b, :len(blocks)].tolist() == blocks
    assert int(head) == P - mgr.num_free_blocks


# ----------------------------------------------------------------------------- drafts
def probs(g, *shape, keep=0.3, sharp=3.0):
    x = torch.randn(*shape, generator=g) * sharp
    gone = torch.rand(*shape, generator=g) > keep
    gone[..., 0] = False                                          # no row without weight
    return x.masked_fill(gone, -math.inf).softmax(-1)


def verify_case(seed, B, K, V, keep=0.5):
    g = torch.Generator().manual_seed(seed)
    target = probs(g, B, K + 1, V, keep=keep)
    near = (target[:, :K].log() + 0.8 * torch.randn(B, K, V, generator=g)).softmax(-1)
    tokens = torch.multinomial(near.reshape(B * K, V), 1, generator=g).reshape(B, K) if K else torch.zeros(
        B, 0, dtype=torch.int64)
    u = torch.rand(B, K + 1, generator=g)
    lens = torch.randint(0, K + 1, (B,), generator=g).int()
    return target, near, tokens, u, lens


def run_verify(target, tokens, u, near, lens):
    want, count = ref.verify(target, tokens, u, near, lens)
    dev = [None if x is None else x.to(DEV) for x in (target, tokens, u, near, lens)]
    got, accepted = ops.verify_drafts(dev[0], dev[1], dev[2], draft_probs=dev[3], draft_lens=dev[4])
    assert accepted.dtype == torch.int32 and torch.equal(accepted.cpu(), count)
    assert got.dtype == torch.int64 and torch.equal(got.cpu(), want), (got.cpu() != want).nonzero()


@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 0, 7), (3, 2, 2), (5, 4, 31), (2, 3, 1000), (9, 1, 1025), (1, 8, 4099),
                                   (70, 3, 513), (2, 5, 33000), (1, 4, 151936), (3, 2, 256000)])
@pytest.mark.parametrize("form", ["probs", "lens", "onehot"])
def test_verify(B, K, V, form):
    target, near, tokens, u, lens = verify_case(B * 7 + K + V, B, K, V)
    run_verify(target, tokens, u, None if form == "onehot" or K == 0 else near, lens if form != "probs" else None)


def test_verify_uniforms_at_the_ends():
    target, near, tokens, u, lens = verify_case(3, 12, 3, 777)
    for value in (0.0, 1.0 - 2.0 ** -24):
        run_verify(target, tokens, torch.full_like(u, value), near, None)
        run_verify(target, tokens, torch.full_like(u, value), None, lens)


def test_verify_skips_entries_without_weight():
    """Rows with weight on few entries: a draw never lands on an entry of weight zero, first or last."""
    V = 5000
    target = torch.zeros(3, 1, V)
    target[0, 0, 4999] = 1.0
    target[1, 0, [7, 2048, 4096]] = torch.tensor([0.25, 0.5, 0.25])
    target[2, 0, 0] = 1.0
    for u in (0.0, 0.25, 0.5, 0.7499999, 0.99999994):
        run_verify(target, torch.zeros(3, 0, dtype=torch.int64), torch.full((3, 1), u), None, None)


def test_verify_nothing_left_and_no_weight():
    """q above p everywhere draws from p; a one-hot draft that held all of p too; a row without weight gives -1."""
    V = 300
    p = torch.zeros(3, 2, V)
    p[0, 0, 5], p[0, 0, 6] = 0.5, 0.25
    p[1, 0, 9] = 0.3
    q = torch.zeros(3, 1, V)
    q[0, 0, 5], q[0, 0, 6] = 0.6, 0.4
    q[1, 0, 9] = 1.0
    q[2, 0, 3] = 1.0
    tokens = torch.tensor([[6], [9], [3]])
    u = torch.tensor([[0.9, 0.8], [0.9, 0.5], [0.5, 0.5]])
    got, n = ops.verify_drafts(p.to(DEV), tokens.to(DEV), u.to(DEV), draft_probs=q.to(DEV))
    assert got.tolist() == [[6, -1], [9, -1], [-1, -1]] and n.tolist() == [0, 0, 0]
    got, n = ops.verify_drafts(p.to(DEV), tokens.to(DEV), u.to(DEV))
    assert got.tolist() == [[5, -1], [9, -1], [-1, -1]] and n.tolist() == [0, 0, 0]


def test_verify_nan_and_bad_tokens():
    """NaN probabilities reject and weigh nothing; a drafted token outside the vocabulary is rejected and reported."""
    target, near, tokens, u, _ = verify_case(5, 3, 2, 400)
    target[1, 0, int(tokens[1, 0])] = float("nan")
    got, n = ops.verify_drafts(target.to(DEV), tokens.to(DEV), u.to(DEV), draft_probs=near.to(DEV))
    assert int(n[1]) == 0 and 0 <= int(got[1, 0]) < 400 and int(got[1, 0]) != int(tokens[1, 0])
    want, _ = ref.verify(target[[0, 2]], tokens[[0, 2]], u[[0, 2]], near[[0, 2]])
    assert torch.equal(got[[0, 2]].cpu(), want)
    for bad in (-1, 400, 1 << 40):
        t = tokens.clone()
        t[0, 1] = bad
        u2 = u.clone()
        u2[0, 0] = 0.0
        got, n = ops.verify_drafts(target.to(DEV), t.to(DEV), u2.to(DEV), draft_probs=near.to(DEV))
        assert int(n[0]) <= 1 and 0 <= int(got[0, int(n[0])]) < 400
        assert N.device_status(clear=True) == N.DEV_BAD_TOKEN


def test_verify_strides():
    """Probabilities as slices of wider rows and of more positions, tokens in column order."""
    target, near, tokens, u, lens = verify_case(8, 4, 3, 1001)
    want = ops.verify_drafts(target.to(DEV), tokens.to(DEV), u.to(DEV), near.to(DEV), lens.to(DEV))
    for pad in (1, 8):
        wide = torch.full((4, 4, 1001 + pad), 9.0, device=DEV)
        wide[..., :1001] = target.to(DEV)
        more = torch.full((4, 5, 1001), 9.0, device=DEV)
        more[:, :3] = near.to(DEV)
        tok = tokens.to(DEV).t().contiguous().t()
        got = ops.verify_drafts(wide[..., :1001], tok, u.to(DEV), more[:, :3], lens.to(DEV))
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    flipped = target.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.verify_drafts(flipped, tokens.to(DEV), u.to(DEV), near.to(DEV), lens.to(DEV))[0], want[0])


def test_verify_refuses():
    target, near, tokens, u, lens = (x.to(DEV) for x in verify_case(9, 2, 2, 50))
    for args in ((target.double(), tokens, u, near, lens), (target, tokens.int(), u, near, lens),
                 (target, tokens[:, :1], u, near, lens), (target, tokens, u[:, :2], near, lens),
                 (target, tokens, u, near[:, :1], lens), (target, tokens, u, near, lens.long()),
                 (target, tokens, u, near, lens[:1]), (target, tokens, u.cpu(), near, lens), (target[0], tokens, u, near, lens)):
        with pytest.raises(RuntimeError):
            ops.verify_drafts(*args)
    out, n = ops.verify_drafts(target[:0], tokens[:0], u[:0])
    assert out.shape == (0, 3) and n.shape == (0,)


def test_verified_tokens_follow_the_target():
    """The point of the rule: over many uniforms the first token of a step is distributed as the target's first row."""
    V, B = 6, 60000
    g = torch.Generator().manual_seed(11)
    p, q = torch.rand(V, generator=g) + 0.05, torch.rand(V, generator=g) + 0.05
    p, q = p / p.sum(), q / q.sum()
    tokens = torch.multinomial(q, B, replacement=True, generator=g)[:, None]
    u = torch.rand(B, 2, generator=g)
    out, _ = ops.verify_drafts(p.expand(B, 2, V).contiguous().to(DEV), tokens.to(DEV), u.to(DEV),
                               draft_probs=q.expand(B, 1, V).contiguous().to(DEV))
    freq = torch.bincount(out[:, 0].cpu(), minlength=V) / B
    # five standard deviations of a frequency over B draws
    assert bool(((freq - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all()), (freq, p)


# ------------------------------------------------------------------------- a whole step
@pytest.mark.parametrize("captured", [False, True])
def test_speculative_steps_over_the_4bit_cache(captured):
    """Slots, quantised writes, attention of the drafted tokens and their verification, run together over
    several steps with the lengths kept on the GPU (as one captured graph, or eagerly), against the same
    steps in 64 bits."""
    B, T, Hq, Hkv, D, bs, P, V = 3, 4, 8, 2, 128, 16, 64, 97
    g = torch.Generator(device=DEV).manual_seed(4)
    order = torch.randperm(P, generator=g, device=DEV).int()
    pool = kv4_pool(P, bs, 1, Hkv, D)
    table = torch.zeros(B, 12, dtype=torch.int32, device=DEV)
    proj = torch.randn(Hq * D, V, generator=g, device=DEV) / math.sqrt(Hq * D) * 4
    held, head, new = i32([0] * B), i32([0]), i32([T] * B)
    x = torch.empty(B * T, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device=DEV)
    tokens = torch.empty(B, T - 1, dtype=torch.int64, device=DEV)
    u = torch.empty(B, T, device=DEV)

    def step():
        plan = ops.assign_slots(table, held, new, order, bs, B * T, free_head=head)
        k = x[:, Hq * D:(Hq + Hkv) * D].unflatten(1, (Hkv, D))
        v = x[:, (Hq + Hkv) * D:].unflatten(1, (Hkv, D))
        ops.kv4_write(k, v, pool, 0, plan.slots)
        ctx = held + new
        out = ops.paged_attention_decode_kv4(x[:, :Hq * D].unflatten(1, (Hq, D)).unflatten(0, (B, T)), pool, 0, table,
                                             ctx, 1 / math.sqrt(D))
        p = ops.softmax(out.float().flatten(2) @ proj)
        toks, n = ops.verify_drafts(p, tokens, u)
        held.add_(n + 1)                                        # the rejected drafts' slots are written again
        head.copy_(plan.free_head)
        return plan, out, p, toks, n

    def fill(i):
        gi = torch.Generator(device=DEV).manual_seed(100 + i)
        x.copy_(torch.randn(x.shape, generator=gi, device=DEV))
        tokens.copy_(torch.randint(0, V, tokens.shape, generator=gi, device=DEV))
        u.copy_(torch.rand(u.shape, generator=gi, device=DEV) * 0.02)   # flat targets: accept some

    graph = None
    if captured:
        fill(0)
        step()                                                    # warm-up, then start again
        held.zero_(), head.zero_(), pool.zero_(), table.zero_()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        held.zero_(), head.zero_()
    lens = [0] * B
    keys = [[] for _ in range(B)]
    vals = [[] for _ in range(B)]
    for i in range(6):
        fill(i)
        if captured:
            graph.replay()
        else:
            res = step()
        plan, out, p, toks, n = res
        assert plan.granted.tolist() == [1] * B
        k = ref.stored(x[:, Hq * D:(Hq + Hkv) * D].unflatten(1, (Hkv, D)).cpu())
        v = ref.stored(x[:, (Hq + Hkv) * D:].unflatten(1, (Hkv, D)).cpu())
        want, count = ref.verify(p.cpu(), tokens.cpu(), u.cpu())
        assert torch.equal(toks.cpu(), want) and torch.equal(n.cpu(), count)
        for b in range(B):
            del keys[b][lens[b]:], vals[b][lens[b]:]
            keys[b] += list(k[b * T:(b + 1) * T])
            vals[b] += list(v[b * T:(b + 1) * T])
            q = x[b * T:(b + 1) * T, :Hq * D].cpu().double().unflatten(1, (Hkv, Hq // Hkv, D))
            kk, vv = torch.stack(keys[b]), torch.stack(vals[b])
            for t in range(T):
                m = lens[b] + t + 1
                z = torch.einsum("hrd,nhd->hrn", q[t], kk[:m]) / math.sqrt(D)
                o = torch.einsum("hrn,nhd->hrd", z.softmax(-1), vv[:m]).flatten(0, 1)
                # bf16 rounding of the result (2^-8), weights of 11 bits over values of |v| < 5 (2^-11 * 10)
                assert float((out[b, t].cpu().double() - o).abs().max()) <= float(o.abs().max()) * 2.0 ** -8 + 2.0 ** -7.6
            lens[b] += int(count[b]) + 1
        assert held.tolist() == lens
