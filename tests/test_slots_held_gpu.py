"""Slot assignment on the GPU where lengths go back, as rejected drafts make them: the caller keeps the count of blocks
that each sequence holds."""
import math
import random

import pytest
import torch

import kv4_reference as ref
from llm_pytorch_inference_b200 import _native as N
from llm_pytorch_inference_b200 import ops
from llm_pytorch_inference_b200.kv_cache import kv4_pool

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _status_clean():
    N.device_status(clear=True)
    yield
    assert N.device_status(clear=True) == 0, "a kernel reported a device-side error"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def run(tables, ctx, new, held, free, bs, n, head=0):
    """One call against the sequences one by one; tables and held (lists) go on as the reference left them."""
    table, count = i32(tables), i32(held)
    plan = ops.assign_slots(table, i32(ctx), i32(new), i32(free), bs, n, free_head=i32([head]), held_blocks=count)
    slots, pos, start, granted, taken = ref.assign_held(tables, ctx, new, held, free, bs, n, head)
    assert plan.slots.tolist() == slots and plan.positions.tolist() == pos
    assert plan.seq_start.tolist() == start and plan.granted.tolist() == granted
    assert plan.free_head.tolist() == [taken] and table.tolist() == tables and count.tolist() == held
    return granted, taken


@pytest.mark.parametrize("batch,most,bs", [(1, 5, 16), (1, 3000, 16), (64, 5, 16), (300, 9, 4), (513, 40, 7), (6143, 2, 16),
                                           (8192, 3, 16), (8193, 3, 16), (20001, 2, 4)])
def test_slots_with_counts(batch, most, bs):
    """Counts at and above what the lengths need, one block to several calls' launches, and too few blocks or rows."""
    r = random.Random(batch + most)
    ctx = [r.randint(0, 3 * bs) for _ in range(batch)]
    new = [r.randint(0, most) for _ in range(batch)]
    width = max(-(-(c + n) // bs) for c, n in zip(ctx, new)) + 1
    held = [min(-(-c // bs) + r.randint(0, 2), width) for c in ctx]
    ids = list(range(batch * width + 7))
    r.shuffle(ids)
    tables = [[ids.pop() if i < h else -3 for i in range(width)] for h in held]
    lack = sum(max(-(-(c + n) // bs) - h, 0) for c, n, h in zip(ctx, new, held))
    for free, room in ((lack, sum(new)), (lack + 3, sum(new) + 20), (lack // 2, sum(new)), (lack, sum(new) // 2)):
        run([list(t) for t in tables], ctx, new, list(held), ids[:free] or [0], bs, room)
        run([list(t) for t in tables], ctx, new, list(held), [0] * 4 + ids[:free], bs, room, head=4)


def test_counts_that_cannot_be_are_refused():
    """A count below what the length needs (a refused sequence whose length moved on), negative, or past the row."""
    tables = [[1, 2, -1], [3, 4, 5], [6, 7, 8], [9, 0, 0], [11, 12, 0]]
    ctx, new = [17, 20, 1, 33, 16], [2] * 5
    granted, taken = run(tables, ctx, new, [1, -1, 4, 3, 1], [20, 21, 22], 16, 10)
    assert granted == [0, 0, 0, 1, 1] and taken == 1 and tables[4] == [11, 20, 0]
    assert N.device_status(clear=True) == N.DEV_BAD_POSITION
    n = 8200
    run([[b, -1, -1] for b in range(n)], [16] * n, [1] * n, [b % 5 for b in range(n)], list(range(n, 3 * n)), 16, n)
    assert N.device_status(clear=True) == N.DEV_BAD_POSITION


@pytest.mark.parametrize("drafted,accept", [(4, 0.0), (5, 0.0), (5, 0.6), (8, 0.6), (17, 0.3)])
@pytest.mark.parametrize("captured", [False, True])
def test_rejected_drafts_lose_no_blocks(drafted, accept, captured):
    """Many steps in which lengths grow by less than was granted: the blocks taken are those in the rows, no block is in
    two places, no entry changes once it is given, and no more blocks are taken than the longest reach needs."""
    B, bs, width, P = 4, 16, 40, 160
    order = list(range(P))
    random.Random(drafted).shuffle(order)
    free, table = i32(order), torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    ctx, new, held, head, more = i32([0, 3, 13, 16]), i32([drafted] * B), i32([0] * B), i32([0]), i32([0] * B)
    start = ctx.clone()

    def step():
        plan = ops.assign_slots(table, ctx, new, free, bs, B * drafted, free_head=head, held_blocks=held)
        ctx.add_(more * plan.granted)
        head.copy_(plan.free_head)
        return plan

    first = ops.assign_slots(table, i32([0] * B), ctx, free, bs, 32, free_head=head, held_blocks=held)   # the prompts
    head.copy_(first.free_head)
    graph = None
    if captured:
        keep = [x.clone() for x in (table, ctx, held, head)]
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan = step()
        for x, y in zip((table, ctx, held, head), keep):
            x.copy_(y)
    r = random.Random(drafted * 100)
    rows, reach = table.tolist(), start.tolist()
    for _ in range(60):
        before = ctx.tolist()
        if max(before) + drafted > width * bs:
            break
        took = []
        for _ in range(B):
            n = 1
            while n < drafted and r.random() < accept:
                n += 1
            took.append(n)
        more.copy_(i32(took))
        if captured:
            graph.replay()
        else:
            plan = step()
        assert plan.granted.tolist() == [1] * B and ctx.tolist() == [n + m for n, m in zip(before, took)]
        now = table.tolist()
        reach = [max(x, n + drafted) for x, n in zip(reach, before)]
        count = [-(-x // bs) for x in reach]
        assert held.tolist() == count and int(head) == sum(count)
        given = [x for row, n in zip(now, count) for x in row[:n]]
        assert given and len(set(given)) == len(given) and sorted(given) == sorted(order[:len(given)])
        for old, row in zip(rows, now):
            assert all(x == y for x, y in zip(old, row) if x >= 0)
        rows = now
        at = [b * drafted + i for b in range(B) for i in range(drafted)]
        slots = plan.slots.tolist()
        for t in at:
            b, pos = t // drafted, before[t // drafted] + t % drafted
            assert slots[t] == now[b][pos // bs] * bs + pos % bs


def test_counts_of_the_wrong_kind_are_refused():
    table, x = i32([[1, 2], [3, 4]]), i32([1, 1])
    for held in (i32([1]), i32([1, 1]).long(), torch.tensor([1, 1], dtype=torch.int32), i32([1, 1, 1, 1])[::2], x,
                 i32([[1, 1]])):
        with pytest.raises(RuntimeError):
            ops.assign_slots(table, x, i32([1, 1]), i32([5]), 16, 2, held_blocks=held)


@pytest.mark.parametrize("captured", [False, True])
def test_refused_sequences_touch_nothing(captured):
    """Speculative steps with too few blocks: a refused sequence keeps its length, gets zeros and changes no record, the
    granted one goes on, and once blocks come back the refused one resumes where it was."""
    B, T, Hq, Hkv, D, bs, V = 3, 2, 4, 2, 64, 16, 11
    g = torch.Generator(device=DEV).manual_seed(5)
    pool = kv4_pool(6, bs, 1, Hkv, D)
    table = torch.zeros(B, 4, dtype=torch.int32, device=DEV)               # entries never given name block 0
    ctx, new, held, head = i32([31, 15, 3]), i32([T] * B), i32([0] * B), i32([0])
    free = i32([0, 1, 2, 3, 5, 4])
    first = ops.assign_slots(table, i32([0] * B), ctx, free[:4], bs, 49, free_head=head, held_blocks=held)
    head.copy_(first.free_head)
    assert table[0, :2].tolist() == [0, 1] and int(table[1, 0]) == 2 and int(table[2, 0]) == 3 and int(head) == 4
    fill = torch.randn(2, 49, Hkv, D, generator=g, device=DEV).bfloat16()
    ops.kv4_write(fill[0], fill[1], pool, 0, first.slots)
    x = torch.randn(B * T, Hq + 2 * Hkv, D, generator=g, device=DEV).bfloat16()
    probs = torch.rand(B, T, V, generator=g, device=DEV)
    drafts = torch.randint(0, V, (B, T - 1), generator=g, device=DEV)
    u = torch.rand(B, T, generator=g, device=DEV)

    def step(n):
        plan = ops.assign_slots(table, ctx, new, free[:n], bs, B * T, free_head=head, held_blocks=held)
        seen = (ctx + new) * plan.granted
        ops.kv4_write(x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], pool, 0, plan.slots)
        out = ops.paged_attention_decode_kv4(x[:, :Hq].unflatten(0, (B, T)), pool, 0, table, seen, 1 / math.sqrt(D))
        tokens, accepted = ops.verify_drafts(probs, drafts, u)
        ctx.add_((accepted + 1) * plan.granted)
        head.copy_(plan.free_head)
        return plan, out

    graph = None
    if captured:
        keep = [t.clone() for t in (table, ctx, held, head, pool)]
        step(4)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan, out = step(4)
        for t, old in zip((table, ctx, held, head, pool), keep):
            t.copy_(old)
    before, length = pool.clone(), 3
    for _ in range(4):
        if captured:
            graph.replay()
        else:
            plan, out = step(4)
        assert plan.granted.tolist() == [0, 0, 1] and plan.slots[:4].tolist() == [-1] * 4
        assert ctx.tolist()[:2] == [31, 15] and length < int(ctx[2]) <= length + T
        assert held.tolist() == [2, 1, 1] and int(head) == 4
        assert not bool(out[:2].any()) and bool(out[2].any())
        assert torch.equal(pool[:, :3], before[:, :3]) and torch.equal(pool[:, 4:], before[:, 4:])
        length = int(ctx[2])
    plan, out = step(6)                                                    # two blocks more
    assert plan.granted.tolist() == [1, 1, 1] and held.tolist() == [3, 2, 1] and int(head) == 6
    assert table.tolist() == [[0, 1, 5, 0], [2, 4, 0, 0], [3, 0, 0, 0]]
    assert plan.slots[:4].tolist() == [31, 5 * 16, 2 * 16 + 15, 4 * 16]
    gk, gv = ops.kv4_read(pool, 0, first.slots)                            # the prompts are as they were written
    assert torch.equal(gk.cpu(), ref.stored(fill[0].cpu()).float().bfloat16())
    assert torch.equal(gv.cpu(), ref.stored(fill[1].cpu()).float().bfloat16())


def test_a_refused_length_that_moved_on_is_refused():
    """The step without the mask: the length counts entries that were never given (zeros: block 0, another sequence's)."""
    table, held, head = i32([[0, 1, 0], [2, 0, 0]]), i32([2, 1]), i32([0])
    for ctx in ([31, 17], [31, 19]):
        plan = ops.assign_slots(table, i32(ctx), i32([2, 2]), i32([9])[:0], 16, 4, free_head=head, held_blocks=held)
        assert plan.granted.tolist() == [0, 0] and plan.slots.tolist() == [-1] * 4 and held.tolist() == [2, 1]
        assert N.device_status(clear=True) == N.DEV_BAD_POSITION


@pytest.mark.parametrize("tokens", [0, 1, 700, 5000])
def test_slots_of_an_empty_batch(tokens):
    """No sequence, any padding, with and without a head: the head stays and every slot is -1."""
    none = i32([])
    for head, n in ((0, 0), (3, 9), (9, 9), (12, 9)):
        for held in (None, none.clone()):
            plan = ops.assign_slots(none.view(0, 4), none, none, i32(list(range(n))), 16, tokens, free_head=i32([head]),
                                    held_blocks=held)
            assert plan.slots.tolist() == [-1] * tokens and plan.seq_start.tolist() == [0]
            assert plan.free_head.tolist() == [head] and plan.granted.numel() == 0
