"""The 4-bit KV cache, slot assignment and draft verification: the calls that are measured.

Five operators of a serving step.  ``assign_slots`` grows the block tables and maps the new tokens
to cache slots, ``kv4_write`` / ``kv4_read`` quantise K and V into a paged 4-bit pool and give the
values back, ``paged_attention_decode_kv4`` attends over that pool, and ``verify_drafts`` accepts or
replaces drafted tokens.  ``run`` computes them with elementary torch operations where ``own`` is
false and calls the package's entry points where it is true.

The pool is uint8 ``[layers, blocks, kv_heads, block_size / 16, 18 * D]``: one record per 16 tokens
of a head, K codes ``[16, D/2]``, V codes ``[16, D/2]``, K (scale, min) pairs ``[16, D/64]`` and V
pairs, bf16.  A group of 64 channels shares one pair; a code u stands for ``min + scale * u``.  Of a
row's 32-bit words, word ``(D/64) * w + g`` holds channels ``64 g + 8 w .. + 7``, lowest nibble first.
"""
import math

import torch

own = False

DEV = "cuda"
GROUP = 64


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a full batch: a slot for each sequence's new token
        dict(name="slots decode b64", op="slots", batch=64, ctx=2048, new=1, block=16),
        # the prompts of a long ragged batch packed into one token batch
        dict(name="slots prefill b200", op="slots", batch=200, ctx=0, new=1000, block=16),
        # a decode step's K and V of one layer appended, Qwen3-8B heads
        dict(name="write decode n64 h8 d128", op="write", tokens=64, heads=8, dim=128, block=16),
        # a prefill's K and V of one layer, 8 prompts of 2048 tokens
        dict(name="write prefill n16384 h8 d128", op="write", tokens=16384, heads=8, dim=128, block=16),
        # the cached prefix of one short prompt read back, Gemma-2-9B heads
        dict(name="read prefix n333 h8 d256", op="read", tokens=333, heads=8, dim=256, block=32),
        # the cached prefixes of a batch read back for a prefill over them
        dict(name="read prefix n32768 h8 d128", op="read", tokens=32768, heads=8, dim=128, block=16),
        # the first steps of one short chat: latency
        dict(name="attend b1 ctx33", op="attend", batch=1, ctx=33, new=1, q_heads=32, heads=8, dim=128, block=16,
             softcap=0.0, window=0),
        # the headline decode batch, lengths of 1024 to 2048
        dict(name="attend b64 ctx2048", op="attend", batch=64, ctx=2048, new=1, q_heads=32, heads=8, dim=128,
             block=16, softcap=0.0, window=0),
        # a Gemma-2-9B global layer at long context: head size 256, capped scores
        dict(name="attend b16 ctx8192 d256 cap", op="attend", batch=16, ctx=8192, new=1, q_heads=16, heads=8,
             dim=256, block=16, softcap=50.0, window=0),
        # five drafted tokens of four long sequences scored at once
        dict(name="attend b4 t5 ctx32768", op="attend", batch=4, ctx=32768, new=5, q_heads=32, heads=8, dim=128,
             block=16, softcap=0.0, window=0),
        # one chat with four drafted tokens
        dict(name="verify b1 k4", op="verify", batch=1, drafts=4, vocab=151936, onehot=False),
        # a full batch, drafts of a small model with its probabilities
        dict(name="verify b64 k5", op="verify", batch=64, drafts=5, vocab=151936, onehot=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["slots", "write", "read", "attend", "attend", "verify"])
    block = rng.choice([16, 16, 32, 64])
    if op == "slots":
        if rng.random() < 0.5:
            return dict(op=op, batch=_log(rng, 1, 1024), ctx=_log(rng, 1, 8192), new=rng.randint(1, 8), block=block)
        new = _log(rng, 1, 4096)
        return dict(op=op, batch=_log(rng, 1, max(1, 200000 // new)), ctx=rng.choice([0, _log(rng, 1, 4096)]), new=new,
                    block=block)
    dim = rng.choice([64, 128, 128, 256])
    if op in ("write", "read"):
        heads = rng.choice([1, 2, 3, 4, 8, 16])
        return dict(op=op, tokens=_log(rng, 1, 32768 * 8 * 128 // (heads * dim) // 2), heads=heads, dim=dim, block=block)
    if op == "attend":
        heads = rng.choice([1, 2, 4, 5, 8])
        group = rng.choice([1, 2, 3, 4, 8]) if dim < 256 else rng.choice([1, 2, 4])
        ctx = _log(rng, 1, 65536)
        batch = _log(rng, 1, max(1, min(256, 16 * 8192 * 8 * 256 // (ctx * heads * dim) // 2)))
        return dict(op=op, batch=batch, ctx=ctx, new=min(rng.choice([1, 1, 1, 2, 4, 7]), ctx), q_heads=heads * group,
                    heads=heads, dim=dim, block=block, softcap=rng.choice([0.0, 0.0, 30.0]),
                    window=rng.choice([0, 0, _log(rng, 1, 4096)]))
    return dict(op=op, batch=_log(rng, 1, 64), drafts=rng.randint(1, 8) if rng.random() < 0.8 else 0,
                vocab=_log(rng, 1000, 100000), onehot=rng.random() < 0.3)


# ----------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lengths(g, lo, hi, n):
    """n lengths spread over [lo, hi], the longest among them, in an order of the seed's: their sum is the case's."""
    return torch.linspace(hi, lo, n, device=DEV).round().long()[torch.randperm(n, generator=g, device=DEV)]


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _keys(g, n, heads, dim):
    """K of unit size with a few channels of several times it, as keys after a rotary embedding have."""
    wide = 1 + 3 * (torch.rand(heads, dim, generator=g, device=DEV) > 0.95).float()
    return (_normal(g, n, heads, dim) * wide * (1.6 / dim ** 0.25)).bfloat16()


def _empty_pool(blocks, block, heads, dim):
    return torch.zeros(1, blocks, heads, block // 16, 18 * dim, dtype=torch.uint8, device=DEV)


def _tables(g, lens, block, spare=0):
    """Block tables of sequences of `lens` tokens over shuffled blocks, and the blocks that stay free."""
    held = (lens + block - 1) // block
    width = int(held.max()) + spare
    order = torch.randperm(int(held.sum()) + (spare + 1) * lens.numel(), generator=g, device=DEV).int()
    at = torch.arange(width, device=DEV)[None]
    start = held.cumsum(0) - held
    has = at < held[:, None]
    table = torch.where(has, order[torch.where(has, start[:, None] + at, 0)], 0)
    return table.contiguous(), order[int(held.sum()):].contiguous(), order.numel()


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["op"] == "slots":
        ctx = _lengths(g, c["ctx"] // 2, c["ctx"], c["batch"])
        new = _lengths(g, max(1, c["new"] // 2), c["new"], c["batch"])
        spare = (c["new"] + c["block"] - 1) // c["block"] + 1
        table, free, _ = _tables(g, torch.clamp(ctx, min=1), c["block"], spare)
        return dict(c, table=table, free=free, lens=ctx.int(), add=new.int(), total=int(new.sum()))
    if c["op"] in ("write", "read"):
        n, block = c["tokens"], c["block"]
        blocks = (n + block - 1) // block + 3
        order = torch.randperm(blocks, generator=g, device=DEV)
        at = torch.arange(n, device=DEV)
        if n <= 256:  # tokens of as many sequences
            slots = torch.randperm(blocks * block, generator=g, device=DEV)[:n]
        else:
            slots = order[at // block] * block + at % block
        k, v = _keys(g, n, c["heads"], c["dim"]), _normal(g, n, c["heads"], c["dim"]).bfloat16()
        pool = _empty_pool(blocks, block, c["heads"], c["dim"])
        s = dict(c, pool=pool, slots=slots)
        if c["op"] == "read":
            _store(pool, k, v, slots, block)
            return s
        return dict(s, k=k, v=v)
    if c["op"] == "attend":
        batch, block = c["batch"], c["block"]
        lens = torch.clamp(_lengths(g, c["ctx"] // 2, c["ctx"], batch), min=c["new"])
        table, _, blocks = _tables(g, lens, block)
        pool = _empty_pool(blocks, block, c["heads"], c["dim"])
        n = blocks * block
        part = max(1, (1 << 25) // (c["heads"] * c["dim"]))
        for lo in range(0, n, part):
            m = min(part, n - lo)
            slots = torch.arange(lo, lo + m, device=DEV)
            _store(pool, _keys(g, m, c["heads"], c["dim"]), _normal(g, m, c["heads"], c["dim"]).bfloat16(), slots, block)
        q = (_normal(g, batch, c["new"], c["q_heads"], c["dim"]) * 1.6 * c["dim"] ** 0.25).bfloat16()
        return dict(c, pool=pool, table=table, lens=lens.int(), q=q, scale=1 / math.sqrt(c["dim"]))
    b, k, vocab = c["batch"], c["drafts"], c["vocab"]
    logits = 3 * _normal(g, b, k + 1, vocab)
    logits = logits.masked_fill(logits < 3.0, -math.inf)  # what a nucleus leaves
    target = logits.softmax(-1)
    near = (logits[:, :k] + 0.7 * _normal(g, b, k, vocab)).softmax(-1)
    if k:
        tokens = torch.multinomial((target[:, :k] if c["onehot"] else near).reshape(b * k, vocab), 1,
                                   generator=g).reshape(b, k)
    else:
        tokens = torch.zeros(b, 0, dtype=torch.int64, device=DEV)
    u = torch.rand(b, k + 1, generator=g, device=DEV)
    lens = torch.clamp(_lengths(g, (k + 1) // 2, k + 2, b), max=k).int()
    return dict(c, target=target, near=None if c["onehot"] else near, tokens=tokens, u=u, lens=lens)


# ------------------------------------------------------------------------------------ plain forms
def _quantise(x):
    """Codes, scales and mins of groups of 64 channels: [..., D] -> [..., D/64, 64], [..., D/64] twice."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low = x.amin(-1).bfloat16().float()
    scale = ((x.amax(-1) - low) / 15).bfloat16().float()
    steps = torch.where(scale[..., None] > 0, (x - low[..., None]) / scale[..., None], 0.0)
    return steps.round().clamp(0, 15).to(torch.uint8), scale, low


def _packed(codes):
    """[..., D/64, 64] codes -> [..., D/2] bytes in the pool's order of words."""
    w = codes.unflatten(-1, (8, 4, 2))
    return (w[..., 0] | (w[..., 1] << 4)).transpose(-3, -2).flatten(-3)


def _pairs(scale, low):
    return torch.stack([scale, low], -1).bfloat16().view(torch.uint8).flatten(-2)


def _store(pool, k, v, slots, block):
    dim = pool.shape[-1] // 18
    blocks, inside = slots // block, slots % block
    rec, row = inside // 16, inside % 16
    flat = pool[0].transpose(1, 2)  # [blocks, records, heads, bytes]
    for x, codes, pairs in ((k, 0, 16 * dim), (v, 8 * dim, 17 * dim)):
        u, scale, low = _quantise(x)
        flat[..., codes:codes + 8 * dim].unflatten(-1, (16, -1)).permute(0, 1, 3, 2, 4)[blocks, rec, row] = _packed(u)
        flat[..., pairs:pairs + dim].unflatten(-1, (16, -1)).permute(0, 1, 3, 2, 4)[blocks, rec, row] = _pairs(scale, low)


def _stands_for(codes, pairs):
    """[..., D/2] bytes and [..., D/16] bytes -> [..., D] values in 32 bits."""
    groups = pairs.shape[-1] // 4
    w = codes.unflatten(-1, (8, groups, 4))
    u = torch.stack([w & 15, w >> 4], -1).flatten(-2).transpose(-3, -2)  # [..., groups, 8, 8]
    p = pairs.contiguous().view(torch.bfloat16).float().unflatten(-1, (groups, 2))
    return (p[..., 0, None, None] * u.float() + p[..., 1, None, None]).flatten(-3)


def _rows(pool, slots, block):
    dim = pool.shape[-1] // 18
    blocks, inside = slots // block, slots % block
    flat = pool[0].transpose(1, 2)[blocks, inside // 16]  # [tokens, heads, bytes]
    row = (inside % 16)[:, None, None, None]

    def of(lo, n):
        x = flat[..., lo:lo + n].unflatten(-1, (16, -1))
        return x.gather(2, row.expand(-1, x.shape[1], 1, x.shape[3])).squeeze(2)

    return _stands_for(of(0, 8 * dim), of(16 * dim, dim)), _stands_for(of(8 * dim, 8 * dim), of(17 * dim, dim))


def _plain_slots(s):
    lens, add, block, total = s["lens"].long(), s["add"].long(), s["block"], s["total"]
    first = (lens + block - 1) // block
    grown = (lens + add + block - 1) // block - first
    base = grown.cumsum(0) - grown
    start = torch.cat([add.new_zeros(1), add.cumsum(0)])
    table, at = s["table"], torch.arange(s["table"].shape[1], device=DEV)[None]
    fresh = (at >= first[:, None]) & (at < (first + grown)[:, None])
    table = torch.where(fresh, s["free"][torch.where(fresh, base[:, None] + at - first[:, None], 0)], table)
    seq = torch.repeat_interleave(torch.arange(lens.numel(), device=DEV), add, output_size=total)
    pos = torch.arange(total, device=DEV) - start[seq] + lens[seq]
    slots = table[seq, pos // block].long() * block + pos % block
    return [slots, pos.int(), start.int(), torch.ones_like(s["lens"]), grown.sum().int().reshape(1), table]


def _plain_attend(s):
    batch, new, hq, dim = s["q"].shape
    heads, block = s["heads"], s["block"]
    group = hq // heads
    rec = s["pool"][0][s["table"].long()].transpose(2, 3).flatten(1, 2)  # [batch, records, heads, bytes]

    def values(codes, pairs):
        c = rec[..., codes:codes + 8 * dim].unflatten(-1, (16, -1))
        p = rec[..., pairs:pairs + dim].unflatten(-1, (16, -1))
        return _stands_for(c, p).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [batch, heads, tokens, D]

    k = values(0, 16 * dim)
    q = s["q"].float().unflatten(2, (heads, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [b, heads, new*group, D]
    score = q @ k.transpose(-1, -2) * s["scale"]
    del k
    if s["softcap"]:
        score = s["softcap"] * torch.tanh(score / s["softcap"])
    sees = s["lens"].long()[:, None] - new + 1 + torch.arange(new, device=DEV)  # keys that each query sees
    at = torch.arange(score.shape[-1], device=DEV)
    mask = at < sees[..., None]
    if s["window"]:
        mask &= at >= sees[..., None] - s["window"]
    mask = mask[:, None, :, None].expand(-1, 1, -1, group, -1).flatten(2, 3)
    score = score.masked_fill(~mask, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p @ values(8 * dim, 17 * dim)) / torch.where(total == 0, 1.0, total)
    return out.unflatten(2, (new, group)).permute(0, 2, 1, 3, 4).flatten(2, 3).to(s["q"].dtype)


def _plain_verify(s):
    target, near, tokens = s["target"], s["near"], s["tokens"]
    b, rows, vocab = target.shape
    k = rows - 1
    each = torch.arange(b, device=DEV)
    p = target[:, :k].gather(-1, tokens[..., None]).squeeze(-1).double()
    q = torch.ones_like(p) if near is None else near.gather(-1, tokens[..., None]).squeeze(-1).double()
    ok = (s["u"][:, :k].double() * q < p) & (torch.arange(k, device=DEV) < s["lens"][:, None])
    n = ok.long().cumprod(-1).sum(-1)
    w = target[each, n].double()
    rejected = n < s["lens"]
    at = torch.clamp(n, max=max(k - 1, 0))
    if k:
        if near is None:
            less = torch.arange(vocab, device=DEV) == tokens[each, at][:, None]
            left = torch.where(less, 0.0, w)
        else:
            left = (w - near[each, at].double()).clamp_min(0)
        left = torch.where(left.sum(-1, keepdim=True) > 0, left, w)
        w = torch.where(rejected[:, None], left, w)
    sums = w.cumsum(-1)
    drawn = (sums > s["u"][:, k:].double() * sums[:, -1:]).long().argmax(-1)
    out = torch.full((b, k + 1), -1, dtype=torch.int64, device=DEV)
    out[:, :k] = torch.where(torch.arange(k, device=DEV) < n[:, None], tokens, -1)
    out[each, n] = drawn
    return [out, n.int()]


# -------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        from llm_pytorch_inference_b200 import ops

        if s["op"] == "slots":
            plan = ops.assign_slots(s["table"], s["lens"], s["add"], s["free"], s["block"], s["total"])
            return [plan.slots, plan.positions, plan.seq_start, plan.granted, plan.free_head, s["table"]]
        if s["op"] == "write":
            ops.kv4_write(s["k"], s["v"], s["pool"], 0, s["slots"])
            return ops.kv4_read(s["pool"], 0, s["slots"])
        if s["op"] == "read":
            return ops.kv4_read(s["pool"], 0, s["slots"])
        if s["op"] == "attend":
            return ops.paged_attention_decode_kv4(s["q"], s["pool"], 0, s["table"], s["lens"], s["scale"],
                                                  softcap=s["softcap"], window=s["window"])
        return ops.verify_drafts(s["target"], s["tokens"], s["u"], draft_probs=s["near"], draft_lens=s["lens"])
    if s["op"] == "slots":
        return _plain_slots(s)
    if s["op"] == "write":
        _store(s["pool"], s["k"], s["v"], s["slots"], s["block"])
        return [x.bfloat16() for x in _rows(s["pool"], s["slots"], s["block"])]
    if s["op"] == "read":
        return [x.bfloat16() for x in _rows(s["pool"], s["slots"], s["block"])]
    if s["op"] == "attend":
        return _plain_attend(s)
    return _plain_verify(s)


def work(case):
    c = case
    if c["op"] == "slots":
        new = c["batch"] * max(1, 0.75 * c["new"])
        # lengths in, starts out; a slot and a position per token; a table entry and a free block per new block
        return {"bytes": c["batch"] * 16 + new * 12 + new / c["block"] * 8, "flops": 0}
    if c["op"] in ("write", "read"):
        n = c["tokens"] * c["heads"] * c["dim"] * 2
        wide, held = n * 2, n * 9 / 16  # bf16; 4 bits and 32 bits per 64 channels
        return {"bytes": (2 * wide + 2 * held if c["op"] == "write" else wide + held) + 8 * c["tokens"], "flops": 4 * n}
    if c["op"] == "attend":
        mean = max(c["new"], 0.75 * c["ctx"])
        keys = min(mean, c["window"] + c["new"] - 1) if c["window"] else mean
        cache = c["batch"] * keys * c["heads"] * c["dim"] * 2 * 9 / 16
        io = c["batch"] * c["new"] * c["q_heads"] * c["dim"] * 2 * 2
        return {"bytes": cache + io, "flops": 4 * c["batch"] * c["new"] * c["q_heads"] * c["dim"] * keys}
    # the drafted tokens' probabilities, and of one position the target's row (and the drafting model's)
    rows = 1 if c["onehot"] or not c["drafts"] else 2
    return {"bytes": c["batch"] * (rows * c["vocab"] * 4 + (c["drafts"] + 1) * 28), "flops": c["batch"] * c["vocab"] * 3}


# ------------------------------------------------------------------------------- 64-bit reference
def _exact_values(x):
    """What a stored row stands for: x in 64 bits, [n, heads, D], by the definition."""
    groups = x.double().reshape(*x.shape[:2], -1, GROUP)
    low = groups.min(-1, keepdim=True).values
    step = ((groups.max(-1, keepdim=True).values - low) / 15).to(torch.bfloat16).double()
    u = torch.where(step > 0, torch.round((groups - low) / torch.where(step > 0, step, 1.0)), 0.0)
    return (low + step * u.clamp(0, 15)).reshape(x.shape)


def _exact_rows(pool, blocks):
    """K and V of all tokens of `blocks` of one sequence in 64 bits, [tokens, heads, D]."""
    heads, recs, nbytes = pool.shape[2:]
    dim = nbytes // 18
    r = pool[0, blocks].permute(0, 2, 1, 3).reshape(-1, heads, nbytes)  # [records, heads, bytes]
    chan = torch.arange(dim, device=DEV)
    grp, word, nib = chan // 64, chan % 64 // 8, chan % 8
    byte = ((dim // 64) * word + grp) * 4 + nib // 2

    def of(codes, pairs):
        c = r[..., codes:codes + 8 * dim].reshape(*r.shape[:2], 16, dim // 2)[..., byte]
        u = torch.div(c, torch.where(nib % 2 == 1, 16, 1), rounding_mode="floor") % 16
        p = r[..., pairs:pairs + dim].reshape(-1, 2).contiguous().view(torch.int16).to(torch.int32) << 16
        p = p.view(torch.float32).double().reshape(*r.shape[:2], 16, dim // 64, 2)
        x = p[..., 1][..., grp] + p[..., 0][..., grp] * u.double()
        return x.permute(0, 2, 1, 3).reshape(-1, heads, dim)

    return of(0, 16 * dim), of(8 * dim, 17 * dim)


def _exact_slots(s):
    """The sequences one after another, as a block manager on the host grows them."""
    block, table, free = s["block"], s["table"].tolist(), s["free"].tolist()
    slots, positions, start, taken = [], [], [0], 0
    for row, n, add in zip(table, s["lens"].tolist(), s["add"].tolist()):
        for at in range(-(-n // block), -(-(n + add) // block)):
            row[at] = free[taken]
            taken += 1
        positions += range(n, n + add)
        slots += [row[at // block] * block + at % block for at in range(n, n + add)]
        start.append(start[-1] + add)
    small = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (positions, start, [1] * len(table), [taken], table)]
    return [torch.tensor(slots, device=DEV)] + small


def _exact_verify(s):
    """Sequence by sequence, draft by draft; the sums in 64 bits."""
    b, rows, _ = s["target"].shape
    out, count = [], []
    for i in range(b):
        row, n, u = [], 0, s["u"][i].tolist()
        drafts = s["tokens"][i].tolist()
        left = s["target"][i, 0].double()
        for n in range(rows):
            left = s["target"][i, n].double()
            if n == int(s["lens"][i]):
                break
            d = drafts[n]
            other = s["near"][i, n].double() if s["near"] is not None else torch.zeros_like(left).index_fill(
                0, torch.tensor([d], device=DEV), 1.0)
            if not u[n] * float(other[d]) < float(left[d]):
                rest = torch.where(other < left, left - other, 0.0)
                if s["near"] is None:
                    rest = torch.where(other > 0, 0.0, left)
                left = rest if float(rest.sum()) > 0 else left
                break
            row.append(d)
        sums = left.cumsum(0)
        row.append(int(torch.searchsorted(sums, (u[-1] * sums[-1]).reshape(1), right=True)))
        count.append(len(row) - 1)
        out.append(row + [-1] * (rows - len(row)))
    return [torch.tensor(out, device=DEV), torch.tensor(count, dtype=torch.int32, device=DEV)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "slots":
        return _exact_slots(s)
    if case["op"] == "write":
        return [_exact_values(s["k"]), _exact_values(s["v"])]
    block = case.get("block")
    if case["op"] == "read":
        blocks, where = torch.unique(s["slots"] // block, return_inverse=True)
        k, v = _exact_rows(s["pool"], blocks)
        at = where * block + s["slots"] % block
        return [k[at], v[at]]
    if case["op"] == "verify":
        return _exact_verify(s)
    b, new, hq, dim = s["q"].shape
    out = torch.zeros(b, new, hq, dim, dtype=torch.float64, device=DEV)
    rep = hq // case["heads"]
    for i in range(b):
        n = int(s["lens"][i])
        k, v = _exact_rows(s["pool"], s["table"][i, :(n + block - 1) // block].long())
        for t in range(new):
            end = n - new + 1 + t
            lo = max(0, end - case["window"]) if case["window"] else 0
            q = s["q"][i, t].double().reshape(case["heads"], rep, dim)
            z = torch.einsum("hrd,nhd->hrn", q, k[lo:end]) * s["scale"]
            if case["softcap"]:
                z = case["softcap"] * torch.tanh(z / case["softcap"])
            out[i, t] = torch.einsum("hrn,nhd->hrd", torch.softmax(z, -1), v[lo:end]).reshape(hq, dim)
    return out
