"""Plain implementations, in 64 bits, of the 4-bit KV cache operators, slot assignment and draft verification."""
import math

import torch


# ------------------------------------------------------------------ the 4-bit pool
def quantise(x: torch.Tensor):
    """codes, scale, min of bf16 x [..., D]: scale and min as stored (bf16, the quotient in fp32)."""
    g = x.double().unflatten(-1, (-1, 64))
    low = g.amin(-1)
    scale = ((g.amax(-1) - low).float() / torch.tensor(15.0)).bfloat16().double()
    step = torch.where(scale > 0, scale, 1.0)[..., None]
    codes = torch.where(scale[..., None] > 0, torch.round((g - low[..., None]) / step), 0.0).clamp(0, 15)
    return codes, scale, low


def stored(x: torch.Tensor) -> torch.Tensor:
    """The values that x reads back as, before the rounding to bf16."""
    codes, scale, low = quantise(x)
    return (low[..., None] + scale[..., None] * codes).flatten(-2)


def pack(pool: torch.Tensor, layer: int, k: torch.Tensor, v: torch.Tensor, slots: list[int], block_size: int) -> None:
    """Writes k, v [tokens, heads, D] (CPU) into a CPU pool, byte by byte as the layout says."""
    D = k.shape[-1]
    ng = D // 64
    for x, code_at, pair_at in ((k, 0, 16 * D), (v, 8 * D, 17 * D)):
        codes, scale, low = quantise(x)
        codes = codes.to(torch.int64)
        pairs = torch.stack([scale, low], -1).to(torch.bfloat16).view(torch.int16).to(torch.int64) & 0xFFFF
        for t, slot in enumerate(slots):
            if slot < 0:
                continue
            block, off = divmod(slot, block_size)
            rec, row = divmod(off, 16)
            for h in range(k.shape[1]):
                r = pool[layer, block, h, rec]
                for g in range(ng):
                    for c in range(64):
                        word = ng * (c // 8) + g
                        at = code_at + row * (D // 2) + 4 * word + (c % 8) // 2
                        keep = 0xF0 if c % 2 == 0 else 0x0F
                        r[at] = (int(r[at]) & keep) | (int(codes[t, h, g, c]) << (4 * (c % 2)))
                    for i in range(2):
                        p = int(pairs[t, h, g, i])
                        at = pair_at + row * 4 * ng + 4 * g + 2 * i
                        r[at], r[at + 1] = p & 255, p >> 8


def unpack(pool: torch.Tensor, layer: int, blocks: torch.Tensor):
    """K and V of all tokens of `blocks`, [tokens, heads, D] in 64 bits (any device)."""
    r = pool[layer, blocks].permute(0, 2, 1, 3).flatten(0, 1)          # [records, heads, 18 D]
    D = pool.shape[-1] // 18
    ng = D // 64

    def of(code_at, pair_at):
        b = r[..., code_at:code_at + 8 * D].reshape(*r.shape[:2], 16, 8, ng, 4).to(torch.int32)
        u = torch.stack([b & 15, b >> 4], -1).flatten(-2)              # [.., 16, 8, ng, 8]
        u = u.transpose(-3, -2).flatten(-2)                            # [.., 16, ng, 64]
        p = r[..., pair_at:pair_at + D].contiguous().view(torch.bfloat16).double().reshape(*r.shape[:2], 16, ng, 2)
        x = (p[..., 1:] + p[..., :1] * u.double()).flatten(-2)
        return x.permute(0, 2, 1, 3).flatten(0, 1)

    return of(0, 16 * D), of(8 * D, 17 * D)


def attention(q, pool, layer, tables, ctx, scale, softcap=0.0, window=0):
    """[B, T, Hq, D] in 64 bits, and how far a kernel may be off: see below."""
    B, T, Hq, D = q.shape
    heads, bs = pool.shape[2], 16 * pool.shape[3]
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = int(ctx[b])
        if n <= 0:
            continue
        blocks = tables[b, :(n + bs - 1) // bs].tolist()
        assert len(blocks) * bs >= n and all(0 <= i < pool.shape[1] for i in blocks)   # before the GPU indexes with them
        k, v = unpack(pool, layer, torch.tensor(blocks, device=pool.device))
        for t in range(T):
            end = n - T + 1 + t
            lo = max(0, end - window) if window else 0
            if end <= lo:
                continue
            qt = q[b, t].double().unflatten(0, (heads, Hq // heads))
            kk, vv = k[lo:end], v[lo:end]
            z = torch.einsum("hrd,nhd->hrn", qt, kk) * scale
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            out[b, t] = torch.einsum("hrn,nhd->hrd", z.softmax(-1), vv).flatten(0, 1)
            # Score: room for a q in 16 bits of its row's largest magnitude (half a step of |q|max / 32512 a channel, against
            # k; attention_each has none), and at most D + 64 fp32 roundings of terms whose magnitudes sum to m (the products, or scale * code
            # products and the min's part, each within 4 times |q| |k|max).  The softmax turns an error d of the scores
            # into 2 d of a weight.  Weights: rounded to 11 bits before the product with the codes (2^-11 of the
            # span of a group), plus 2^-21 for exp2 and sums.
            span = (vv.unflatten(-1, (-1, 64)).amax(-1) - vv.unflatten(-1, (-1, 64)).amin(-1)).amax()
            m = 4 * torch.einsum("hrd,nhd->hrn", qt.abs(), kk.abs()).amax(-1) * scale    # codes and min apart
            held = qt.abs().amax(-1) / 32512 / 2 * kk.abs().sum(-1).amax(0)[:, None] * scale
            weight = 2 * (held + (D + 64) * 2.0 ** -24 * m + 2.0 ** -21)
            vmax = vv.abs().amax()
            tol[b, t] = (weight[..., None] * vmax + 2.0 ** -11 * 1.1 * (span + 2.0 ** -10 * vmax)).expand(
                -1, -1, D).flatten(0, 1)
    return out, tol + out.abs() * 2.0 ** -8                            # and the rounding of the result to bf16


def attention_each(q, pool, layer, tables, ctx, scale, softcap=0.0, window=0):
    """The same, with a bound for each output by itself: from what its row's scores and the values of its group of
    channels, weighted as they are, can lose.

    A score is sum_g s_g (q_g . u_g) + m_g sum(q_g), with q exact.  With M = sum |q| (|k - m| + |m|) of the key, its terms
    magnitude by magnitude, fp32 sums of 64 terms, truncated by the matrix instruction (2^-23 each, a running sum and a
    term), and some 2 a group and 8 more roundings put it off by (4 * 64 + 2 groups + 8) 2^-24 M; a capped score by 2^-21
    of the cap more; its factor, its distance to the reference and exp2 by 2^-22 of its magnitude and 2^-21 of the weight.
    An error e_n of weight n moves the output by p_n e_n (v_n - out).  The weight in the product with the codes is rounded
    to 11 bits: 2^-11 p_n |v_n - m_n|.  A p s below 2^-14 as scaled is off by 2^-25 there, times a code of 15.  The largest
    p s of the output's row and group, or their sum, is scaled to 2^0 at least, so in the channel of its largest code, 14 at
    least, the sum of p |v - m| stands at 14 or above: n errors are 15 / 14 n 2^-25 of that channel's sum.  fp32 sums of the outputs, over 16 keys at
    a time, lose 2^-23 of the magnitudes each, twice where a part is scaled again and joined."""
    B, T, Hq, D = q.shape
    heads, bs, ng = pool.shape[2], 16 * pool.shape[3], q.shape[-1] // 64
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = int(ctx[b])
        if n <= 0:
            continue
        blocks = tables[b, :(n + bs - 1) // bs].tolist()
        assert len(blocks) * bs >= n and all(0 <= i < pool.shape[1] for i in blocks)   # before the GPU indexes with them
        at = torch.tensor(blocks, device=pool.device)
        k, v = unpack(pool, layer, at)
        km, vm = mins(pool, layer, at)                                  # [tokens, heads, D]: the group's min
        for t in range(T):
            end = n - T + 1 + t
            lo = max(0, end - window) if window else 0
            if end <= lo:
                continue
            qt = q[b, t].double().unflatten(0, (heads, Hq // heads))
            z = torch.einsum("hrd,nhd->hrn", qt, k[lo:end]) * scale
            M = torch.einsum("hrd,nhd->hrn", qt.abs(), (k - km)[lo:end].abs() + km[lo:end].abs()) * abs(scale)
            off = (4 * 64 + 2 * ng + 8) * 2.0 ** -24 * M
            if softcap:
                z = softcap * torch.tanh(z / softcap)
                off = off + 2.0 ** -21 * softcap
            p = z.softmax(-1)
            off = off + 2.0 ** -22 * (z.abs() + z.amax(-1, keepdim=True).abs()) + 2.0 ** -21
            vv, part = v[lo:end], (v - vm)[lo:end].abs()
            o = torch.einsum("hrn,nhd->hrd", p, vv)
            away = (vv.permute(1, 0, 2)[:, None] - o[:, :, None]).abs()  # [heads, rows, n, D]
            err = torch.einsum("hrn,hrnd->hrd", p * off, away) * 1.05
            err = err + 2.0 ** -11 * torch.einsum("hrn,nhd->hrd", p, part)
            top = torch.einsum("hrn,nhd->hrd", p, part).unflatten(-1, (ng, 64)).amax(-1)   # of the group
            err = err + 2.0 ** -25 * 15 / 14 * (end - lo) * top.repeat_interleave(64, -1)
            steps = (end - lo) // 16 + 4
            err = err + 2.0 ** -22 * steps * torch.einsum("hrn,nhd->hrd", p, part + vm[lo:end].abs())
            out[b, t], tol[b, t] = o.flatten(0, 1), err.flatten(0, 1)
    return out, tol + out.abs() * 2.0 ** -8                            # and the rounding of the result to bf16


def mins(pool, layer, blocks):
    """The group minima of K and V of all tokens of `blocks`, [tokens, heads, D] in 64 bits."""
    r = pool[layer, blocks].permute(0, 2, 1, 3).flatten(0, 1)
    D = pool.shape[-1] // 18

    def of(at):
        p = r[..., at:at + D].contiguous().view(torch.bfloat16).double().reshape(*r.shape[:2], 16, D // 64, 2)[..., 1]
        return p.permute(0, 2, 1, 3).flatten(0, 1).repeat_interleave(64, -1)

    return of(16 * D), of(17 * D)


# ------------------------------------------------------------------ slots
def assign(tables, ctx, new, free, block_size, num_tokens, head=0):
    """The sequences one after another; lists in, lists out (tables is changed)."""
    slots, positions, start, granted = [-1] * num_tokens, [0] * num_tokens, [0], []
    taken = max(head, 0)
    for row, n, add in zip(tables, ctx, new):
        ok = n >= 0 and add >= 0
        add = max(add, 0)
        end = start[-1] + add
        held, need = -(-max(n, 0) // block_size), -(-(max(n, 0) + add) // block_size)
        ok = ok and max(n, 0) + add <= len(row) * block_size and end <= num_tokens
        ok = ok and taken + need - held <= max(len(free), taken)
        if ok:
            for i in range(held, need):
                row[i] = free[taken]
                taken += 1
        for i in range(add):
            t, pos = start[-1] + i, max(n, 0) + i
            if t < num_tokens:
                positions[t] = pos
                slots[t] = row[pos // block_size] * block_size + pos % block_size if ok else -1
        start.append(end)
        granted.append(int(ok))
    return slots, positions, start, granted, taken


def assign_held(tables, ctx, new, held, free, block_size, num_tokens, head=0):
    """The same with the count of blocks that each sequence holds (a list, changed)."""
    slots, positions, start, granted = [-1] * num_tokens, [0] * num_tokens, [0], []
    taken = max(head, 0)
    for b, (row, n, add) in enumerate(zip(tables, ctx, new)):
        ok = n >= 0 and add >= 0 and -(-n // block_size) <= held[b] <= len(row)
        add = max(add, 0)
        end = start[-1] + add
        need = -(-(max(n, 0) + add) // block_size)
        ok = ok and need <= len(row) and end <= num_tokens
        ok = ok and taken + max(need - held[b], 0) <= max(len(free), taken)
        if ok:
            for i in range(held[b], need):
                row[i] = free[taken]
                taken += 1
            held[b] = max(held[b], need)
        for i in range(add):
            t, pos = start[-1] + i, max(n, 0) + i
            if t < num_tokens:
                positions[t] = pos
                block = row[pos // block_size] if ok else -1          # an entry that names no block gives no slot
                slots[t] = block * block_size + pos % block_size if block >= 0 else -1
        start.append(end)
        granted.append(int(ok))
    return slots, positions, start, granted, taken


# ------------------------------------------------------------------ drafts
def verify(target, tokens, uniforms, draft=None, lens=None):
    """(tokens [B, K + 1], accepted [B]) on the CPU; probabilities in, sums in 64 bits."""
    B, rows, V = target.shape
    out, count = [], []
    for b in range(B):
        n_drafts = rows - 1 if lens is None else int(lens[b])
        row = []
        w = None
        for i in range(n_drafts):
            d = int(tokens[b, i])
            p = target[b, i].double()
            q = draft[b, i].double() if draft is not None else torch.zeros(V, dtype=torch.float64).index_fill_(
                0, torch.tensor([d]), 1.0)
            if float(uniforms[b, i]) * float(q[d]) < float(p[d]):
                row.append(d)
                continue
            w = (p - q).clamp_min(0) if draft is not None else p.index_fill(0, torch.tensor([d]), 0.0)
            if not float(w.sum()) > 0:
                w = p
            break
        if w is None:
            w = target[b, len(row)].double()
        total = math.fsum(w.tolist())
        pick, acc = -1, 0.0
        if total > 0:
            sums = w.cumsum(0)
            pick = int(torch.searchsorted(sums, float(uniforms[b, -1]) * sums[-1], right=True))
        count.append(len(row))
        row.append(pick)
        out.append(row + [-1] * (rows - len(row)))
    return torch.tensor(out), torch.tensor(count, dtype=torch.int32)
