"""4-bit weights and 8-bit rows: the calls that are measured.

The linear layers of a serving step with weights in 4 bits.  ``quantise_w4`` turns a bf16 weight
matrix into codes with group scales, ``linear_w4`` multiplies rows by it: bf16 rows, or the 8-bit rows
with one scale each that ``fused_add_rmsnorm_q8`` and ``swiglu_q8`` / ``geglu_q8`` make.  ``run`` computes
them with elementary torch operations where ``own`` is false and calls the package's entry points where it
is true.

A weight is ``scale * (code - zero)``: codes and zeros of 0 to 15, bf16 scales, one scale and zero per row and
group of 32, 64 or 128 columns.  They are held in records of 16 rows by 128 columns, uint8 ``[records, 1024 + 64 *
(128 / group)]``.  First the codes, 64 bytes a row: 16 bytes at place ``p`` of row ``r`` hold the columns
``32 i + 8 t .. + 7`` of word ``i = 0 .. 3``, with ``t = p ^ (r / 2 % 4)``, and a word's nibbles, lowest first, are its
columns 0, 2, 4, 6, 1, 3, 5, 7.  Then for each row one 32-bit word per group: the scale's bits, and the bf16 number
``128 + zero`` above them.  What lies behind the last row or column is zero.  The records of 128 rows stand
together: for each 128 columns the 8 (behind the last whole 128 rows: the remaining) records of those rows.
"""
import math

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step's residual addition and norm before a projection, full batch of the headline workload
        dict(name="norm decode r64 h4096", op="norm", rows=64, hidden=4096, plus_one=False),
        # the same of a long prefill, Gemma-2-9B width, (1 + w) norm; an odd number of tokens
        dict(name="norm prefill r16001 h3584", op="norm", rows=16001, hidden=3584, plus_one=True),
        # the MLP's activation of a small batch, Qwen3-8B
        dict(name="gated decode r5 i12288", op="gated", rows=5, inter=12288, act="silu"),
        # the same of a prefill of Gemma-2-9B
        dict(name="gated prefill r8192 i14336", op="gated", rows=8192, inter=14336, act="gelu"),
        # a loader turns a matrix into 4 bits: o_proj, and gate and up together, Qwen3-8B
        dict(name="quantise n4096 k4096 g128", op="quantise", n=4096, k=4096, group=128),
        dict(name="quantise n24576 k4096 g64", op="quantise", n=24576, k=4096, group=64),
        # one sequence: q of Qwen3-0.6B (the smallest product: latency)
        dict(name="linear bf16 m1 n2048 k1024", op="linear", rows=1, n=2048, k=1024, group=128, q8=False),
        # one sequence with two drafted tokens: down_proj of Qwen3-8B
        dict(name="linear q8 m3 n4096 k12288", op="linear", rows=3, n=4096, k=12288, group=128, q8=True),
        # one sequence: the vocabulary's logits
        dict(name="linear bf16 m1 n151936 k4096", op="linear", rows=1, n=151936, k=4096, group=128, q8=False),
        # the headline batch: gate and up of Qwen3-8B, both types of rows
        dict(name="linear bf16 m64 n24576 k4096", op="linear", rows=64, n=24576, k=4096, group=64, q8=False),
        dict(name="linear q8 m64 n24576 k4096", op="linear", rows=64, n=24576, k=4096, group=128, q8=True),
        # a prefill chunk: q, k and v of Qwen3-8B
        dict(name="linear q8 m2048 n6144 k4096", op="linear", rows=2048, n=6144, k=4096, group=128, q8=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["norm", "gated", "quantise", "linear", "linear", "linear", "linear"])
    if op == "norm":
        rows = _log(rng, 1, 16384)
        return dict(op=op, rows=rows, hidden=_log(rng, 64, min(16384, 16000 * 3584 // rows)), plus_one=rng.random() < 0.3)
    if op == "gated":
        rows = _log(rng, 1, 16384)
        return dict(op=op, rows=rows, inter=_log(rng, 64, min(32768, 8192 * 14336 // rows)),
                    act=rng.choice(["silu", "gelu"]))
    group = rng.choice([32, 64, 128, 128])
    k = 32 * _log(rng, 1, 512)
    if op == "quantise":
        return dict(op=op, n=_log(rng, 1, min(65536, 24576 * 4096 // k)), k=k, group=group)
    rows = _log(rng, 1, 64) if rng.random() < 0.7 else _log(rng, 64, 4096)
    n = _log(rng, 1, min(65536, 24576 * 4096 // k, 2048 * 6144 * 4096 // (rows * k)))
    return dict(op=op, rows=rows, n=n, k=k, group=group, q8=rng.random() < 0.5)


# ----------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rows(g, rows, width):
    """Activations: rows of different sizes, a few channels of several times the others'."""
    wide = 1 + 7 * (torch.rand(width, generator=g, device=DEV) > 0.99).float()
    size = torch.exp(0.5 * _normal(g, rows, 1))
    return (_normal(g, rows, width) * wide * size).bfloat16()


def _records(codes, scales, zeros, group):
    """Codes [N, K] and zeros [N, G] (uint8) and scales [N, G] (bf16) in the layout of the records."""
    n, k = codes.shape
    tiles, blocks = (n + 15) // 16, (k + 127) // 128
    per = 128 // group
    full = codes.new_zeros(tiles * 16, blocks * 128)
    full[:n, :k] = codes
    word = full.view(tiles, 16, blocks, 4, 4, 8)[..., [0, 2, 4, 6, 1, 3, 5, 7]].unflatten(-1, (4, 2))
    word = (word[..., 0] | (word[..., 1] << 4)).permute(0, 2, 1, 4, 3, 5)  # [tiles, blocks, 16, t, i, 4]
    row = torch.arange(16, device=DEV)[:, None]
    place = torch.arange(4, device=DEV)[None] ^ (row // 2 % 4)
    out = codes.new_zeros(tiles, blocks, 1024 + 64 * per)
    out[..., :1024] = word[:, :, row, place].flatten(2)
    del full, word
    pairs = torch.zeros(tiles * 16, blocks * per, 2, dtype=torch.int16, device=DEV)
    pairs[:n, :scales.shape[1], 0] = scales.view(torch.int16)
    pairs[:n, :scales.shape[1], 1] = zeros.to(torch.int16) + 0x4300  # the bits of 128 + zero
    pairs = pairs.view(tiles, 16, blocks, per, 2).transpose(1, 2).contiguous()
    out[..., 1024:] = pairs.view(torch.uint8).flatten(2)
    head = tiles // 8 * 8
    return torch.cat([out[:head].unflatten(0, (-1, 8)).transpose(1, 2).flatten(0, 2), out[head:].transpose(0, 1).flatten(0, 1)])


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["op"] == "norm":
        x, res = _rows(g, c["rows"], c["hidden"]), _rows(g, c["rows"], c["hidden"])
        w = 0.2 * _normal(g, c["hidden"])
        return dict(c, x=x, res=res, w=(w if c["plus_one"] else 1 + w).bfloat16(), eps=1e-6, total=torch.empty_like(res))
    if c["op"] == "gated":
        return dict(c, x=_rows(g, c["rows"], 2 * c["inter"]))
    n, k, group = c["n"], c["k"], c["group"]
    groups = (k + group - 1) // group
    if c["op"] == "quantise":
        size = torch.exp(0.3 * _normal(g, n, 1))
        return dict(c, w=(0.02 * _normal(g, n, k) * size).bfloat16())
    codes = torch.empty(n, k, dtype=torch.uint8, device=DEV)
    for lo in range(0, n, 16384):
        part = codes[lo:lo + 16384]
        part.copy_((7.5 + 2.6 * _normal(g, *part.shape)).round().clamp(0, 15))
    scales = (0.02 * torch.exp(0.3 * _normal(g, n, groups))).bfloat16()
    zeros = (7.5 + 0.8 * _normal(g, n, groups)).round().clamp(0, 15).to(torch.uint8)
    s = dict(c, records=_records(codes, scales, zeros, group))
    x = _rows(g, c["rows"], k)
    if not c["q8"]:
        return dict(s, x=x)
    amax = x.float().abs().amax(-1)
    return dict(s, x=(x.float() * 127 / amax[:, None]).round().to(torch.int8), a=amax / 127)


# ------------------------------------------------------------------------------------ plain forms
def _weights(records, n, k, group):
    """What the records stand for, in 32 bits: [N, K]."""
    tiles, blocks, per = (n + 15) // 16, (k + 127) // 128, 128 // group
    head, size = tiles // 8 * 8, records.shape[1]
    r = torch.cat([records[:head * blocks].view(head // 8, blocks, 8, size).transpose(1, 2).flatten(0, 1),
                   records[head * blocks:].view(blocks, tiles - head, size).transpose(0, 1)])
    row = torch.arange(16, device=DEV)[:, None]
    place = torch.arange(4, device=DEV)[None] ^ (row // 2 % 4)
    word = r[..., :1024].view(tiles, blocks, 16, 4, 4, 4)[:, :, row, place].permute(0, 2, 1, 4, 3, 5)
    u = torch.stack([word & 15, word >> 4], -1).flatten(-2)[..., [0, 4, 1, 5, 2, 6, 3, 7]]
    u = u.reshape(tiles * 16, blocks * per, group)
    p = r[..., 1024:].reshape(tiles, blocks, 16, per, 4).transpose(1, 2).contiguous()
    p = p.view(torch.bfloat16).float().reshape(tiles * 16, blocks * per, 2)
    return (p[..., :1] * (u.float() - (p[..., 1:] - 128).clamp_min(0))).flatten(1)[:n, :k]


def _quantised(w, group):
    """Codes, scales and zeros of w [N, K]; K is filled up with zeros, which change no group."""
    n, k = w.shape
    groups = (k + group - 1) // group
    x = torch.nn.functional.pad(w.float(), (0, groups * group - k)).view(n, groups, group)
    low = x.amin(-1).clamp_max(0)
    scale = ((x.amax(-1).clamp_min(0) - low) / 15).bfloat16()
    s = torch.where(scale > 0, scale.float(), 1.0)
    zero = (-low / s).round().clamp(0, 15)
    u = ((x / s[..., None]).round() + zero[..., None]).clamp(0, 15)
    return u.flatten(1)[:, :k].to(torch.uint8), scale, zero.to(torch.uint8)


def _as_q8(y):
    """Rows y (32 bits) in codes of 8 bits: the codes, and what 127 stands for."""
    amax = y.abs().amax(-1, keepdim=True)
    return (y * 127 / torch.where(amax > 0, amax, 1.0)).round(), amax


def _plain(s):
    if s["op"] == "norm":
        h = (s["res"].float() + s["x"].float()).bfloat16()
        f = h.float()
        codes, amax = _as_q8(f * (1 + s["w"].float() if s["plus_one"] else s["w"].float()))
        scale = amax * torch.rsqrt((f * f).mean(-1, keepdim=True) + s["eps"]) / 127
        return [(codes * scale).bfloat16(), h]
    if s["op"] == "gated":
        gate, up = s["x"].float().chunk(2, -1)
        if s["act"] == "silu":
            y = gate / (1 + torch.exp(-gate)) * up
        else:
            y = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3))) * up
        codes, amax = _as_q8(y)
        return (codes * (amax / 127)).bfloat16()
    n, k, group = s["n"], s["k"], s["group"]
    if s["op"] == "quantise":
        records = _records(*_quantised(s["w"], group), group)
        return _weights(records, n, k, group).bfloat16()
    y = s["x"].float() @ _weights(s["records"], n, k, group).T
    return (y * s["a"][:, None] if s["q8"] else y).bfloat16()


# -------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        from llm_pytorch_inference_b200 import ops

        if s["op"] == "norm":
            rows, total = ops.fused_add_rmsnorm_q8(s["res"], s["x"], s["w"], s["eps"], plus_one=s["plus_one"],
                                                   residual_out=s["total"])
            return [ops.dequantise_q8(rows), total]
        if s["op"] == "gated":
            gate, up = s["x"].chunk(2, -1)
            return ops.dequantise_q8((ops.swiglu_q8 if s["act"] == "silu" else ops.geglu_q8)(gate, up))
        if s["op"] == "quantise":
            return ops.dequantise_w4(ops.quantise_w4(s["w"], s["group"]))
        w = ops.W4Weight(s["records"], s["n"], s["k"], s["group"])
        return ops.linear_w4(ops.Q8Rows(s["x"], s["a"]) if s["q8"] else s["x"], w)
    return _plain(s)


def work(case):
    c = case
    if c["op"] == "norm":
        n = c["rows"] * c["hidden"]
        # both inputs, the sum and the codes; the codes once more and the values that they stand for
        return {"bytes": n * (2 + 2 + 2 + 1) + n * (1 + 2) + 2 * c["hidden"] + 8 * c["rows"], "flops": 8 * n}
    if c["op"] == "gated":
        n = c["rows"] * c["inter"]
        return {"bytes": n * (4 + 1) + n * (1 + 2) + 8 * c["rows"], "flops": 12 * n}
    n, k = c["n"], c["k"]
    held = n * k / 2 + n * ((k + c["group"] - 1) // c["group"]) * 2.5  # codes; a scale and a zero per group
    if c["op"] == "quantise":
        return {"bytes": 2 * n * k + 2 * held + 2 * n * k, "flops": 6 * n * k}
    x = c["rows"] * (k + 4 if c["q8"] else 2 * k)
    return {"bytes": held + x + 2 * c["rows"] * n, "flops": 2 * c["rows"] * n * k}


# ------------------------------------------------------------------------------- 64-bit reference
def _exact_part(records, rows, n, k, group):
    """Rows `rows` of the matrix in 64 bits, each weight looked up by its byte."""
    width, blocks = records.shape[1], (k + 127) // 128
    tile, col = rows // 16, torch.arange(k, device=DEV)
    together = torch.clamp((n + 15) // 16 - tile // 8 * 8, max=8)  # records that stand with this one
    first = tile // 8 * 8 * blocks + tile % 8
    at = (first[:, None] + col // 128 * together[:, None]) * width  # byte of the record
    r, flat = (rows % 16)[:, None], records.reshape(-1)
    place = col % 32 // 8 ^ torch.div(r, 2, rounding_mode="floor") % 4
    nibble = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7], device=DEV)[col % 8]
    u = flat[at + 64 * r + 16 * place + 4 * (col % 128 // 32) + nibble // 2].int()
    u = torch.where(nibble % 2 == 1, u // 16, u % 16)
    pair = at + 1024 + 512 // group * r + 4 * (col % 128 // group)
    scale = ((flat[pair].int() << 16) + (flat[pair + 1].int() << 24)).view(torch.float32).double()
    return scale * (u - flat[pair + 2].int() % 128).double()


def _exact_rows(y):
    """What the 8-bit form of rows y (64 bits) stands for."""
    top = y.abs().max(-1, keepdim=True).values
    return torch.round(y / torch.where(top > 0, top, 1.0) * 127) * top / 127


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = (s["res"].double() + s["x"].double()).to(torch.bfloat16)
        w = s["w"].double() + (1.0 if case["plus_one"] else 0.0)
        r = 1 / torch.sqrt(h.double().square().sum(-1, keepdim=True) / case["hidden"] + s["eps"])
        return [_exact_rows(h.double() * w) * r, h.double()]
    if case["op"] == "gated":
        inter = case["inter"]
        a, b = s["x"][:, :inter].double(), s["x"][:, inter:].double()
        if case["act"] == "silu":
            return _exact_rows(a * torch.sigmoid(a) * b)
        return _exact_rows(a * b * torch.sigmoid((8 / math.pi) ** 0.5 * a * (1 + 0.044715 * a * a)))  # tanh's form
    n, k, group = case["n"], case["k"], case["group"]
    if case["op"] == "quantise":
        out = torch.zeros(n, k, dtype=torch.float64, device=DEV)
        for lo in range(0, k, group):
            w = s["w"][:, lo:lo + group].double()
            low, high = w.min(-1, keepdim=True).values.clamp(max=0), w.max(-1, keepdim=True).values.clamp(min=0)
            step = ((high - low) / 15).to(torch.bfloat16).double()
            safe = torch.where(step > 0, step, 1.0)
            zero = torch.round(-low / safe).clamp(0, 15)
            out[:, lo:lo + group] = step * (torch.clamp(torch.round(w / safe) + zero, 0, 15) - zero)
        return out
    x = s["x"].double() * (s["a"].double()[:, None] if case["q8"] else 1.0)
    out = torch.empty(case["rows"], n, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 25) // k)
    for lo in range(0, n, step):
        rows = torch.arange(lo, min(lo + step, n), device=DEV)
        out[:, lo:lo + step] = x @ _exact_part(s["records"], rows, n, k, group).T
    return out
