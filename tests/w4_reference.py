"""Plain 64-bit forms of the 8-bit rows and the 4-bit weights, element by element from their definitions."""
import math

import torch


# ------------------------------------------------------------------------------- rows in 8 bits
def q8(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Exact quotients 127 y / amax and scales amax / 127 of rows y (64 bits)."""
    amax = y.abs().amax(-1, keepdim=True)
    return 127 * y / torch.where(amax > 0, amax, 1.0), (amax / 127).squeeze(-1)


def normed(h: torch.Tensor, w: torch.Tensor, eps: float, plus_one: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """h w, and 1 / sqrt(mean(h^2) + eps), of h and w in 64 bits."""
    r = 1 / torch.sqrt(h.square().mean(-1) + eps)
    return h * (1 + w if plus_one else w), r


def gated(gate: torch.Tensor, up: torch.Tensor, gelu: bool) -> torch.Tensor:
    z = gate * (1 + 0.044715 * gate.square()) * math.sqrt(8 / math.pi) if gelu else gate
    return gate * torch.sigmoid(z) * up


# ----------------------------------------------------------------------------- weights in 4 bits
def quantise(w: torch.Tensor, group: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Codes [n, k], scales and zeros [n, groups] of w (bf16), the numbers in 64 bits."""
    n, k = w.shape
    codes, scales, zeros = torch.zeros(n, k, dtype=torch.long), [], []
    for lo in range(0, k, group):
        x = w[:, lo:lo + group].double().cpu()
        low, high = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
        step = ((high - low).float() / 15).to(torch.bfloat16).double()
        safe = torch.where(step > 0, step, 1.0)
        zero = (-low / safe).round().clamp(0, 15)
        codes[:, lo:lo + group] = ((x / safe[:, None]).round() + zero[:, None]).clamp(0, 15).long()
        scales.append(step)
        zeros.append(zero.long())
    return codes, torch.stack(scales, -1), torch.stack(zeros, -1)


def record_bytes(group: int) -> int:
    return 1024 + 16 * (128 // group) * 4


def place(row: int, col: int, n: int, k: int, group: int) -> tuple[int, int, int]:
    """Byte and nibble of the code of (row, col), and the byte of its group's word."""
    tile, block, tiles = row // 16, col // 128, -(-n // 16)
    first = tile // 8 * 8
    at = (first * -(-k // 128) + block * min(8, tiles - first) + tile - first) * record_bytes(group)
    r, c = row % 16, col % 128
    nibble = (0, 4, 1, 5, 2, 6, 3, 7)[c % 8]
    code = at + 64 * r + 16 * ((c % 32 // 8) ^ (r // 2 % 4)) + 4 * (c // 32) + nibble // 2
    return code, nibble % 2, at + 1024 + (r * (128 // group) + c // group) * 4


def unpack(records: torch.Tensor, n: int, k: int, group: int):
    """Codes, scales and zeros that records hold (on the CPU)."""
    flat = records.cpu().flatten()
    rows, cols = torch.meshgrid(torch.arange(n), torch.arange(k), indexing="ij")
    tile, block, tiles = rows // 16, cols // 128, -(-n // 16)
    first = tile // 8 * 8
    at = (first * -(-k // 128) + block * torch.clamp(tiles - first, max=8) + tile - first) * record_bytes(group)
    r, c = rows % 16, cols % 128
    nibble = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7])[c % 8]
    byte = flat[at + 64 * r + 16 * ((c % 32 // 8) ^ (r // 2 % 4)) + 4 * (c // 32) + nibble // 2].long()
    codes = torch.where(nibble % 2 == 1, byte >> 4, byte & 15)
    word = (at + 1024 + (r * (128 // group) + c // group) * 4)[:, ::group]
    half = flat[word].long() | flat[word + 1].long() << 8
    scales = (half.int() << 16).view(torch.float32).double()
    return codes, scales, flat[word + 2].long() & 15


def values(codes, scales, zeros, group: int) -> torch.Tensor:
    """What they stand for, in 64 bits."""
    of = torch.arange(codes.shape[1]) // group
    return scales[:, of] * (codes - zeros[:, of]).double()


def linear_bound(x: torch.Tensor, w: torch.Tensor, group: int, exact: torch.Tensor) -> torch.Tensor:
    """How far a product of x [m, k] and w [n, k] (64 bits) may be off: rounded once to bf16; its sums held in 32 bits,
    at most one unit of 2^-23 of all that is added for each of a group's products and each group; and elements of x
    held to 2^-20 of the largest of their group."""
    k = x.shape[1]
    size = x.abs() @ w.abs().T
    held = torch.zeros_like(size)
    for lo in range(0, k, group):
        held += x[:, lo:lo + group].abs().amax(-1, keepdim=True) * w[:, lo:lo + group].abs().sum(-1)
    return 2.0 ** -8 * exact.abs() * 1.001 + (min(group, k) + -(-k // group)) * 2.0 ** -23 * size + 2.0 ** -20 * held
