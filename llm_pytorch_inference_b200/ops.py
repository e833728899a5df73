"""Drop-in mirror of the reference's ``mini_vllm.ops`` API on the sm_100a kernels.

Same function / class names, argument meaning and return conventions as
``mini_vllm/ops/__init__.py:1-51``; every call goes through the C ABI of
``libmvb200.so``.  There is no CPU path: a CPU tensor raises ``RuntimeError``
(the reference would fall back to PyTorch, ``mini_vllm/ops/_utils.py:70-78``).

Numerics match the reference's PyTorch expressions (see the per-function notes);
the one deliberate difference is ``apply_rotary_pos_emb``, which broadcasts cos/sin
per sequence for K as well as Q (the reference's CUDA branch expands cos to Q's
shape and indexes it with K's rows, ``mini_vllm/ops/rope.py:59-70``).
"""
from __future__ import annotations

import functools
import threading
from typing import NamedTuple

import torch
import torch.nn as nn
from torch.nn.parameter import Parameter

from . import _native as N

__all__ = [
    "rmsnorm", "rmsnorm_plus_one", "fused_add_rmsnorm", "fused_add_rmsnorm_plus_one", "RMSNorm",
    "precompute_freqs_cis", "rotate_half", "apply_rotary_pos_emb", "silu", "gelu", "swiglu", "geglu",
    "greedy_sample", "top_k_top_p_filter", "softmax_multinomial_sample", "embedding", "Embedding", "softmax",
    "FusedMLP", "linear", "paged_attention_decode", "qk_norm_rope_kv_write", "sample", "kv4_write", "kv4_read",
    "paged_attention_decode_kv4", "assign_slots", "SlotPlan", "verify_drafts", "Q8Rows", "quantise_q8",
    "dequantise_q8", "rmsnorm_q8", "fused_add_rmsnorm_q8", "swiglu_q8", "geglu_q8", "W4Weight", "quantise_w4",
    "pack_w4", "dequantise_w4", "linear_w4", "FusedMLPW4",
]


def _st(t: torch.Tensor) -> int:
    return N.stream_handle(t.device)


def _w(weight: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    w = weight if weight.dtype == like.dtype else weight.to(like.dtype)
    return w.contiguous()


# ----------------------------------------------------------------------- RMSNorm
def _rms(x, weight, eps, plus_one, semantics):
    N.require_cuda(x, weight)
    w = _w(weight, x)
    xc = x.contiguous()
    out = torch.empty_like(xc)
    H = xc.shape[-1]
    rows = xc.numel() // H if H else 0
    with torch.cuda.device(xc.device):
        N.check(N.lib().mvb_rmsnorm(out.data_ptr(), H, xc.data_ptr(), H, w.data_ptr(), rows, H, float(eps),
                                    int(plus_one), semantics, N.dtype_code(xc), _st(xc)), "rmsnorm")
    return out


def rmsnorm(input: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``ops/rmsnorm.py:12-20``: ``(w * x * rsqrt(mean(x^2) + eps))`` in the input dtype."""
    return _rms(input, weight, eps, False, N.NORM_OPS)


def rmsnorm_plus_one(input: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``ops/rmsnorm.py:23-31``: ``(1 + w) * x * rsqrt(...)``."""
    return _rms(input, weight, eps, True, N.NORM_OPS)


def _fused(residual, input, weight, eps, plus_one):
    N.require_cuda(residual, input, weight)
    if not residual.is_contiguous() or not input.is_contiguous():
        raise RuntimeError("fused_add_rmsnorm: residual and input must be contiguous")
    if residual.shape != input.shape or residual.dtype != input.dtype:
        raise RuntimeError("fused_add_rmsnorm: residual and input must match in shape and dtype")
    w = _w(weight, input)
    out = torch.empty_like(input)
    H = input.shape[-1]
    with torch.cuda.device(input.device):
        N.check(N.lib().mvb_fused_add_rmsnorm(out.data_ptr(), residual.data_ptr(), input.data_ptr(), w.data_ptr(),
                                              input.numel() // H, H, float(eps), int(plus_one), N.NORM_OPS,
                                              N.dtype_code(input), _st(input)), "fused_add_rmsnorm")
    return out, residual


def fused_add_rmsnorm(residual: torch.Tensor, input: torch.Tensor, weight: torch.Tensor,
                      eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """``ops/rmsnorm.py:34-42``: ``residual += input`` (in place), returns ``(norm(residual), residual)``."""
    return _fused(residual, input, weight, eps, False)


def fused_add_rmsnorm_plus_one(residual: torch.Tensor, input: torch.Tensor, weight: torch.Tensor,
                               eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """``ops/rmsnorm.py:45-53``."""
    return _fused(residual, input, weight, eps, True)


class RMSNorm(nn.Module):
    """``ops/rmsnorm.py:60-76``: weight init ones (or zeros for the (1+w) form)."""

    def __init__(self, hidden_size: int, eps: float = 1e-6, plus_one: bool = False):
        super().__init__()
        self.weight = Parameter(torch.zeros(hidden_size) if plus_one else torch.ones(hidden_size))
        self.eps = eps
        self.plus_one = plus_one

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return rmsnorm_plus_one(x, self.weight, self.eps) if self.plus_one else rmsnorm(x, self.weight, self.eps)


# --------------------------------------------------------------------------- RoPE
def precompute_freqs_cis(dim: int, seq_len: int, theta: float = 10000.0, device="cpu",
                         dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """Table construction as ``ops/rope.py:15-37`` (host-side set-up, not a decode kernel)."""
    freqs = 1.0 / (theta ** (torch.arange(0, dim, 2, device=device, dtype=dtype) / dim))
    t = torch.arange(seq_len, device=device, dtype=dtype)
    emb = torch.cat((torch.outer(t, freqs),) * 2, dim=-1)
    return emb.cos(), emb.sin()


def rotate_half(x: torch.Tensor) -> torch.Tensor:
    """``ops/rope.py:40-44`` (tensor utility)."""
    h = x.shape[-1] // 2
    return torch.cat((-x[..., h:], x[..., :h]), dim=-1)


def _rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    D = x.shape[-1]
    c = cos.expand_as(x).reshape(-1, D).contiguous().to(x.dtype)
    s = sin.expand_as(x).reshape(-1, D).contiguous().to(x.dtype)
    xf = x.reshape(-1, D).contiguous()
    out = torch.empty_like(xf)
    with torch.cuda.device(x.device):
        N.check(N.lib().mvb_rotary_pos_emb(out.data_ptr(), xf.data_ptr(), c.data_ptr(), s.data_ptr(), xf.shape[0], D,
                                           N.dtype_code(xf), _st(xf)), "rotary_pos_emb")
    return out.reshape(x.shape)


def apply_rotary_pos_emb(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor,
                         sin: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``ops/rope.py:47-77``: ``x*cos + rotate_half(x)*sin`` for q ``[B,Hq,S,D]`` and k ``[B,Hkv,S,D]``
    with cos/sin broadcastable ``[B,1,S,D]``; each product and the sum round to the dtype."""
    N.require_cuda(q, k, cos, sin)
    return _rope(q, cos, sin), _rope(k, cos, sin)


# -------------------------------------------------------------------- activations
def _act(x, act):
    N.require_cuda(x)
    xc = x.contiguous()
    out = torch.empty_like(xc)
    with torch.cuda.device(xc.device):
        N.check(N.lib().mvb_activation(out.data_ptr(), xc.data_ptr(), xc.numel(), act, N.dtype_code(xc), _st(xc)),
                "activation")
    return out


def _gated(g, u, act):
    N.require_cuda(g, u)
    if g.shape != u.shape:
        raise RuntimeError("gate and up must have the same shape")
    gc, uc = g.contiguous(), u.contiguous().to(g.dtype)
    out = torch.empty_like(gc)
    with torch.cuda.device(gc.device):
        N.check(N.lib().mvb_gated_activation(out.data_ptr(), gc.data_ptr(), uc.data_ptr(), gc.numel(), act,
                                             N.dtype_code(gc), _st(gc)), "gated_activation")
    return out


def silu(input: torch.Tensor) -> torch.Tensor:
    """``ops/activation.py:10-19``."""
    return _act(input, N.ACT_SILU)


def gelu(input: torch.Tensor) -> torch.Tensor:
    """``ops/activation.py:22-31`` (tanh approximation)."""
    return _act(input, N.ACT_GELU_TANH)


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``ops/activation.py:34-48``: ``silu(gate) * up``."""
    return _gated(gate, up, N.ACT_SILU)


def geglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``ops/activation.py:51-66``: ``gelu(gate) * up``."""
    return _gated(gate, up, N.ACT_GELU_TANH)


# ------------------------------------------------------------------------ sampling
def greedy_sample(logits: torch.Tensor) -> torch.Tensor:
    """``ops/sampling.py:10-21``: row argmax (lowest index among ties), int64 ``[B]``."""
    N.require_cuda(logits)
    x = logits.contiguous()
    V = x.shape[-1]
    rows = x.numel() // V
    out = torch.empty(rows, dtype=torch.int64, device=x.device)
    with torch.cuda.device(x.device):
        N.check(N.lib().mvb_greedy_sample(out.data_ptr(), x.data_ptr(), rows, V, V, N.dtype_code(x), _st(x)),
                "greedy_sample")
    return out


def top_k_top_p_filter(logits: torch.Tensor, top_k: int = 0, top_p: float = 1.0) -> torch.Tensor:
    """``ops/sampling.py:24-50``: filtered copy, non-survivors ``-inf`` (untempered logits).
    Among logits tied at the top-p cutoff the lower indices survive."""
    N.require_cuda(logits)
    x = logits.clone().contiguous()
    V = x.shape[-1]
    with torch.cuda.device(x.device):
        N.check(N.lib().mvb_top_k_top_p_filter(x.data_ptr(), x.numel() // V, V, int(top_k), float(top_p),
                                               N.dtype_code(x), _st(x)), "top_k_top_p_filter")
    return x


_rng_lock = threading.Lock()
_rng_fallback = [0]


def _next_seed_offset(device: torch.device, rows: int) -> tuple[int, int]:
    """(seed, offset) from torch's default CUDA generator, advanced like a draw of ``rows`` values."""
    gen = torch.cuda.default_generators[device.index if device.index is not None else torch.cuda.current_device()]
    seed = int(gen.initial_seed())
    with _rng_lock:
        if hasattr(gen, "get_offset"):
            off = int(gen.get_offset())
            gen.set_offset(off + 4 * ((rows + 3) // 4 + 1))
        else:
            off = _rng_fallback[0]
            _rng_fallback[0] += 1
    return seed, off


def softmax_multinomial_sample(logits: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """``ops/sampling.py:53-73``: ``softmax(logits / T)`` and one draw per row (int64 ``[B]``).
    The draw is a Philox4x32-10 inverse CDF seeded from torch's CUDA generator state."""
    N.require_cuda(logits)
    x = logits.contiguous()
    V = x.shape[-1]
    rows = x.numel() // V
    out = torch.empty(rows, dtype=torch.int64, device=x.device)
    seed, off = _next_seed_offset(x.device, rows)
    with torch.cuda.device(x.device):
        N.check(N.lib().mvb_softmax_multinomial_sample(out.data_ptr(), x.data_ptr(), rows, V, float(temperature),
                                                       seed, off, N.dtype_code(x), _st(x)),
                "softmax_multinomial_sample")
    return out


def sample(logits: torch.Tensor, temperature: torch.Tensor | float, top_k: torch.Tensor | int,
           top_p: torch.Tensor | float, seed: int, offset: int, probs_out: torch.Tensor | None = None,
           out: torch.Tensor | None = None, offset_dev: torch.Tensor | None = None) -> torch.Tensor:
    """Fused per-row sampler (greedy if T == 0, else top-k, top-p, /T, softmax, Philox draw).
    Per-row parameters may be CUDA tensors (fp32 / int32 / fp32 of length B) or scalars."""
    N.require_cuda(logits)
    x = logits if logits.stride(-1) == 1 else logits.contiguous()
    V = x.shape[-1]
    rows = x.numel() // V
    dev = x.device

    def vec(v, dt):
        if isinstance(v, torch.Tensor):
            return v.to(device=dev, dtype=dt).contiguous()
        return torch.full((rows,), v, dtype=dt, device=dev)

    t, k, p = vec(temperature, torch.float32), vec(top_k, torch.int32), vec(top_p, torch.float32)
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        N.check(N.lib().mvb_sample(out.data_ptr(), N.ptr(probs_out), x.data_ptr(), rows, V, x.stride(-2) if x.dim() > 1
                                   else V, t.data_ptr(), k.data_ptr(), p.data_ptr(), int(seed), int(offset),
                                   N.ptr(offset_dev), N.dtype_code(x), _st(x)), "sample")
    return out


# ------------------------------------------------------------- embedding / softmax
def embedding(input_ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``ops/embedding.py:11-35``: ``W[ids] * scale``; output shape ``ids.shape + [H]``."""
    N.require_cuda(input_ids, weight)
    ids = input_ids.reshape(-1).contiguous()
    if ids.dtype not in (torch.int32, torch.int64):
        ids = ids.to(torch.int64)
    w = weight.contiguous()
    V, H = w.shape
    out = torch.empty(ids.numel(), H, dtype=w.dtype, device=w.device)
    with torch.cuda.device(w.device):
        N.check(N.lib().mvb_embedding(out.data_ptr(), ids.data_ptr(), N.dtype_code(ids), w.data_ptr(), ids.numel(), H,
                                      V, float(scale), N.dtype_code(w), _st(w)), "embedding")
    return out.reshape(*input_ids.shape, H) if input_ids.dim() > 1 else out


class Embedding(nn.Module):
    """``ops/embedding.py:38-50``."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0):
        super().__init__()
        self.weight = Parameter(torch.empty(num_embeddings, embedding_dim))
        self.scale = scale
        nn.init.normal_(self.weight, mean=0.0, std=0.02)

    def forward(self, input_ids: torch.Tensor) -> torch.Tensor:
        return embedding(input_ids, self.weight, self.scale)


def softmax(input: torch.Tensor, dim: int = -1) -> torch.Tensor:
    """``ops/softmax.py:5-25``: last-dim softmax in fp32, one rounding to the input dtype."""
    if dim != -1 and dim != input.dim() - 1:
        raise RuntimeError("softmax: only the last dimension is implemented by the kernel")
    N.require_cuda(input)
    x = input.contiguous()
    out = torch.empty_like(x)
    n = x.shape[-1]
    with torch.cuda.device(x.device):
        N.check(N.lib().mvb_softmax(out.data_ptr(), x.data_ptr(), x.numel() // n, n, N.dtype_code(x), _st(x)),
                "softmax")
    return out


# ----------------------------------------------------------------------- GEMM / MLP
class _Workspaces:
    """Zero-initialised scratch per device for the stream-K GEMM and split-KV attention.
    The kernels leave their counters at zero, so a buffer is reusable call after call
    on one stream (concurrent calls on different streams need separate buffers)."""

    def __init__(self):
        self._buf: dict[tuple[int, str], torch.Tensor] = {}
        self._lock = threading.Lock()

    def get(self, device: torch.device, kind: str, nbytes: int) -> torch.Tensor:
        key = (device.index if device.index is not None else torch.cuda.current_device(), kind)
        with self._lock:
            b = self._buf.get(key)
            if b is None or b.numel() < nbytes:
                b = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
                self._buf[key] = b
            return b


WORKSPACES = _Workspaces()


def linear(x: torch.Tensor, weight: torch.Tensor, epilogue: int = N.EPI_STORE, aux: torch.Tensor | None = None,
           out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``y = x @ weight.T`` (bf16, tcgen05).  ``epilogue``: EPI_STORE, EPI_SWIGLU (weight =
    cat([gate, up]); y = silu(gate) * up) or EPI_RESADD (y = aux + x @ W.T)."""
    N.require_cuda(x, weight)
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise RuntimeError("linear: the tcgen05 GEMM takes bf16 operands")
    K = x.shape[-1]
    xf = x.reshape(-1, K)
    if xf.stride(-1) != 1:
        xf = xf.contiguous()
    w = weight if weight.stride(-1) == 1 else weight.contiguous()
    Nn = w.shape[0]
    M = xf.shape[0]
    cols = Nn // 2 if epilogue == N.EPI_SWIGLU else Nn
    if out is None:
        out = torch.empty(M, cols, dtype=torch.bfloat16, device=x.device)
    auxf = None if aux is None else aux.reshape(-1, cols)
    dev = x.device
    with torch.cuda.device(dev):
        # + a fixed 1 MiB counter reserve: shapes sharing the cached buffer keep their partials
        # clear of every other shape's counters (up to 256K output tiles)
        need = N.lib().mvb_gemm_workspace_bytes(M, Nn, K, dev.index if dev.index is not None else 0) + (1 << 20)
        ws = workspace if workspace is not None else WORKSPACES.get(dev, "gemm", need)
        N.check(N.lib().mvb_gemm_bf16(out.data_ptr(), out.stride(0), xf.data_ptr(), xf.stride(0), w.data_ptr(),
                                      w.stride(0), M, Nn, K, epilogue, None if auxf is None else auxf.data_ptr(),
                                      0 if auxf is None else auxf.stride(0), ws.data_ptr(), ws.numel(), _st(x)),
                "gemm_bf16")
    return out.reshape(*x.shape[:-1], cols)


_ACT_CODE = {"silu": 0, "gelu": 1, "gelu_new": 1}   # ops/mlp.py:9-13


class FusedMLP(nn.Module):
    """``ops/mlp.py:46-84``: gate_up GEMM -> act(gate) * up -> down GEMM.

    For SiLU the activation runs in the gate_up GEMM's epilogue (one kernel); GELU uses
    the standalone fused_mlp kernel between the two GEMMs."""

    def __init__(self, hidden_size: int, intermediate_size: int, hidden_act: str = "silu"):
        super().__init__()
        self.gate_up_proj = nn.Linear(hidden_size, 2 * intermediate_size, bias=False)
        self.down_proj = nn.Linear(intermediate_size, hidden_size, bias=False)
        self.intermediate_size = intermediate_size
        self.hidden_act = hidden_act
        if hidden_act not in _ACT_CODE:
            raise ValueError(f"unsupported activation {hidden_act!r}")
        self._act_code = _ACT_CODE[hidden_act]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self._act_code == 0:
            h = linear(x, self.gate_up_proj.weight, N.EPI_SWIGLU)
        else:
            gu = linear(x, self.gate_up_proj.weight)
            h = fused_mlp_forward(gu, self.intermediate_size, self._act_code)
        return linear(h, self.down_proj.weight)


def fused_mlp_forward(gate_up: torch.Tensor, intermediate_size: int, activation: int) -> torch.Tensor:
    """``fused_mlp_forward`` (``mlp_kernel.cu:61-93``): ``act(gate_up[..., :I]) * gate_up[..., I:]``."""
    N.require_cuda(gate_up)
    g = gate_up.contiguous()
    rows = g.numel() // (2 * intermediate_size)
    out = torch.empty(*g.shape[:-1], intermediate_size, dtype=g.dtype, device=g.device)
    with torch.cuda.device(g.device):
        N.check(N.lib().mvb_fused_mlp(out.data_ptr(), g.data_ptr(), rows, intermediate_size, int(activation),
                                      N.dtype_code(g), _st(g)), "fused_mlp")
    return out


# ------------------------------------------------- paged decode attention / KV write
def qk_norm_rope_kv_write(qkv: torch.Tensor, kv_cache: torch.Tensor, layer: int, positions: torch.Tensor,
                          block_tables: torch.Tensor, cos_table: torch.Tensor, sin_table: torch.Tensor,
                          num_q_heads: int, num_kv_heads: int, q_norm_w: torch.Tensor | None = None,
                          k_norm_w: torch.Tensor | None = None, eps: float = 1e-6,
                          q_out: torch.Tensor | None = None, plus_one: bool = False) -> torch.Tensor:
    """Per-head QK-norm + RoPE of one new token per sequence and its K/V written into
    ``kv_cache[layer, 0|1, block_tables[b][pos // bs], pos % bs]``; returns q ``[B, Hq, D]``.
    ``plus_one`` selects Gemma's ``(1 + w)`` norm scale."""
    N.require_cuda(qkv, kv_cache, positions, block_tables, cos_table, sin_table)
    L, _, P, bs, nkv, D = kv_cache.shape
    B = qkv.shape[0]
    if q_out is None:
        q_out = torch.empty(B, num_q_heads, D, dtype=torch.bfloat16, device=qkv.device)
    with torch.cuda.device(qkv.device):
        N.check(N.lib().mvb_qk_norm_rope_kv_write(
            q_out.data_ptr(), kv_cache.data_ptr(), qkv.data_ptr(), qkv.stride(0), N.ptr(q_norm_w), N.ptr(k_norm_w),
            cos_table.data_ptr(), sin_table.data_ptr(), cos_table.shape[0], positions.data_ptr(),
            block_tables.data_ptr(), block_tables.shape[1], B, num_q_heads, num_kv_heads, D, L, layer, P, bs,
            float(eps), int(plus_one), _st(qkv)), "qk_norm_rope_kv_write")
    return q_out


def paged_attention_decode(q: torch.Tensor, kv_cache: torch.Tensor, layer: int, block_tables: torch.Tensor,
                           ctx_lens: torch.Tensor, scale: float, out: torch.Tensor | None = None,
                           workspace: torch.Tensor | None = None, softcap: float = 0.0,
                           window: int = 0) -> torch.Tensor:
    """Decode attention of q ``[B, Hq, D]`` over each sequence's first ``ctx_lens[b]`` cached
    tokens of ``layer`` (read through ``block_tables``); returns ``[B, Hq, D]``.  ``softcap`` > 0
    soft-caps the scaled scores (``softcap * tanh(s / softcap)``); ``window`` > 0 keeps only the
    newest ``window`` keys of each sequence."""
    N.require_cuda(q, kv_cache, block_tables, ctx_lens)
    L, _, P, bs, nkv, D = kv_cache.shape
    B, Hq, _ = q.shape
    if out is None:
        out = torch.empty_like(q)
    dev = q.device
    with torch.cuda.device(dev):
        need = N.lib().mvb_paged_attention_workspace_bytes(B, Hq, D, dev.index if dev.index is not None else 0) + (1 << 16)
        ws = workspace if workspace is not None else WORKSPACES.get(dev, "attention", need)
        N.check(N.lib().mvb_paged_attention_decode_ex(
            out.data_ptr(), out.stride(0), q.data_ptr(), q.stride(0), kv_cache.data_ptr(), block_tables.data_ptr(),
            block_tables.shape[1], ctx_lens.data_ptr(), B, Hq, nkv, D, L, layer, P, bs, float(scale), float(softcap),
            int(window), ws.data_ptr(), ws.numel(), _st(q)), "paged_attention_decode")
    return out


# ------------------------------------------------------------------ 4-bit paged KV cache
def _refuse(what: str, name: str, t, index: int, dtype: torch.dtype, dims: int) -> None:
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{what}: {name} must be a tensor")
    N.require_cuda(t)
    if t.get_device() != index:
        raise RuntimeError(f"{what}: {name} is on {t.device}, not on cuda:{index}")
    if t.dtype != dtype:
        raise RuntimeError(f"{what}: {name} must be {dtype}, not {t.dtype}")
    raise RuntimeError(f"{what}: {name} must have {dims} dimensions, not {t.dim()}")


def _expect(what: str, name: str, t, index: int, dtype: torch.dtype, dims: int) -> None:
    """A CUDA tensor of device ``index`` with this dtype and number of dimensions."""
    if not (isinstance(t, torch.Tensor) and t.get_device() == index and index >= 0 and t.dtype is dtype
            and t.dim() == dims):
        _refuse(what, name, t, index, dtype, dims)


def _joint(what: str, index: int, *wanted) -> None:
    """The detailed checks of ``(name, tensor, dtype, dims)`` one by one, for the caller whose joint test failed."""
    for name, t, dtype, dims in wanted:
        _expect(what, name, t, index, dtype, dims)


_I32, _I64, _F32, _BF16, _U8 = torch.int32, torch.int64, torch.float32, torch.bfloat16, torch.uint8


def _kv4_geometry(what: str, kv4: torch.Tensor, layer: int) -> tuple[int, int, int, int, int, int]:
    """(device, layers, blocks, KV heads, block size, head size) of a pool of ``kv_cache.kv4_pool``."""
    index = kv4.get_device() if isinstance(kv4, torch.Tensor) else -1
    if index < 0 or kv4.dtype is not _U8 or kv4.dim() != 5:
        _expect(what, "kv4", kv4, index, _U8, 5)
    L, P, nkv, recs, rec = kv4.shape
    if rec % 18 or not kv4.is_contiguous():
        raise RuntimeError(f"{what}: kv4 must be a contiguous pool of kv_cache.kv4_pool, not {tuple(kv4.shape)}")
    if not 0 <= layer < L:
        raise RuntimeError(f"{what}: layer {layer} of {L}")
    return index, L, P, nkv, 16 * recs, rec // 18


def _kv4_rows(t: torch.Tensor, heads: int, head_dim: int) -> tuple[torch.Tensor, int, int]:
    """``t`` [tokens, heads, D] if its rows can be read with 16-byte loads, else a copy; and the elements
    between tokens and between heads (a dimension of one has any stride, so a dense tensor's are not asked)."""
    if t.data_ptr() % 16 == 0 and not t.is_contiguous():
        s0, s1, s2 = t.stride()
        if s2 == 1 and s0 % 8 == 0 and s1 % 8 == 0:
            return t, s0, s1
    if t.data_ptr() % 16 or not t.is_contiguous():
        t = t.clone(memory_format=torch.contiguous_format)
    return t, heads * head_dim, head_dim


def kv4_write(k: torch.Tensor, v: torch.Tensor, kv4: torch.Tensor, layer: int, slots: torch.Tensor) -> None:
    """Quantises K and V ``[tokens, Hkv, D]`` (bf16, any strides) of ``layer`` to 4 bits into the slots
    ``slots`` (int64 ``[tokens]``, ``block * block_size + offset``; negative: not written) of a pool of
    ``kv_cache.kv4_pool``.  Per group of 64 channels: ``min``, ``scale = (max - min) / 15`` (both bf16) and
    ``round((x - min) / scale)``.  A group with a NaN or an infinity reads back as NaN.  The slots of one
    call must differ: what a slot given twice holds afterwards is undefined."""
    what = "kv4_write"
    index, L, P, nkv, bs, D = _kv4_geometry(what, kv4, layer)
    try:
        ok = (k.dtype is _BF16 and v.dtype is _BF16 and slots.dtype is _I64 and slots.dim() == 1
              and k.get_device() == index and v.get_device() == index and slots.get_device() == index)
    except AttributeError:
        ok = False
    if not ok:
        _joint(what, index, ("k", k, _BF16, 3), ("v", v, _BF16, 3), ("slots", slots, _I64, 1))
    n = slots.numel()
    want = (n, nkv, D)
    if k.shape != want or v.shape != want:
        raise RuntimeError(f"{what}: k and v must be {want}, not {tuple(k.shape)} and {tuple(v.shape)}")
    if n == 0:
        return
    (k, k0, k1), (v, v0, v1), slots = _kv4_rows(k, nkv, D), _kv4_rows(v, nkv, D), slots.contiguous()
    N.on_device(index, what, N.lib().mvb_kv4_write, kv4.data_ptr(), k.data_ptr(), k0, k1, v.data_ptr(), v0, v1,
                slots.data_ptr(), n, nkv, D, L, int(layer), P, bs)


def kv4_read(kv4: torch.Tensor, layer: int, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V ``[tokens, Hkv, D]`` (bf16) that the slots ``slots`` (int64) of ``layer`` stand for; zeros for
    a negative slot."""
    what = "kv4_read"
    index, L, P, nkv, bs, D = _kv4_geometry(what, kv4, layer)
    _expect(what, "slots", slots, index, torch.int64, 1)
    n = slots.numel()
    slots = slots.contiguous()
    k = torch.empty(n, nkv, D, dtype=torch.bfloat16, device=kv4.device)
    v = torch.empty_like(k)
    if n:
        N.on_device(index, what, N.lib().mvb_kv4_read, k.data_ptr(), v.data_ptr(), kv4.data_ptr(), slots.data_ptr(), n,
                    nkv, D, L, int(layer), P, bs)
    return k, v


_KV4_UNSPLIT_TOKENS = 128  # tables of at most this many tokens need no workspace: their cache is never split


@functools.lru_cache(maxsize=1024)
def _kv4_workspace_bytes(B: int, T: int, Hq: int, nkv: int, D: int, index: int) -> int:
    return N.lib().mvb_paged_attention_decode_kv4_workspace_bytes(B, T, Hq, nkv, D, index)


def paged_attention_decode_kv4(q: torch.Tensor, kv4: torch.Tensor, layer: int, block_tables: torch.Tensor,
                               ctx_lens: torch.Tensor, scale: float, out: torch.Tensor | None = None,
                               workspace: torch.Tensor | None = None, softcap: float = 0.0,
                               window: int = 0) -> torch.Tensor:
    """``paged_attention_decode`` over a 4-bit pool.  q ``[B, Hq, D]``, or ``[B, T, Hq, D]`` for the T newest
    tokens of each sequence (drafted tokens scored at once); ``ctx_lens`` counts the cached tokens, the
    query tokens among them: query i sees the first ``ctx_lens[b] - T + 1 + i`` keys, with ``window`` > 0
    the newest ``window`` of those.  A query without a key gives zeros.  Returns the shape of q.
    ``workspace``: uint8 of ``mvb_paged_attention_decode_kv4_workspace_bytes`` (any content, not shared by
    calls that overlap); by default each call takes its own from torch's allocator, where it needs one."""
    what = "paged_attention_decode_kv4"
    index, L, P, nkv, bs, D = _kv4_geometry(what, kv4, layer)
    dims = q.dim() if isinstance(q, torch.Tensor) else 0
    if dims == 4:
        B, T, Hq, qd = q.shape
    elif dims == 3:
        B, Hq, qd = q.shape
        T = 1
    else:
        raise RuntimeError(f"{what}: q must be [B, Hq, D] or [B, T, Hq, D]")
    try:
        ok = (q.dtype is _BF16 and block_tables.dtype is _I32 and ctx_lens.dtype is _I32 and q.get_device() == index
              and block_tables.get_device() == index and ctx_lens.get_device() == index and block_tables.dim() == 2
              and ctx_lens.dim() == 1)
    except AttributeError:
        ok = False
    if not ok:
        _joint(what, index, ("q", q, _BF16, dims), ("block_tables", block_tables, _I32, 2),
               ("ctx_lens", ctx_lens, _I32, 1))
    if qd != D or Hq % nkv or not Hq:
        raise RuntimeError(f"{what}: q {tuple(q.shape)} over {nkv} KV heads of {D}")
    rows, width = block_tables.shape
    if rows != B or ctx_lens.numel() != B:
        raise RuntimeError(f"{what}: {B} sequences, {rows} block tables, {ctx_lens.numel()} lengths")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _expect(what, "out", out, index, torch.bfloat16, dims)
        if out.shape != q.shape or not out.is_contiguous() or out.data_ptr() % 16:
            raise RuntimeError(f"{what}: out must be contiguous and 16-byte aligned, of the shape of q")
    if B == 0 or T == 0:
        return out
    if width == 0:
        return out.zero_()
    q_stride = Hq * D
    if not q.is_contiguous():
        q = q.reshape(B * T, Hq, D)
        q_stride = q.stride(0)
        if q.stride(2) != 1 or q.stride(1) != D or q_stride % 8 or q_stride < Hq * D:
            q, q_stride = q.clone(memory_format=torch.contiguous_format), Hq * D
    if q.data_ptr() % 16:
        q, q_stride = q.clone(memory_format=torch.contiguous_format), Hq * D
    t_stride = width
    if not block_tables.is_contiguous():
        t_stride = block_tables.stride(0)
        if block_tables.stride(1) != 1 or t_stride < width:
            block_tables, t_stride = block_tables.contiguous(), width
    ctx_lens = ctx_lens.contiguous()
    ws_at, ws_bytes = None, 0
    if workspace is None:
        if width * bs > _KV4_UNSPLIT_TOKENS:
            ws_bytes = _kv4_workspace_bytes(B, T, Hq, nkv, D, index)
            workspace = torch.empty(ws_bytes, dtype=_U8, device=q.device)
            ws_at = workspace.data_ptr()
    else:
        _expect(what, "workspace", workspace, index, torch.uint8, 1)
        if not workspace.is_contiguous():
            raise RuntimeError(f"{what}: workspace must be contiguous")
        ws_at, ws_bytes = workspace.data_ptr(), workspace.numel()
    N.on_device(index, what, N.lib().mvb_paged_attention_decode_kv4, out.data_ptr(), Hq * D, q.data_ptr(), q_stride,
                kv4.data_ptr(), block_tables.data_ptr(), t_stride, width, ctx_lens.data_ptr(), B, T, Hq, nkv, D, L,
                int(layer), P, bs, float(scale), float(softcap), int(window), ws_at, ws_bytes)
    return out


# ------------------------------------------------------- block tables and slots of a step
class SlotPlan(NamedTuple):
    """Where a step's tokens go (``assign_slots``)."""
    slots: torch.Tensor      # int64 [num_tokens]: block * block_size + offset; -1: none
    positions: torch.Tensor  # int32 [num_tokens]
    seq_start: torch.Tensor  # int32 [B + 1]: first token of each sequence
    granted: torch.Tensor    # int32 [B]: 1 where the sequence got its blocks
    free_head: torch.Tensor  # int32 [1]: the free list's head after this step


def assign_slots(block_tables: torch.Tensor, ctx_lens: torch.Tensor, new_lens: torch.Tensor,
                 free_blocks: torch.Tensor, block_size: int, num_tokens: int,
                 free_head: torch.Tensor | None = None, held_blocks: torch.Tensor | None = None) -> SlotPlan:
    """Grows the block tables of a step on the GPU and maps its tokens to slots, in the order in which
    ``KVCacheManager`` pops its free list.  Sequence b holds ``ctx_lens[b]`` tokens (int32) in the first
    blocks of its row of ``block_tables`` (int32 ``[B, max_blocks]``, updated in place) and takes
    ``new_lens[b]`` more; the blocks it lacks come off ``free_blocks`` (int32), from ``free_head``
    (int32 ``[1]``, default 0) on.  ``num_tokens``: length of the per-token outputs, at least the sum of
    ``new_lens`` for every sequence to be granted; the entries behind the last token are -1.  A sequence that does not
    fit (its table row, the free list, ``num_tokens``) takes nothing: ``granted`` 0 and slots -1, and its length must
    stay as it was.

    ``held_blocks`` (int32 ``[B]``, updated in place): how many entries of its row each sequence holds, 0 for a new
    one.  Needed where lengths go back, as rejected drafts make them: the blocks behind a shorter length are then used
    again, where without a count new ones would be taken over them.  A count below what ``ctx_lens`` needs, or past the
    row, is refused like a negative length.

    The outputs are cut from one allocation: one that is kept keeps all of it."""
    return _assign_slots(block_tables, ctx_lens, new_lens, free_blocks, block_size, num_tokens, free_head, held_blocks)


def _assign_slots(block_tables, ctx_lens, new_lens, free_blocks, block_size, num_tokens, free_head=None,
                  held_blocks=None, apart: bool = False) -> SlotPlan:
    """``assign_slots``; with ``apart`` each output is a tensor of its own."""
    what = "assign_slots"
    index = block_tables.get_device() if isinstance(block_tables, torch.Tensor) else -1
    try:
        ok = (index >= 0 and block_tables.dtype is _I32 and ctx_lens.dtype is _I32 and new_lens.dtype is _I32
              and free_blocks.dtype is _I32 and ctx_lens.get_device() == index and new_lens.get_device() == index
              and free_blocks.get_device() == index and block_tables.dim() == 2 and ctx_lens.dim() == 1
              and new_lens.dim() == 1 and free_blocks.dim() == 1)
    except AttributeError:
        ok = False
    if not ok:
        _joint(what, index, ("block_tables", block_tables, _I32, 2), ("ctx_lens", ctx_lens, _I32, 1),
               ("new_lens", new_lens, _I32, 1), ("free_blocks", free_blocks, _I32, 1))
    B, width = block_tables.shape
    if ctx_lens.numel() != B or new_lens.numel() != B:
        raise RuntimeError(f"{what}: {B} block tables, {ctx_lens.numel()} and {new_lens.numel()} lengths")
    t_stride = width
    if not block_tables.is_contiguous():
        t_stride = block_tables.stride(0) if B > 1 else width
        if width > 1 and block_tables.stride(1) != 1 or t_stride < width:
            raise RuntimeError(f"{what}: the rows of block_tables must be contiguous and apart")
    if free_head is not None:
        _expect(what, "free_head", free_head, index, torch.int32, 1)
        if free_head.numel() != 1:
            raise RuntimeError(f"{what}: free_head must hold one number")
    if held_blocks is not None:
        _expect(what, "held_blocks", held_blocks, index, torch.int32, 1)
        if held_blocks.numel() != B or not held_blocks.is_contiguous():
            raise RuntimeError(f"{what}: held_blocks must be contiguous, one number for each of {B} sequences")
    if num_tokens < 0:
        raise RuntimeError(f"{what}: num_tokens {num_tokens}")
    ctx_lens, new_lens, free_blocks = ctx_lens.contiguous(), new_lens.contiguous(), free_blocks.contiguous()
    device = block_tables.device
    if apart:
        slots = torch.empty(num_tokens, dtype=_I64, device=device)
        positions, seq_start, granted, head = (torch.empty(n, dtype=_I32, device=device) for n in (num_tokens, B + 1, B, 1))
        at = [t.data_ptr() for t in (slots, positions, seq_start, granted, head)]
    else:  # one allocation: slots (two words each), positions, starts, granted, the head
        words = torch.empty(3 * num_tokens + 2 * B + 2, dtype=_I32, device=device)
        base = words.data_ptr()
        slots, positions, seq_start, granted, head = words.split_with_sizes((2 * num_tokens, num_tokens, B + 1, B, 1))
        slots = slots.view(_I64)
        start = base + 12 * num_tokens
        at = (base, base + 8 * num_tokens, start, start + 4 * (B + 1), start + 4 * (2 * B + 1))
    ws, ws_bytes = None, 0
    if B > 8192:
        ws_bytes = N.lib().mvb_assign_slots_workspace_bytes(B)
        ws = torch.empty(ws_bytes, dtype=_U8, device=device)
    N.on_device(index, what, N.lib().mvb_assign_slots_ex, *at, block_tables.data_ptr(), t_stride, width,
                ctx_lens.data_ptr(), new_lens.data_ptr(), N.ptr(held_blocks), free_blocks.data_ptr(), free_blocks.numel(),
                N.ptr(free_head), B, int(block_size), int(num_tokens), N.ptr(ws), ws_bytes)
    return SlotPlan(slots, positions, seq_start, granted, head)


# ------------------------------------------------------------------ drafted tokens
def _prob_rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``t`` [B, n, V] with rows of stride-1 entries a fixed distance apart, else a copy; and that distance."""
    B, n, V = t.shape
    if t.is_contiguous():
        return t, V
    s0, s1, s2 = t.stride()
    row = s1 if n > 1 else s0 if B > 1 else V
    if (s2 == 1 or V == 1) and row >= V and (B == 1 or n == 1 or s0 == n * s1):
        return t, row
    return t.contiguous(), V


def verify_drafts(target_probs: torch.Tensor, draft_tokens: torch.Tensor, uniforms: torch.Tensor,
                  draft_probs: torch.Tensor | None = None,
                  draft_lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Accepts or replaces the drafted tokens of a batch (speculative sampling).

    ``target_probs`` fp32 ``[B, K + 1, V]``: the target's distributions at each draft and after the last
    (``sample(..., probs_out=)`` gives them, filtered and tempered); ``draft_tokens`` int64 ``[B, K]``,
    the first ``draft_lens[b]`` (int32, default K) of them given; ``draft_probs`` fp32 ``[B, K, V]``: what
    the drafts were drawn from, or None for greedy or looked-up drafts; ``uniforms`` fp32 ``[B, K + 1]`` in
    [0, 1).  Draft i is accepted while ``uniforms[i] * q(d) < p(d)``; the first rejected one is replaced by
    a draw from ``max(p - q, 0)``, and where all pass one more token is drawn from the row behind them
    (inverse CDF in vocabulary order with the last uniform, sums in 64 bits).  Returns ``(tokens
    int64 [B, K + 1], accepted int32 [B])``: accepted drafts, the drawn token, then -1."""
    what = "verify_drafts"
    index = target_probs.get_device() if isinstance(target_probs, torch.Tensor) else -1
    try:
        ok = (index >= 0 and target_probs.dtype is _F32 and draft_tokens.dtype is _I64 and uniforms.dtype is _F32
              and target_probs.dim() == 3 and draft_tokens.get_device() == index and uniforms.get_device() == index)
    except AttributeError:
        ok = False
    if not ok:
        _joint(what, index, ("target_probs", target_probs, _F32, 3), ("draft_tokens", draft_tokens, _I64, 2),
               ("uniforms", uniforms, _F32, 2))
    B, rows, V = target_probs.shape
    K = rows - 1
    if K < 0 or V == 0 or draft_tokens.shape != (B, K) or uniforms.shape != (B, rows):
        raise RuntimeError(f"{what}: target_probs {tuple(target_probs.shape)}, draft_tokens "
                           f"{tuple(draft_tokens.shape)}, uniforms {tuple(uniforms.shape)}")
    if draft_probs is not None:
        _expect(what, "draft_probs", draft_probs, index, torch.float32, 3)
        if draft_probs.shape != (B, K, V):
            raise RuntimeError(f"{what}: draft_probs must be {(B, K, V)}, not {tuple(draft_probs.shape)}")
    if draft_lens is not None:
        _expect(what, "draft_lens", draft_lens, index, torch.int32, 1)
        if draft_lens.shape[0] != B:
            raise RuntimeError(f"{what}: {B} sequences, {draft_lens.shape[0]} draft_lens")
        draft_lens = draft_lens.contiguous()
    out = torch.empty(B, rows, dtype=torch.int64, device=target_probs.device)
    accepted = torch.empty(B, dtype=torch.int32, device=target_probs.device)
    if B == 0:
        return out, accepted
    target_probs, p_stride = _prob_rows(target_probs)
    q_stride = V
    if draft_probs is not None:
        if K == 0:
            draft_probs = None
        else:
            draft_probs, q_stride = _prob_rows(draft_probs)
    draft_tokens, uniforms = draft_tokens.contiguous(), uniforms.contiguous()
    N.on_device(index, what, N.lib().mvb_verify_drafts, out.data_ptr(), accepted.data_ptr(), target_probs.data_ptr(),
                p_stride, N.ptr(draft_probs), q_stride, draft_tokens.data_ptr(), uniforms.data_ptr(),
                N.ptr(draft_lens), B, K, V)
    return out, accepted


# --------------------------------------------------------------------- rows in 8 bits
class Q8Rows(NamedTuple):
    """Rows in 8 bits with one scale each: element i of a row stands for ``values[..., i] * scales[...]``."""
    values: torch.Tensor  # int8 [..., width], codes of -127 to 127
    scales: torch.Tensor  # fp32 [...]


_I8, _F16 = torch.int8, torch.float16
_DTYPE_CODE = {_F32: N.F32, _F16: N.F16, _BF16: N.BF16}


def _refuse_rows(what: str, name: str, t, index: int | None = None, dtype=None, shape=None) -> None:
    """Why ``t`` is not rows of a float type on a GPU, or not those of the other operand."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{what}: {name} must be a tensor")
    N.require_cuda(t)
    if t.dtype not in _DTYPE_CODE or t.dim() == 0 or t.shape[-1] == 0:
        raise RuntimeError(f"{what}: {name} must be rows of float32, float16 or bfloat16, not {tuple(t.shape)} {t.dtype}")
    raise RuntimeError(f"{what}: {name} is {tuple(t.shape)} {t.dtype} on {t.device}, not {tuple(shape)} {dtype} on "
                       f"cuda:{index}")


def _float_rows(what: str, name: str, t) -> tuple[int, int, torch.Size]:
    """Rows of a float type on a GPU: device, dtype code, shape."""
    try:
        index, code, shape = t.get_device(), _DTYPE_CODE[t.dtype], t.shape
        if index >= 0 and shape[-1]:
            return index, code, shape
    except (AttributeError, KeyError, IndexError, TypeError):
        pass
    return _refuse_rows(what, name, t)


def _same_rows(what: str, name: str, t, index: int, dtype: torch.dtype, shape: torch.Size) -> None:
    """The other operand's rows: its device, type and shape."""
    try:
        if t.dtype is dtype and t.shape == shape and t.get_device() == index:
            return
    except AttributeError:
        pass
    _refuse_rows(what, name, t, index, dtype, shape)


def _row_view(t: torch.Tensor) -> tuple[torch.Tensor, int] | None:
    """``t`` as rows of stride-1 elements a fixed distance apart, and that distance; None if it is not."""
    shape = t.shape
    width = shape[-1]
    if t.is_contiguous():
        return t, width
    strides = t.stride()
    if width > 1 and strides[-1] != 1:
        return None
    if len(shape) == 2:
        row = strides[0] if shape[0] > 1 else width
        return (t, row) if row >= width else None
    row, size = None, 1  # rows of the dimensions so far are `row` apart; 0 where one is broadcast
    for n, stride in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n == 1:
            continue
        if row is None:
            row = stride
        elif stride != row * size:
            return None
        size *= n
    if row is None:
        row = width
    return (t, row) if row >= width else None


def _rows_of(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``_row_view``, of a copy where ``t`` is laid out otherwise."""
    if t.is_contiguous():
        return t, t.shape[-1]
    view = _row_view(t)
    return view if view is not None else (t.contiguous(), t.shape[-1])


def _q8_out(like: torch.Tensor, shape: torch.Size) -> Q8Rows:
    return Q8Rows(like.new_empty(shape, dtype=_I8), like.new_empty(shape[:-1], dtype=_F32))


def quantise_q8(input: torch.Tensor) -> Q8Rows:
    """Rows ``[..., width]`` in 8 bits: per row ``amax = max |x|``, codes ``rint(127 x / amax)``, scale
    ``amax / 127``.  A row with an infinity or a NaN reads back as NaN."""
    what = "quantise_q8"
    index, code, shape = _float_rows(what, "input", input)
    x, stride = _rows_of(input)
    out = _q8_out(x, shape)
    values, scales = out
    rows = scales.numel()
    if rows:
        N.on_device(index, what, N.lib().mvb_quantise_q8, values.data_ptr(), scales.data_ptr(), x.data_ptr(), stride, rows,
                    shape[-1], code)
    return out


def _norm_weight(what: str, weight, index: int, width: int, dtype: torch.dtype) -> torch.Tensor:
    try:
        ok = weight.shape == (width,) and weight.get_device() == index
    except AttributeError:
        ok = False
    if not ok:
        if isinstance(weight, torch.Tensor):
            N.require_cuda(weight)
        raise RuntimeError(f"{what}: weight must be [{width}] on cuda:{index}")
    if weight.dtype is not dtype:
        weight = weight.to(dtype)
    return weight if weight.is_contiguous() else weight.contiguous()


def rmsnorm_q8(input: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, plus_one: bool = False) -> Q8Rows:
    """``rmsnorm`` (``plus_one``: with ``1 + weight``) whose result goes to 8 bits from its 32, without a
    rounding to the dtype in between.  Rows, non-finite ones too, as in ``quantise_q8``; the mean of the squares and the
    products with the weight are held in 32 bits, so a row reads back as zeros where the sum of its squares passes fp32's
    range (elements of some 1e19, as in ``rmsnorm``), and as NaN where a product ``x * weight`` does."""
    what = "rmsnorm_q8"
    index, code, shape = _float_rows(what, "input", input)
    width = shape[-1]
    w = _norm_weight(what, weight, index, width, input.dtype)
    x, stride = _rows_of(input)
    out = _q8_out(x, shape)
    values, scales = out
    rows = scales.numel()
    if rows:
        N.on_device(index, what, N.lib().mvb_rmsnorm_q8, values.data_ptr(), scales.data_ptr(), x.data_ptr(), stride,
                    w.data_ptr(), rows, width, float(eps), int(plus_one), code)
    return out


def fused_add_rmsnorm_q8(residual: torch.Tensor, input: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                         plus_one: bool = False,
                         residual_out: torch.Tensor | None = None) -> tuple[Q8Rows, torch.Tensor]:
    """``fused_add_rmsnorm`` with its result in 8 bits: ``residual + input``, rounded to the dtype, goes to
    ``residual_out`` (default: into ``residual``, in place; it may be ``input`` too, but overlap neither of them
    otherwise, nor ``weight``), its norm to 8 bits as in ``rmsnorm_q8``.  Returns ``(rows, residual_out)``."""
    what = "fused_add_rmsnorm_q8"
    index, code, shape = _float_rows(what, "input", input)
    dtype, width = input.dtype, shape[-1]
    _same_rows(what, "residual", residual, index, dtype, shape)
    w = _norm_weight(what, weight, index, width, dtype)
    if residual_out is None:
        residual_out = residual
    else:
        _same_rows(what, "residual_out", residual_out, index, dtype, shape)
    view = _row_view(residual_out)
    if view is None:
        raise RuntimeError(f"{what}: the rows of {'residual' if residual_out is residual else 'residual_out'} must be "
                           "contiguous and evenly apart: they are written")
    x, stride = _rows_of(input)
    res, res_stride = _rows_of(residual)
    out = _q8_out(x, shape)
    values, scales = out
    rows = scales.numel()
    if rows:
        N.on_device(index, what, N.lib().mvb_fused_add_rmsnorm_q8, values.data_ptr(), scales.data_ptr(),
                    residual_out.data_ptr(), view[1], res.data_ptr(), res_stride, x.data_ptr(), stride, w.data_ptr(), rows,
                    width, float(eps), int(plus_one), code)
    return out, residual_out


def _gated_q8(what: str, gate, up, act: int) -> Q8Rows:
    index, code, shape = _float_rows(what, "gate", gate)
    _same_rows(what, "up", up, index, gate.dtype, shape)
    (g, g_stride), (u, u_stride) = _rows_of(gate), _rows_of(up)
    out = _q8_out(g, shape)
    values, scales = out
    rows = scales.numel()
    if rows:
        N.on_device(index, what, N.lib().mvb_gated_q8, values.data_ptr(), scales.data_ptr(), g.data_ptr(), g_stride,
                    u.data_ptr(), u_stride, rows, shape[-1], act, code)
    return out


def swiglu_q8(gate: torch.Tensor, up: torch.Tensor) -> Q8Rows:
    """``swiglu`` with its result in 8 bits: ``silu(gate) * up`` in 32 bits, then as in ``quantise_q8``.  The halves
    of a projection's ``[..., 2 I]`` output (``.chunk(2, -1)``) are read where they are."""
    return _gated_q8("swiglu_q8", gate, up, N.ACT_SILU)


def geglu_q8(gate: torch.Tensor, up: torch.Tensor) -> Q8Rows:
    """``geglu`` (tanh approximation) with its result in 8 bits, as ``swiglu_q8``."""
    return _gated_q8("geglu_q8", gate, up, N.ACT_GELU_TANH)


def _check_q8(what: str, rows) -> int:
    """Device of rows in 8 bits, checked."""
    try:
        v, s = rows
        index, shape = v.get_device(), v.shape
        if (v.dtype is _I8 and s.dtype is _F32 and index >= 0 and s.get_device() == index and len(shape)
                and s.shape == shape[:-1] and shape[-1]):
            return index
    except (AttributeError, TypeError, ValueError):  # no pair, or not of tensors
        raise RuntimeError(f"{what}: rows must be Q8Rows, values and scales both tensors") from None
    N.require_cuda(v, s)
    raise RuntimeError(f"{what}: values {tuple(v.shape)} {v.dtype} and scales {tuple(s.shape)} {s.dtype} are not int8 "
                       "rows with an fp32 scale each, on one GPU")


def dequantise_q8(rows: Q8Rows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """What rows in 8 bits stand for, rounded to ``dtype`` (float32, float16 or bfloat16)."""
    what = "dequantise_q8"
    index = _check_q8(what, rows)
    code = _DTYPE_CODE.get(dtype)
    if code is None:
        raise RuntimeError(f"{what}: float32, float16 or bfloat16, not {dtype}")
    values, scales = rows
    v, stride = _rows_of(values)
    scales = scales.contiguous()
    out = v.new_empty(v.shape, dtype=dtype)
    n = scales.numel()
    if n:
        N.on_device(index, what, N.lib().mvb_dequantise_q8, out.data_ptr(), v.data_ptr(), stride, scales.data_ptr(), n,
                    v.shape[-1], code)
    return out


# --------------------------------------------------------------------- weights in 4 bits
class W4Weight(NamedTuple):
    """A weight matrix ``[n, k]`` in 4 bits with group scales, as ``quantise_w4`` and ``pack_w4`` lay it out."""
    records: torch.Tensor  # uint8 [ceil(n / 16) * ceil(k / 128), 1024 + 64 * (128 / group)]
    n: int
    k: int
    group: int


def _w4_records(what: str, n: int, k: int, group: int, device: torch.device) -> torch.Tensor:
    if group not in _W4_BYTES:
        raise RuntimeError(f"{what}: groups of 32, 64 or 128 columns, not {group}")
    if k <= 0 or k % 32:
        raise RuntimeError(f"{what}: a multiple of 32 columns, not {k}")
    return torch.empty((n + 15) // 16 * ((k + 127) // 128), _W4_BYTES[group], dtype=_U8, device=device)


def quantise_w4(weight: torch.Tensor, group: int = 128) -> W4Weight:
    """A bf16 weight matrix ``[n, k]`` (k a multiple of 32) in 4 bits, once, for ``linear_w4``.  Per row and group
    of 32, 64 or 128 columns: ``lo = min(0, min w)``, ``hi = max(0, max w)``, ``scale = bf16((hi - lo) / 15)``,
    ``zero = rint(-lo / scale)``, ``code = rint(w / scale) + zero``; a weight stands for
    ``scale * (code - zero)``.  A group with a NaN or an infinity, or whose ``hi - lo`` leaves fp32's range, reads back
    as NaN."""
    what = "quantise_w4"
    index = weight.get_device() if isinstance(weight, torch.Tensor) else -1
    _expect(what, "weight", weight, index, _BF16, 2)
    n, k = weight.shape
    records = _w4_records(what, n, k, group, weight.device)
    w, stride = _rows_of(weight)
    if w.data_ptr() % 16 or stride % 8:
        w, stride = w.clone(memory_format=torch.contiguous_format), k
    if n:
        N.on_device(index, what, N.lib().mvb_quantise_w4, records.data_ptr(), w.data_ptr(), stride, n, k, group)
    return W4Weight(records, n, k, group)


def pack_w4(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, group: int = 128) -> W4Weight:
    """The same from a checkpoint's numbers: ``codes`` uint8 ``[n, k]``, ``scales`` bf16 and ``zeros`` uint8
    ``[n, ceil(k / group)]`` (None: 8 everywhere, a symmetric checkpoint).  Of codes and zeros the low 4 bits count.
    A checkpoint's fp16 scales lose three of their 11 bits in bf16."""
    what = "pack_w4"
    index = codes.get_device() if isinstance(codes, torch.Tensor) else -1
    _expect(what, "codes", codes, index, _U8, 2)
    _expect(what, "scales", scales, index, _BF16, 2)
    n, k = codes.shape
    records = _w4_records(what, n, k, group, codes.device)
    want = (n, (k + group - 1) // group)
    if zeros is not None:
        _expect(what, "zeros", zeros, index, _U8, 2)
    if scales.shape != want or zeros is not None and zeros.shape != want:
        raise RuntimeError(f"{what}: scales and zeros of {tuple(codes.shape)} codes in groups of {group} must be {want}")
    codes, scales = codes.contiguous(), scales.contiguous()
    if codes.data_ptr() % 8:
        codes = codes.clone()
    if zeros is not None:
        zeros = zeros.contiguous()
    if n:
        N.on_device(index, what, N.lib().mvb_pack_w4, records.data_ptr(), codes.data_ptr(), scales.data_ptr(),
                    N.ptr(zeros), n, k, group)
    return W4Weight(records, n, k, group)


_W4_BYTES = {32: 1280, 64: 1152, 128: 1088}  # of a record, by the group


def _check_w4(what: str, weight: W4Weight) -> int:
    """Device of a 4-bit weight, checked."""
    try:
        r, n, k, group = weight
        index = r.get_device()
        if (r.dtype is _U8 and r.shape == ((n + 15) // 16 * ((k + 127) // 128), _W4_BYTES[group]) and r.is_contiguous()
                and index >= 0 and k > 0 and k % 32 == 0 and r.data_ptr() % 16 == 0):
            return index
    except (AttributeError, KeyError, TypeError, ValueError):
        raise RuntimeError(f"{what}: weight must be what quantise_w4 or pack_w4 gave") from None
    N.require_cuda(r)
    raise RuntimeError(f"{what}: weight must be what quantise_w4 or pack_w4 gave")


def dequantise_w4(weight: W4Weight, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The matrix ``[n, k]`` that a 4-bit weight stands for, rounded to bfloat16, or in float32."""
    what = "dequantise_w4"
    index = _check_w4(what, weight)
    if dtype not in (_BF16, _F32):
        raise RuntimeError(f"{what}: float32 or bfloat16, not {dtype}")
    records, n, k, group = weight
    out = torch.empty(n, k, dtype=dtype, device=records.device)
    if n:
        N.on_device(index, what, N.lib().mvb_dequantise_w4, out.data_ptr(), records.data_ptr(), n, k, group,
                    _DTYPE_CODE[dtype])
    return out


def linear_w4(x: torch.Tensor | Q8Rows, weight: W4Weight, out: torch.Tensor | None = None) -> torch.Tensor:
    """``linear`` with a 4-bit weight: ``x @ w.T`` (bf16) for bf16 rows ``[..., k]`` or rows in 8 bits (``Q8Rows``), one
    row (of at most 262144) to many.  Sums run in 32 bits and are rounded once; no weight or product is rounded before.
    k is at most 32768.  A bf16 row with an infinity or a NaN has results that are not finite (NaN in calls
    of few rows), and leaves the other rows alone.  ``out``: bf16 ``[rows, n]`` with contiguous rows, and then what is
    returned; it must not overlap ``x``."""
    what = "linear_w4"
    index = _check_w4(what, weight)
    records, n, k, group = weight
    scales = None
    if type(x) is Q8Rows:
        if _check_q8(what, x) != index:
            raise RuntimeError(f"{what}: x is on {x.values.device}, the weight on {records.device}")
        x, scales = x
        scales = scales.contiguous()
    elif not isinstance(x, torch.Tensor) or x.dtype is not _BF16 or x.get_device() != index or x.dim() == 0:
        if isinstance(x, torch.Tensor):
            N.require_cuda(x)
        raise RuntimeError(f"{what}: x must be bfloat16 rows or Q8Rows on {records.device}")
    shape = x.shape
    if shape[-1] != k:
        raise RuntimeError(f"{what}: rows of {shape[-1]} elements for {k} columns")
    x, ldx = _rows_of(x)
    if x.data_ptr() % 16 or ldx * x.element_size() % 16:
        x, ldx = x.clone(memory_format=torch.contiguous_format), k
    rows = x.numel() // k
    if out is None:
        y = x.new_empty(shape[:-1] + (n,), dtype=_BF16)
        ldy = n
    else:
        _expect(what, "out", out, index, _BF16, 2)
        ldy = out.stride(0) if rows > 1 else n
        if out.shape != (rows, n) or n > 1 and out.stride(1) != 1 or ldy < n:
            raise RuntimeError(f"{what}: out must be {(rows, n)} with contiguous rows, apart")
        y = out
    if rows and n:
        N.on_device(index, what, N.lib().mvb_linear_w4, y.data_ptr(), ldy, x.data_ptr(), ldx, N.ptr(scales),
                    records.data_ptr(), rows, n, k, group)
    return y


class FusedMLPW4(nn.Module):
    """A ``FusedMLP`` with weights in 4 bits, made from one: gate_up product, act(gate) * up, down product.

    ``rows``: what the products read.  8: rows in 8 bits (bf16 rows that come in are quantised, ``Q8Rows``
    from ``fused_add_rmsnorm_q8`` taken as they are; the activation's result goes to 8 bits where it is made).
    16: bf16 rows."""

    def __init__(self, mlp: FusedMLP, group: int = 128, rows: int = 8):
        super().__init__()
        if rows not in (8, 16):
            raise ValueError(f"rows of 8 or 16 bits, not {rows}")
        self.rows, self.group, self._act_code = rows, group, mlp._act_code
        self.intermediate_size, self.hidden_size = mlp.intermediate_size, mlp.down_proj.weight.shape[0]
        for name in ("gate_up", "down"):
            weight = getattr(mlp, name + "_proj").weight.detach()
            self.register_buffer(name, quantise_w4(weight.to(torch.bfloat16), group).records)

    def forward(self, x: torch.Tensor | Q8Rows) -> torch.Tensor:
        inter, hidden = self.intermediate_size, self.hidden_size
        gate_up, down = W4Weight(self.gate_up, 2 * inter, hidden, self.group), W4Weight(self.down, hidden, inter, self.group)
        if self.rows == 8 and type(x) is not Q8Rows:
            x = quantise_q8(x)
        gu = linear_w4(x, gate_up)
        if self.rows == 16:
            return linear_w4(fused_mlp_forward(gu, inter, self._act_code), down)
        gate, up = gu.chunk(2, -1)
        return linear_w4((swiglu_q8 if self._act_code == 0 else geglu_q8)(gate, up), down)
