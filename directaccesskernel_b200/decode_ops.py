"""Element-wise steps of a Llama decode layer on the GPU (RMSNorm with a fused
residual add, rotary q/k, SiLU-gated product), one launch each.  They follow
transformers' Llama arithmetic op by op (app/python/llama/vanila_llama.py:
227-400 runs the same ops as separate torch kernels)."""
from __future__ import annotations

import ctypes
import math

import torch

from ._lib import LIB, RotaryArgs, check
from .runtime import dak_dtype
from .trace import traced


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def stream_of(device: int) -> int:
    """The current stream's handle on the current device, without building a
    ``torch.cuda.Stream`` (3 us of a call's host time)."""
    return torch._C._cuda_getCurrentRawStream(device)


def current_device_of(t: torch.Tensor, name: str) -> int:
    """The index of t's device, which must be the current CUDA device."""
    device = t.get_device()
    if device < 0 or device != torch._C._cuda_getDevice():
        raise RuntimeError(f"{name} must be on the current CUDA device")
    return device


def _check16(*ts):
    for t in ts:
        if t.dtype not in (torch.float16, torch.bfloat16) or not t.is_cuda:
            raise RuntimeError("decode ops take float16/bfloat16 CUDA tensors")
        if t.stride(-1) != 1:
            raise RuntimeError("decode ops need a contiguous last dimension")


@traced
def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """RMSNorm of x [rows, cols]; with ``residual``, first x + residual, written back
    into ``residual`` (the running hidden state), then normalised."""
    _check16(x, weight)
    rows, cols = x.shape
    if residual is not None:
        _check16(residual)
        if residual.shape != x.shape or residual.stride() != x.stride():
            raise RuntimeError("residual must match x in shape and strides")
    if weight.numel() != cols or not weight.is_contiguous():
        raise RuntimeError("weight must be a contiguous [cols] tensor")
    if out is None:
        out = torch.empty(rows, cols, dtype=x.dtype, device=x.device)
    rp = residual.data_ptr() if residual is not None else None
    check(LIB.dak_rmsnorm(x.data_ptr(), rp, weight.data_ptr(), out.data_ptr(), rp, rows, cols, x.stride(0),
                          float(eps), dak_dtype(x.dtype), _stream()), "rmsnorm")
    return out


@traced
def rope_qk(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, q_heads: int, kv_heads: int,
            head_dim: int, q_out: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor) -> None:
    """Rotary q/k of a fused qkv [B, (q_heads + 2 kv_heads) * head_dim] into q_out
    [B, q_heads, head_dim] and k_out [B, kv_heads, head_dim]; v is copied to v_out."""
    _check16(qkv, q_out, k_out, v_out)
    if positions.dtype != torch.int32 or not positions.is_cuda or inv_freq.dtype != torch.float32:
        raise RuntimeError("positions must be int32 CUDA, inv_freq float32 CUDA")
    if not (q_out.is_contiguous() and k_out.is_contiguous() and v_out.is_contiguous()):
        raise RuntimeError("q_out, k_out and v_out must be contiguous")
    check(LIB.dak_rope_qk(qkv.data_ptr(), qkv.stride(0), positions.data_ptr(), inv_freq.data_ptr(), q_out.data_ptr(),
                          k_out.data_ptr(), v_out.data_ptr(), qkv.shape[0], q_heads, kv_heads, head_dim,
                          dak_dtype(qkv.dtype), _stream()), "rope_qk")


@traced
def silu_mul(gate_up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """silu(gate) * up for gate_up [rows, 2 * cols] = [gate | up]."""
    _check16(gate_up)
    rows, two = gate_up.shape
    cols = two // 2
    if out is None:
        out = torch.empty(rows, cols, dtype=gate_up.dtype, device=gate_up.device)
    check(LIB.dak_silu_mul(gate_up.data_ptr(), gate_up.stride(0), out.data_ptr(), rows, cols,
                           dak_dtype(gate_up.dtype), _stream()), "silu_mul")
    return out


def rope_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None,
                     max_position: int | None = None, device="cuda") -> tuple[torch.Tensor, float]:
    """(inv_freq [rotary_dim / 2] float32, attention factor) of a rotary embedding.

    ``scaling`` is a model configuration's rope dictionary: ``rope_type``
    "default", "linear" (positions divided by ``factor``), "llama3" (long
    wavelengths divided by ``factor``, with a smooth transition between
    ``low_freq_factor`` and ``high_freq_factor``) or "yarn" (interpolation ramped
    over the number of turns within the original context, and an attention
    factor of 0.1 ln(factor) + 1 unless given).  ``max_position`` is the context
    that "yarn" extends when the dictionary does not name
    ``original_max_position_embeddings``."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise RuntimeError("rotary_dim must be positive and even")
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    inv = 1.0 / (theta ** (torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim))
    attention = 1.0
    if kind == "linear":
        inv = inv / float(scaling["factor"])
    elif kind == "llama3":
        factor, low, high = (float(scaling[k]) for k in ("factor", "low_freq_factor", "high_freq_factor"))
        turns = float(scaling["original_max_position_embeddings"]) * inv / (2 * math.pi)
        smooth = ((turns - low) / (high - low)).clamp(0.0, 1.0)  # 0: divided by factor, 1: as it is
        inv = (1 - smooth) * inv / factor + smooth * inv
    elif kind == "yarn":
        factor = float(scaling["factor"])
        context = scaling.get("original_max_position_embeddings") or max_position
        if context is None:
            raise RuntimeError("yarn scaling needs original_max_position_embeddings or max_position")

        def dim_of(turns: float) -> float:  # the (fractional) pair that makes this many turns in the context
            return rotary_dim * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = dim_of(float(scaling.get("beta_fast") or 32)), dim_of(float(scaling.get("beta_slow") or 1))
        if scaling.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        inv = inv / factor * ramp + inv * (1 - ramp)
        attention = scaling.get("attention_factor")
        if attention is None:
            def mscale(m: float) -> float:
                return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

            m, m_all = scaling.get("mscale"), scaling.get("mscale_all_dim")
            attention = mscale(m) / mscale(m_all) if m and m_all else mscale(1.0)
    elif kind != "default":
        raise RuntimeError(f"rope_type {kind!r} is not supported (default, linear, llama3 or yarn)")
    return inv.to(torch.float32).to(device), float(attention)


@traced
def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False,
           rope_scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions of x [tokens, heads, head_dim]: the first
    2 * inv_freq.numel() dims rotated by positions [tokens] (int32) times
    inv_freq, in pairs (i, i + R/2) or, ``interleaved``, (2i, 2i + 1), scaled by
    ``rope_scale`` (the attention factor of ``rope_frequencies``); the other dims
    copied.  FP32 arithmetic, one rounding, angles exact at any position.  Token
    and head strides are free (multiples of 8), so x may be the q and k heads of
    a fused projection; ``out`` may be x itself, else must not overlap it."""
    device = current_device_of(x, "x")
    dtype = x.dtype
    if x.dim() != 3 or dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("x must be a float16 or bfloat16 [tokens, heads, head_dim] tensor")
    T, H, D = shape = x.shape
    xt, xh, xd = x.stride()
    if xd != 1 and D > 1:
        raise RuntimeError("x must have a contiguous last dimension")
    _check_rope(positions, inv_freq, T, D, device)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype != dtype or out.get_device() != device:
        raise RuntimeError("out must match x in shape, dtype and device")
    if T and H:
        ot, oh, od = out.stride()
        if od != 1 and D > 1:
            raise RuntimeError("out must have a contiguous last dimension")
        a = RotaryArgs()
        a.x, a.out, a.positions, a.inv_freq = x.data_ptr(), out.data_ptr(), positions.data_ptr(), inv_freq.data_ptr()
        # A dimension of one entry has no stride to speak of.
        if T > 1:
            a.x_stride_t, a.o_stride_t = xt, ot
        if H > 1:
            a.x_stride_h, a.o_stride_h = xh, oh
        a.tokens, a.heads, a.head_dim, a.rotary_dim = T, H, D, 2 * inv_freq.numel()
        a.interleaved, a.rope_scale, a.dtype = interleaved, rope_scale, dak_dtype(dtype)
        check(LIB.dak_rotary(ctypes.byref(a), stream_of(device)), "rotary")
    return out


def _check_rope(positions: torch.Tensor, inv_freq: torch.Tensor, tokens: int, head_dim: int, device: int) -> None:
    if positions.dtype != torch.int32 or positions.get_device() != device or positions.numel() != tokens \
            or not positions.is_contiguous():
        raise RuntimeError("positions must be a contiguous int32 CUDA tensor with one entry per token")
    check_inv_freq(inv_freq, head_dim, device)


def check_inv_freq(inv_freq: torch.Tensor, head_dim: int, device: int) -> None:
    if inv_freq.dtype != torch.float32 or inv_freq.get_device() != device or not inv_freq.is_contiguous() \
            or 2 * inv_freq.numel() > head_dim:
        raise RuntimeError("inv_freq must be a contiguous float32 CUDA tensor of at most head_dim / 2 entries")
