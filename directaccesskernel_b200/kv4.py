"""The 4-bit tiered, paged KV cache: rotary + append, read-back and decode attention.

The cache of ``attention.decode_paged`` at a quarter of the bytes, for batches
whose KV is bound by HBM or, in pinned host memory, by the host link.  A pool is
one uint8 tensor [pages, kv_heads, slab] per tier (HBM, pinned host); the slab
of one (page, head) holds the codes of K and V and a float16 (scale, zero) pair
for every token and group of dims:

    K codes [P, 64] | K pairs [P, 128 / group, 2] | V codes [P, 64] | V pairs

with dim 2i in the low nibble of byte i and value = scale * code + zero.
``page_bytes`` gives the slab's bytes; page size (16, 32 or 64 tokens) and group
(32, 64 or 128 dims) follow from them.  Smaller groups are more exact: a page of
group 128 takes 4.25 bits per value, 64: 4.5, 32: 5.  Block tables name pages as
in ``attention.decode_paged``; entries outside their pool are recorded in the
device error word, skipped by the append and read as zeros.

Head dim 128.  Every call runs on the current stream of the current device,
which must be the tensors' own.  No reference counterpart: the reference's cache
is 16-bit (app/python/pinned_static_cache.py:8-115).
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import LIB, check
from .attention import HEAD_DIM, _stream_ptr, auto_split_size
from .decode_ops import _check_rope
from .runtime import dak_dtype
from .trace import traced

PAGE_SIZES = (16, 32, 64)
GROUPS = (32, 64, 128)
MAX_BLOCK_HEADS = 8  # query heads that one CTA of the attention serves


def page_bytes(page_size: int, group: int = 128) -> int:
    """Bytes of one (page, KV head) slab: a pool is [pages, kv_heads, page_bytes] uint8."""
    if page_size not in PAGE_SIZES or group not in GROUPS:
        raise RuntimeError(f"page_size must be one of {PAGE_SIZES} and group one of {GROUPS}")
    return 2 * page_size * (HEAD_DIM // 2 + 4 * (HEAD_DIM // group))


_FORMATS = {page_bytes(p, g): (p, g) for p in PAGE_SIZES for g in GROUPS}


def page_format(pool: torch.Tensor) -> tuple[int, int]:
    """(page_size, group) of a pool [pages, kv_heads, page_bytes]."""
    fmt = _FORMATS.get(pool.shape[-1])
    if fmt is None:
        raise RuntimeError(f"{pool.shape[-1]} bytes per (page, head) is no page_bytes(page_size, group)")
    return fmt


def _cache(device: torch.device, pool_dev, pool_host, block_table: torch.Tensor) -> _lib.Kv4Cache:
    """The checked pools and table as the C ABI takes them."""
    pool = pool_dev if pool_dev is not None else pool_host
    if pool is None:
        raise RuntimeError("no KV pool given")
    for t, nm in ((pool_dev, "pool_dev"), (pool_host, "pool_host")):
        if t is None:
            continue
        if t.dtype != torch.uint8 or t.dim() != 3 or not t.is_contiguous():
            raise RuntimeError(f"{nm} must be a contiguous uint8 [pages, kv_heads, page_bytes] tensor")
        if t.shape[1:] != pool.shape[1:]:
            raise RuntimeError("the pools must share kv_heads and page_bytes")
    if pool_dev is not None and pool_dev.device != device:
        raise RuntimeError("pool_dev is on the wrong device")
    if pool_host is not None and (pool_host.is_cuda or not pool_host.is_pinned()):
        raise RuntimeError("pool_host must be pinned host memory")
    if block_table.dtype != torch.int32 or block_table.device != device or block_table.dim() != 2 \
            or (block_table.size(1) > 1 and block_table.stride(1) != 1):
        raise RuntimeError("block_table must be an int32 CUDA tensor [B, max_pages]")
    c = _lib.Kv4Cache()
    c.page_size, c.group = page_format(pool)
    c.kv_heads = pool.shape[1]
    if pool_dev is not None and pool_dev.shape[0]:
        c.pool_dev, c.dev_pages = pool_dev.data_ptr(), pool_dev.shape[0]
    if pool_host is not None and pool_host.shape[0]:
        c.pool_host, c.host_pages = pool_host.data_ptr(), pool_host.shape[0]
    c.batch, c.max_pages = block_table.shape
    c.block_table = block_table.data_ptr()
    c.table_stride = block_table.stride(0) if c.batch > 1 else c.max_pages
    return c


def _on_current(device: torch.device) -> None:
    if device.type != "cuda" or device.index != torch.cuda.current_device():
        raise RuntimeError(f"tensors must be on the current CUDA device, got {device}")


def _check_tokens(positions: torch.Tensor, seq_index: torch.Tensor | None, device, batch: int) -> int:
    if positions.dtype != torch.int32 or positions.device != device or positions.dim() != 1 \
            or not positions.is_contiguous():
        raise RuntimeError("positions must be a contiguous int32 CUDA tensor [tokens]")
    T = positions.numel()
    if seq_index is None:
        if T != batch:
            raise RuntimeError("without seq_index there is one token per sequence of the block table")
    elif seq_index.dtype != torch.int32 or seq_index.device != device or seq_index.shape != positions.shape \
            or not seq_index.is_contiguous():
        raise RuntimeError("seq_index must be a contiguous int32 CUDA tensor [tokens]")
    return T


@traced
def rope_kv_append_q4(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor | None, q_heads: int,
                      q_out: torch.Tensor | None, pool_dev: torch.Tensor | None, pool_host: torch.Tensor | None,
                      block_table: torch.Tensor, *, seq_index: torch.Tensor | None = None, interleaved: bool = False,
                      rope_scale: float = 1.0) -> None:
    """Rotary embedding, 4-bit quantisation and append in one launch.

    ``qkv`` [tokens, (q_heads + 2 kv_heads) * 128] is the fused projection; its q
    heads are rotated into ``q_out`` [tokens, q_heads, 128] (None with q_heads 0),
    its k heads rotated and quantised and its v heads quantised into slot
    ``positions[t]`` of sequence ``seq_index[t]`` (None: one token per sequence,
    in order, as in a decode step; else any tokens of a prompt).  ``inv_freq``,
    ``interleaved`` and ``rope_scale`` are ``decode_ops.rotary``'s; inv_freq None
    rotates nothing.  Two tokens of one call must not share a sequence and
    position.  A NaN is stored as code 0 and values beyond float16 saturate: the
    cache holds finite numbers only."""
    device = qkv.device
    _on_current(device)
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("qkv must be a 16-bit [tokens, (q_heads + 2 kv_heads) * 128] tensor, last dim contiguous")
    c = _cache(device, pool_dev, pool_host, block_table)
    T = _check_tokens(positions, seq_index, device, c.batch)
    _check_rope(positions, inv_freq, T, HEAD_DIM)
    if qkv.shape[0] != T or qkv.shape[1] != (q_heads + 2 * c.kv_heads) * HEAD_DIM:
        raise RuntimeError(f"qkv must be [{T}, {(q_heads + 2 * c.kv_heads) * HEAD_DIM}]")
    if q_heads and (q_out is None or not q_out.is_contiguous() or q_out.dtype != qkv.dtype or q_out.device != device
                    or q_out.numel() != T * q_heads * HEAD_DIM):
        raise RuntimeError("q_out must be a contiguous [tokens, q_heads, 128] tensor of the qkv dtype")
    if T == 0:
        return
    a = _lib.Kv4AppendArgs()
    a.qkv, a.ld = qkv.data_ptr(), qkv.stride(0) if T > 1 else qkv.shape[1]
    a.positions, a.seq_index = positions.data_ptr(), seq_index.data_ptr() if seq_index is not None else None
    if inv_freq is not None:
        a.inv_freq, a.rotary_dim = inv_freq.data_ptr(), 2 * inv_freq.numel()
    a.rope_scale, a.interleaved = rope_scale, int(interleaved)
    a.q_out = q_out.data_ptr() if q_heads else None
    a.tokens, a.q_heads, a.dtype = T, q_heads, dak_dtype(qkv.dtype)
    check(LIB.dak_rope_kv_append_q4(ctypes.byref(c), ctypes.byref(a), _stream_ptr()), "rope_kv_append_q4")


@traced
def kv_read_q4(pool_dev: torch.Tensor | None, pool_host: torch.Tensor | None, block_table: torch.Tensor,
               positions: torch.Tensor, *, seq_index: torch.Tensor | None = None, dtype: torch.dtype = torch.float16,
               k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [tokens, kv_heads, 128] that the cache holds for the given tokens, in
    16 bits: what attention over the cache sees, for a prompt whose prefix is
    already cached."""
    device = block_table.device
    _on_current(device)
    if dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("dtype must be float16 or bfloat16")
    c = _cache(device, pool_dev, pool_host, block_table)
    T = _check_tokens(positions, seq_index, device, c.batch)
    shape = (T, c.kv_heads, HEAD_DIM)
    outs = []
    for t, nm in ((k_out, "k_out"), (v_out, "v_out")):
        if t is None:
            t = torch.empty(shape, dtype=dtype, device=device)
        elif t.shape != shape or t.dtype != dtype or t.device != device or not t.is_contiguous():
            raise RuntimeError(f"{nm} must be a contiguous [tokens, kv_heads, 128] tensor of dtype")
        outs.append(t)
    if T:
        check(LIB.dak_kv_read_q4(ctypes.byref(c), positions.data_ptr(),
                                 seq_index.data_ptr() if seq_index is not None else None, outs[0].data_ptr(),
                                 outs[1].data_ptr(), T, dak_dtype(dtype), _stream_ptr()), "kv_read_q4")
    return outs[0], outs[1]


def merge_counter_count(batch: int, q_heads: int, kv_heads: int) -> int:
    """Entries of ``decode_paged_q4``'s merge_counters."""
    return batch * kv_heads * -(-(q_heads // kv_heads) // MAX_BLOCK_HEADS)


@traced
def decode_paged_q4(query: torch.Tensor, pool_dev: torch.Tensor | None, pool_host: torch.Tensor | None,
                    block_table: torch.Tensor, seq_lens: torch.Tensor, scaling: float, split_size: int | None = None, *,
                    out: torch.Tensor | None = None, partial_o: torch.Tensor | None = None,
                    partial_ml: torch.Tensor | None = None, max_seq_len: int | None = None,
                    merge_counters: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention over the 4-bit cache; returns [B, Hq, 128].

    ``query`` [B, Hq, 128], any number of query heads per KV head; ``seq_lens``
    [B] int32 on the GPU (0: the row is zeros; longer than ``max_seq_len``: cut to
    it).  ``max_seq_len`` defaults to what the block table can name.  Scratch:
    partial_o [B, Hq, splits, 128] and partial_ml [B, Hq, splits, 2] float32,
    allocated when not given.  With ``merge_counters`` (int32 CUDA,
    ``merge_counter_count`` entries, zero before the first call and left zero by
    every call) the last split merges the splits inside the attention kernel
    instead of a second launch; the result is the same.  Calls that may overlap
    on the GPU need scratch and counters of their own."""
    device = query.device
    _on_current(device)
    if query.dim() != 3 or query.size(2) != HEAD_DIM or query.stride(2) != 1:
        raise RuntimeError("query must be [B, Hq, 128] with a contiguous last dimension")
    if query.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("query must be float16 or bfloat16")
    c = _cache(device, pool_dev, pool_host, block_table)
    B, Hq = query.size(0), query.size(1)
    if block_table.size(0) != B:
        raise RuntimeError("block_table must have one row per sequence")
    if seq_lens.dtype != torch.int32 or seq_lens.device != device or seq_lens.numel() != B \
            or not seq_lens.is_contiguous():
        raise RuntimeError("seq_lens must be a contiguous int32 CUDA tensor [B]")
    if Hq % c.kv_heads:
        raise RuntimeError("the KV heads must divide the query heads")
    if max_seq_len is None:
        max_seq_len = c.max_pages * c.page_size
    blocks = -(-(Hq // c.kv_heads) // MAX_BLOCK_HEADS)
    if split_size is None:
        split_size = auto_split_size(B * blocks, c.kv_heads, max_seq_len)
    if split_size <= 0:
        raise RuntimeError("split_size must be positive")
    splits = -(-max_seq_len // split_size)
    if out is None:
        out = torch.empty((B, Hq, HEAD_DIM), dtype=query.dtype, device=device)
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != device or out.stride(2) != 1:
        raise RuntimeError("out must be [B, Hq, 128] of the query dtype with a contiguous last dimension")
    a = _lib.AttnQ4Args()
    if splits > 1:
        for t, n, nm in ((partial_o, HEAD_DIM, "partial_o"), (partial_ml, 2, "partial_ml")):
            if t is not None and (t.dtype != torch.float32 or t.device != device or not t.is_contiguous()
                                  or t.numel() < B * Hq * splits * n):
                raise RuntimeError(f"{nm} must be a contiguous float32 CUDA tensor of B * Hq * {splits} * {n} entries")
        if partial_o is None:
            partial_o = torch.empty(B * Hq * splits * HEAD_DIM, dtype=torch.float32, device=device)
        if partial_ml is None:
            partial_ml = torch.empty(B * Hq * splits * 2, dtype=torch.float32, device=device)
        a.partial_o, a.partial_ml = partial_o.data_ptr(), partial_ml.data_ptr()
        if merge_counters is not None:
            if merge_counters.dtype != torch.int32 or merge_counters.device != device \
                    or merge_counters.numel() < B * c.kv_heads * blocks or not merge_counters.is_contiguous():
                raise RuntimeError("merge_counters must be a contiguous int32 CUDA tensor of merge_counter_count entries")
            a.merge_counters = merge_counters.data_ptr()
    a.query = query.data_ptr()
    a.q_stride_b, a.q_stride_h = query.stride(0) if B > 1 else 0, query.stride(1) if Hq > 1 else 0
    a.seq_lens = seq_lens.data_ptr()
    a.out = out.data_ptr()
    a.o_stride_b, a.o_stride_h = out.stride(0) if B > 1 else 0, out.stride(1) if Hq > 1 else 0
    a.num_q_heads, a.max_seq_len, a.split_size = Hq, max_seq_len, split_size
    a.scaling, a.dtype = scaling, dak_dtype(query.dtype)
    check(LIB.dak_attn_decode_paged_q4(ctypes.byref(c), ctypes.byref(a), _stream_ptr()), "decode_paged_q4")
    return out
