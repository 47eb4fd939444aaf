"""The 4-bit tiered, paged KV cache: rotary + append, read-back and decode attention.

The cache of ``attention.decode_paged`` at a quarter of the bytes, for batches
whose KV is bound by HBM or, in pinned host memory, by the host link.  A pool is
one uint8 tensor [pages, kv_heads, slab] per tier (HBM, pinned host); the slab
of one (page, head) holds the codes of K and V and a float16 (scale, zero) pair
for every token and group of dims:

    K codes [P, 64] | K pairs [P, 128 / group, 2] | V codes [P, 64] | V pairs

with dim 2i in the low nibble of byte i and value = scale * code + zero, scale >= 0.
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
from .attention import HEAD_DIM
from .decode_ops import check_inv_freq, current_device_of, stream_of
from .runtime import NUM_SMS, dak_dtype
from .trace import traced

PAGE_SIZES = (16, 32, 64)
GROUPS = (32, 64, 128)
MAX_BLOCK_HEADS = 8  # query heads that one CTA of the attention serves
MAX_SEQ_LEN = 2**31 - 65  # int32 positions, whole chunks
SHORT_ROWS = 512     # tokens up to which the attention does not split a row


def page_bytes(page_size: int, group: int = 128) -> int:
    """Bytes of one (page, KV head) slab: a pool is [pages, kv_heads, page_bytes] uint8."""
    if page_size not in PAGE_SIZES or group not in GROUPS:
        raise RuntimeError(f"page_size must be one of {PAGE_SIZES} and group one of {GROUPS}")
    return 2 * page_size * (HEAD_DIM // 2 + 4 * (HEAD_DIM // group))


_FORMATS = {page_bytes(p, g): (p, g) for p in PAGE_SIZES for g in GROUPS}


def page_format(pool: torch.Tensor) -> tuple[int, int]:
    """(page_size, group) of a pool [pages, kv_heads, page_bytes]."""
    if pool.shape[-1] not in _FORMATS:
        raise RuntimeError(f"{pool.shape[-1]} bytes per (page, head) is no page_bytes(page_size, group)")
    return _FORMATS[pool.shape[-1]]


def _cache(device: int, pool_dev, pool_host, block_table: torch.Tensor) -> _lib.Kv4Cache:
    """The checked pools and table as the C ABI takes them."""
    c = _lib.Kv4Cache()
    shape = None
    if pool_dev is not None:
        if pool_dev.get_device() != device:
            raise RuntimeError("pool_dev is on the wrong device")
        shape = _pool_shape(pool_dev, "pool_dev")
        if shape[0]:
            c.pool_dev, c.dev_pages = pool_dev.data_ptr(), shape[0]
    if pool_host is not None:
        if pool_host.is_cuda or not pool_host.is_pinned():
            raise RuntimeError("pool_host must be pinned host memory")
        host = _pool_shape(pool_host, "pool_host")
        if shape is not None and host[1:] != shape[1:]:
            raise RuntimeError("the pools must share kv_heads and page_bytes")
        shape = host
        if shape[0]:
            c.pool_host, c.host_pages = pool_host.data_ptr(), shape[0]
    if shape is None:
        raise RuntimeError("no KV pool given")
    if block_table.dtype != torch.int32 or block_table.get_device() != device or block_table.dim() != 2:
        raise RuntimeError("block_table must be an int32 CUDA tensor [B, max_pages]")
    (rows, pages), (row_stride, stride) = block_table.shape, block_table.stride()
    if pages > 1 and stride != 1:
        raise RuntimeError("block_table must have contiguous rows")
    c.page_size, c.group = page_format(pool_dev if pool_dev is not None else pool_host)
    c.kv_heads, c.batch, c.max_pages = shape[1], rows, pages
    c.block_table, c.table_stride = block_table.data_ptr(), row_stride if rows > 1 else pages
    return c


def _pool_shape(t: torch.Tensor, name: str):
    if t.dtype != torch.uint8 or t.dim() != 3 or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous uint8 [pages, kv_heads, page_bytes] tensor")
    return t.shape


def _check_tokens(positions: torch.Tensor, seq_index: torch.Tensor | None, device: int, batch: int) -> int:
    if positions.dtype != torch.int32 or positions.get_device() != device or positions.dim() != 1 \
            or not positions.is_contiguous():
        raise RuntimeError("positions must be a contiguous int32 CUDA tensor [tokens]")
    T = positions.numel()
    if seq_index is None:
        if T != batch:
            raise RuntimeError("without seq_index there is one token per sequence of the block table")
    elif seq_index.dtype != torch.int32 or seq_index.get_device() != device or seq_index.dim() != 1 \
            or seq_index.numel() != T or not seq_index.is_contiguous():
        raise RuntimeError("seq_index must be a contiguous int32 CUDA tensor [tokens]")
    return T


@traced
def rope_kv_append_q4(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor | None, q_heads: int,
                      q_out: torch.Tensor | None, pool_dev: torch.Tensor | None, pool_host: torch.Tensor | None,
                      block_table: torch.Tensor, *, seq_index: torch.Tensor | None = None, interleaved: bool = False,
                      rope_scale: float = 1.0) -> None:
    """Rotary embedding, 4-bit quantisation and append in one launch.

    ``qkv`` [tokens, (q_heads + 2 kv_heads) * 128] is the fused projection; its q
    heads are rotated into ``q_out`` [tokens, q_heads, 128] (None with q_heads 0; not
    over ``qkv``),
    its k heads rotated and quantised and its v heads quantised into slot
    ``positions[t]`` of sequence ``seq_index[t]`` (None: one token per sequence,
    in order, as in a decode step; else any tokens of a prompt).  ``inv_freq``,
    ``interleaved`` and ``rope_scale`` are ``decode_ops.rotary``'s; inv_freq None
    rotates nothing.  Two tokens of one call must not share a sequence and
    position.  The cache holds finite numbers only: a NaN is stored as code 0, the
    minimum of its group's numbers (0 in a group of nothing but NaN), and a
    group's zero and scale saturate at float16's largest value, so that a
    read-back in float16 of numbers at its very end may be infinite."""
    device = current_device_of(qkv, "qkv")
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("qkv must be a 16-bit [tokens, (q_heads + 2 kv_heads) * 128] tensor, last dim contiguous")
    c = _cache(device, pool_dev, pool_host, block_table)
    T = _check_tokens(positions, seq_index, device, c.batch)
    if inv_freq is not None:
        check_inv_freq(inv_freq, HEAD_DIM, device)
    if qkv.shape[0] != T or qkv.shape[1] != (q_heads + 2 * c.kv_heads) * HEAD_DIM:
        raise RuntimeError(f"qkv must be [{T}, {(q_heads + 2 * c.kv_heads) * HEAD_DIM}]")
    if q_heads and (q_out is None or not q_out.is_contiguous() or q_out.dtype != qkv.dtype or q_out.get_device() != device
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
    check(LIB.dak_rope_kv_append_q4(ctypes.byref(c), ctypes.byref(a), stream_of(device)), "rope_kv_append_q4")


@traced
def kv_read_q4(pool_dev: torch.Tensor | None, pool_host: torch.Tensor | None, block_table: torch.Tensor,
               positions: torch.Tensor, *, seq_index: torch.Tensor | None = None, dtype: torch.dtype = torch.float16,
               k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [tokens, kv_heads, 128] that the cache holds for the given tokens, in
    16 bits: what attention over the cache sees, for a prompt whose prefix is
    already cached.  ``k_out`` and ``v_out`` must not overlap."""
    device = current_device_of(block_table, "block_table")
    if dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("dtype must be float16 or bfloat16")
    c = _cache(device, pool_dev, pool_host, block_table)
    T = _check_tokens(positions, seq_index, device, c.batch)
    shape = (T, c.kv_heads, HEAD_DIM)
    for t, nm in ((k_out, "k_out"), (v_out, "v_out")):
        if t is not None and (t.shape != shape or t.dtype != dtype or t.get_device() != device or not t.is_contiguous()):
            raise RuntimeError(f"{nm} must be a contiguous [tokens, kv_heads, 128] tensor of dtype")
    if k_out is None:
        k_out = block_table.new_empty(shape, dtype=dtype)
    if v_out is None:
        v_out = torch.empty_like(k_out)
    if T:
        check(LIB.dak_kv_read_q4(ctypes.byref(c), positions.data_ptr(),
                                 seq_index.data_ptr() if seq_index is not None else None, k_out.data_ptr(),
                                 v_out.data_ptr(), T, dak_dtype(dtype), stream_of(device)), "kv_read_q4")
    return k_out, v_out


def merge_counter_count(batch: int, q_heads: int, kv_heads: int) -> int:
    """Entries of ``decode_paged_q4``'s merge_counters."""
    return batch * kv_heads * -(-(q_heads // kv_heads) // MAX_BLOCK_HEADS)


def scratch_floats(batch: int, q_heads: int, kv_heads: int, page_size: int, group: int, max_seq_len: int) -> int:
    """Entries of ``decode_paged_q4``'s scratch on the current device."""
    c = _lib.Kv4Cache()
    c.pool_dev, c.dev_pages, c.block_table = 16, 1, 16  # checked for presence only
    c.table_stride = c.max_pages = -(-max_seq_len // page_size)
    c.batch, c.kv_heads, c.page_size, c.group = batch, kv_heads, page_size, group
    n = LIB.dak_attn_q4_scratch(ctypes.byref(c), q_heads, max_seq_len)
    if n < 0:
        raise RuntimeError("decode_paged_q4 does not serve these sizes")
    return n


@traced
def decode_paged_q4(query: torch.Tensor, pool_dev: torch.Tensor | None, pool_host: torch.Tensor | None,
                    block_table: torch.Tensor, seq_lens: torch.Tensor, scaling: float, *,
                    out: torch.Tensor | None = None, scratch: torch.Tensor | None = None,
                    max_seq_len: int | None = None, merge_counters: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention over the 4-bit cache; returns [B, Hq, 128].

    ``query`` [B, Hq, 128], any number of query heads per KV head; ``seq_lens``
    [B] int32 on the GPU (0: the row is zeros; longer than ``max_seq_len``: cut to
    it).  ``max_seq_len`` defaults to what the block table can name; the work is
    spread over the GPU by the lengths themselves.  ``scratch``: float32,
    ``scratch_floats`` entries, allocated when not given and needed.  With
    ``merge_counters`` (int32 CUDA, ``merge_counter_count`` entries, zero before
    the first call and left zero by every call) rows that were split are merged
    inside the attention kernel instead of by a second launch; the result is the
    same.  ``out`` may be the query itself, else must not overlap it.  Calls that may overlap on the GPU need
    scratch and counters of their own."""
    device = current_device_of(query, "query")
    dtype = query.dtype
    if query.dim() != 3 or query.shape[2] != HEAD_DIM or query.stride(2) != 1:
        raise RuntimeError("query must be [B, Hq, 128] with a contiguous last dimension")
    if dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("query must be float16 or bfloat16")
    c = _cache(device, pool_dev, pool_host, block_table)
    B, Hq, _ = query.shape
    if c.batch != B:
        raise RuntimeError("block_table must have one row per sequence")
    if seq_lens.dtype != torch.int32 or seq_lens.get_device() != device or seq_lens.numel() != B \
            or not seq_lens.is_contiguous():
        raise RuntimeError("seq_lens must be a contiguous int32 CUDA tensor [B]")
    if Hq % c.kv_heads:
        raise RuntimeError("the KV heads must divide the query heads")
    if max_seq_len is None:
        max_seq_len = min(c.max_pages * c.page_size, MAX_SEQ_LEN)
    elif not 0 < max_seq_len <= min(c.max_pages * c.page_size, MAX_SEQ_LEN):
        raise RuntimeError("max_seq_len must be positive and within the block table's pages")
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    elif out.shape != query.shape or out.dtype != dtype or out.get_device() != device or out.stride(2) != 1:
        raise RuntimeError("out must be [B, Hq, 128] of the query dtype with a contiguous last dimension")
    a = _lib.AttnQ4Args()
    # A call of short rows, no more of them than SMs, takes none.
    short = max_seq_len <= SHORT_ROWS and B * Hq <= NUM_SMS
    need = 0 if short else LIB.dak_attn_q4_scratch(ctypes.byref(c), Hq, max_seq_len)
    if need > 0:
        if scratch is None:
            scratch = query.new_empty(need, dtype=torch.float32)
        elif scratch.dtype != torch.float32 or scratch.get_device() != device or scratch.numel() < need \
                or not scratch.is_contiguous():
            raise RuntimeError(f"scratch must be a contiguous float32 CUDA tensor of {need} entries")
        a.scratch, a.scratch_floats = scratch.data_ptr(), need
        if merge_counters is not None:
            if merge_counters.dtype != torch.int32 or merge_counters.get_device() != device \
                    or merge_counters.numel() < merge_counter_count(B, Hq, c.kv_heads) or not merge_counters.is_contiguous():
                raise RuntimeError("merge_counters must be a contiguous int32 CUDA tensor of merge_counter_count entries")
            a.merge_counters = merge_counters.data_ptr()
    a.query, a.seq_lens, a.out = query.data_ptr(), seq_lens.data_ptr(), out.data_ptr()
    # A dimension of one entry has no stride to speak of.
    qb, qh, _ = query.stride()
    ob, oh, _ = out.stride()
    a.q_stride_b, a.q_stride_h = qb if B > 1 else 0, qh if Hq > 1 else 0
    a.o_stride_b, a.o_stride_h = ob if B > 1 else 0, oh if Hq > 1 else 0
    a.num_q_heads, a.max_seq_len, a.scaling, a.dtype = Hq, max_seq_len, scaling, dak_dtype(dtype)
    check(LIB.dak_attn_decode_paged_q4(ctypes.byref(c), ctypes.byref(a), stream_of(device)), "decode_paged_q4")
    return out
