"""Pages of a tiered KV cache: which sequence owns which, and moving them.

``copy_pages`` copies pages within HBM, within pinned host memory or between
the two, in every layer of the pools with one launch; it serves the 16-bit pools
of ``attention.decode_paged`` and the 4-bit pools of ``kv4`` alike.  ``PageTable``
is the host-side bookkeeping that decides what to copy: it hands out pages,
shares them between forked sequences, frees them and compacts the live ones.
Replaces no reference function: the reference's cache has one fixed row per
sequence (app/python/pinned_static_cache.py:8-115).
"""
from __future__ import annotations

import math
from array import array

import torch

from ._lib import LIB, check
from .decode_ops import current_device_of, stream_of
from .trace import traced

MAX_MOVES = 3584  # pages per launch


def _entries(t, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        try:
            t = array("i", t)
        except (TypeError, OverflowError) as e:
            raise RuntimeError(f"{name} must be a list or a 1-D CPU tensor of page entries ({e})") from None
        return torch.frombuffer(t, dtype=torch.int32) if t else torch.empty(0, dtype=torch.int32)
    if t.is_cuda or t.dim() != 1:
        raise RuntimeError(f"{name} must be a list or a 1-D CPU tensor of page entries")
    if t.dtype == torch.int32:
        return t if t.is_contiguous() else t.contiguous()
    if t.is_floating_point() or t.is_complex():
        raise RuntimeError(f"{name} must be a list or a 1-D CPU tensor of page entries, whole numbers")
    if t.numel() and (int(t.max()) > 2**31 - 1 or int(t.min()) < -2**31):
        raise RuntimeError(f"{name} does not fit int32")
    return t.to(torch.int32).contiguous()


@traced
def copy_pages(pool_dev: torch.Tensor | None, pool_host: torch.Tensor | None, src, dst, *, page_dim: int = 0) -> None:
    """Copies page ``src[i]`` to page ``dst[i]`` for every i (v >= 0: page v of
    ``pool_dev``, v < 0: page -1 - v of the pinned ``pool_host``).

    The pools are contiguous, with pages along ``page_dim``; every dimension
    before it (layers, K and V) is a slab in which the same pages are copied.
    ``src`` and ``dst`` are lists or CPU integer tensors and may be reused at
    once.  All copies of a call run at the same time, so a page may be copied to
    several destinations, but a destination named twice, or also as a source, is
    refused.  A host page is complete when the stream has run the copy."""
    pool = pool_dev if pool_dev is not None else pool_host
    if pool is None:
        raise RuntimeError("no KV pool given")
    if not 0 <= page_dim < pool.dim():
        raise RuntimeError("page_dim is outside the pool's dimensions")
    device = current_device_of(pool_dev, "pool_dev") if pool_dev is not None else torch.cuda.current_device()
    shape = pool.shape
    if not pool.is_contiguous():
        raise RuntimeError("the pools must be contiguous")
    if pool_host is not None:
        if pool_host.is_cuda or not pool_host.is_pinned():
            raise RuntimeError("pool_host must be pinned host memory")
        if pool_host.dtype != pool.dtype or pool_host.shape[:page_dim] != shape[:page_dim] \
                or pool_host.shape[page_dim + 1:] != shape[page_dim + 1:] or not pool_host.is_contiguous():
            raise RuntimeError("the pools must be contiguous and differ in nothing but their pages")
    src, dst = _entries(src, "src"), _entries(dst, "dst")
    n = src.numel()
    if dst.numel() != n:
        raise RuntimeError("src and dst must have the same length")
    slabs = math.prod(shape[:page_dim]) if page_dim else 1
    page = math.prod(shape[page_dim + 1:]) * pool.element_size()
    if n == 0 or slabs == 0 or page == 0:
        return
    nd = pool_dev.shape[page_dim] if pool_dev is not None else 0
    nh = pool_host.shape[page_dim] if pool_host is not None else 0
    dev = pool_dev.data_ptr() if nd else None
    host = pool_host.data_ptr() if nh else None
    if n <= MAX_MOVES:
        check(LIB.dak_copy_pages(dev, nd, host, nh, page, slabs, nd * page, nh * page, src.data_ptr(), dst.data_ptr(), n,
                                 stream_of(device)), "copy_pages")
        return
    # Several launches: what one launch refuses is refused over all of them, before the first.
    d = dst.sort().values
    if bool((d[1:] == d[:-1]).any()):
        raise RuntimeError("copy_pages: a page is a destination twice")
    if bool(torch.isin(src, dst).any()):
        raise RuntimeError("copy_pages: a page is both a source and a destination")
    both = torch.cat([src, dst])
    if int(both.max()) >= nd or int(both.min()) < -nh:
        raise RuntimeError("copy_pages: an entry is outside its pool")
    for i in range(0, n, MAX_MOVES):
        s, d = src[i:i + MAX_MOVES], dst[i:i + MAX_MOVES]
        check(LIB.dak_copy_pages(dev, nd, host, nh, page, slabs, nd * page, nh * page, s.data_ptr(), d.data_ptr(), s.numel(),
                                 stream_of(device)), "copy_pages")


class PageTable:
    """Which pages each sequence holds, on the host (no GPU work).

    Pages are named as in a block table: v >= 0 in HBM, v < 0 host page -1 - v.
    Sequences are any hashable keys.  Calls that must move data return (src, dst)
    lists for ``copy_pages``; run the copy on the stream before anything that uses
    the new rows.  A call that runs out of pages raises and changes nothing."""

    def __init__(self, dev_pages: int, host_pages: int, page_size: int):
        if dev_pages < 0 or host_pages < 0 or page_size <= 0:
            raise RuntimeError("page counts must not be negative and page_size must be positive")
        self.page_size = page_size
        self.dev_pages, self.host_pages = dev_pages, host_pages
        self._free_dev = list(range(dev_pages - 1, -1, -1))  # the lowest page is taken first
        self._free_host = list(range(-host_pages, 0))
        self._refs: dict[int, int] = {}
        self._rows: dict = {}

    def free_pages(self) -> tuple[int, int]:
        """(HBM, host) pages that nothing holds."""
        return len(self._free_dev), len(self._free_host)

    def pages(self, seq) -> list[int]:
        """The entries of a sequence, in token order."""
        return list(self._rows[seq])

    def _take(self, count: int, host: bool) -> list[int]:
        free = self._free_host if host else self._free_dev
        if count > len(free):
            raise RuntimeError(f"out of {'host' if host else 'HBM'} pages: {count} wanted, {len(free)} free")
        got = [free.pop() for _ in range(count)]
        for v in got:
            self._refs[v] = 1
        return got

    def _drop(self, v: int) -> None:
        self._refs[v] -= 1
        if self._refs[v] == 0:
            del self._refs[v]
            (self._free_host if v < 0 else self._free_dev).append(v)

    def grow(self, seq, tokens: int, host: bool = False) -> list[int]:
        """Gives ``seq`` (a new one too) pages for ``tokens`` tokens in all, the new
        ones from the given tier; returns the new entries."""
        row = self._rows.get(seq, [])
        need = -(-tokens // self.page_size) - len(row)
        new = self._take(need, host) if need > 0 else []
        self._rows[seq] = row + new
        return new

    def fork(self, seq, new, tokens: int) -> tuple[list[int], list[int]]:
        """``new`` continues ``seq`` after its first ``tokens`` tokens: full pages are
        shared, a partly filled last page is copied (to its own tier), because both
        go on writing it.  Returns the copy as (src, dst)."""
        if new in self._rows:
            raise RuntimeError(f"sequence {new!r} exists")
        row = self._rows[seq]
        full, rest = divmod(tokens, self.page_size)
        if tokens < 0 or full + (rest > 0) > len(row):
            raise RuntimeError(f"sequence {seq!r} holds fewer than {tokens} tokens")
        src = [row[full]] if rest else []
        dst = self._take(1, row[full] < 0) if rest else []
        for v in row[:full]:
            self._refs[v] += 1
        self._rows[new] = row[:full] + dst
        return src, dst

    def free(self, seq) -> None:
        """Gives back what ``seq`` holds; pages that it shares live on."""
        for v in self._rows.pop(seq):
            self._drop(v)

    def move(self, seq, first: int, count: int, host: bool) -> tuple[list[int], list[int]]:
        """Moves pages first .. first + count - 1 of ``seq`` to the given tier (those
        that lie there already stay), with every sequence that shares them; returns
        the copies as (src, dst)."""
        row = self._rows[seq]
        if first < 0 or count < 0 or first + count > len(row):
            raise RuntimeError(f"sequence {seq!r} has {len(row)} pages")
        src = [v for v in row[first:first + count] if (v < 0) != host]
        dst = self._take(len(src), host)
        self._rename(dict(zip(src, dst)))
        return src, dst

    def compact(self) -> tuple[list[int], list[int]]:
        """Moves live HBM pages so that they fill the pool from page 0 without holes;
        returns the copies as (src, dst), sources above and destinations below the
        number of live pages."""
        live = sorted(v for v in self._refs if v >= 0)
        n = len(live)
        src = [v for v in live if v >= n]
        dst = sorted(set(range(n)) - set(live))
        self._rename(dict(zip(src, dst)))
        self._free_dev = list(range(self.dev_pages - 1, n - 1, -1))
        return src, dst

    def _rename(self, to: dict[int, int]) -> None:
        for old, v in to.items():
            self._refs[v] = self._refs.pop(old)
            (self._free_host if old < 0 else self._free_dev).append(old)
        for row in self._rows.values():
            row[:] = [to.get(v, v) for v in row]

    def block_table(self, seqs, width: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """int32 [len(seqs), width] CPU table of the given sequences, entries past a
        sequence's pages 0; ``out`` (pinned, for instance) is filled when given."""
        rows = [self._rows[s] for s in seqs]
        longest = max((len(r) for r in rows), default=0)
        if out is None:
            out = torch.zeros(len(rows), max(1, longest if width is None else width), dtype=torch.int32)
        if out.dim() != 2 or out.dtype != torch.int32 or out.shape[0] != len(rows) or out.shape[1] < longest:
            raise RuntimeError(f"the table must be int32 [{len(rows)}, at least {longest}]")
        out.zero_()
        for i, r in enumerate(rows):
            out[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
        return out
