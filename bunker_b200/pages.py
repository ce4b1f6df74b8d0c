"""A key/value cache in pages: the host's handle on a pool whose tables, lengths and reference counts live on the device.

The pool and its metadata are buffers of the caller (device pointers, as everywhere in this package); ``PagePool`` keeps their
description (``bkPages`` of include/bunker_cuda.h, where the rules stand) and enqueues on the library stream.  No call waits for the
GPU: whether a request was served is in its ``ok`` word on the device.
"""
from __future__ import annotations

import ctypes as C

from . import runtime as R
from .runtime import _check, cu

MAX_LIST = 1024


def scratch_bytes(n_pages: int, n_seqs: int) -> int:
    return int(R.load_library().bkPagesScratchBytes(n_pages, n_seqs))


class PagePool:
    """Pages [plane][page][head][page_rows][row_bytes] at ``base``, tables int32 [n_seqs][max_pages], ``lens`` int32 [n_seqs], ``ref``
    int32 [n_pages]; a new pool starts with lens and ref 0.  Lists (``src``, ``seqs``, ...) are device int32 arrays of n entries."""

    def __init__(self, *, base: int, n_planes: int, n_pages: int, heads: int, page_rows: int, row_bytes: int, n_seqs: int, max_pages: int,
                 ref: int, table: int, lens: int, scratch: int, scratch_bytes: int, plane_bytes: int | None = None):
        self.desc = R.bkPages(base=base, plane_bytes=n_pages * heads * page_rows * row_bytes if plane_bytes is None else plane_bytes, ref=ref,
                              table=table, lens=lens, scratch=scratch, scratch_bytes=scratch_bytes, n_planes=n_planes, n_pages=n_pages,
                              heads=heads, page_rows=page_rows, row_bytes=row_bytes, n_seqs=n_seqs, max_pages=max_pages)

    def plane(self, i: int) -> int:
        """Device pointer of plane i (what ``paged_attn_args`` takes as k_pages or v_pages)."""
        if not 0 <= i < self.desc.n_planes:
            raise IndexError(f"plane {i} of {self.desc.n_planes}")
        return self.desc.base + i * self.desc.plane_bytes

    def copy(self, to: "PagePool", src: int, dst: int, n: int) -> None:
        """Page src[i] of this pool into page dst[i] of ``to`` (may be this pool), all planes."""
        _check(cu().bkPagesCopy(C.byref(self.desc), C.byref(to.desc), src, dst, n))

    def fork(self, src: int, dst: int, n: int, ok: int = 0) -> None:
        """Empty sequence dst[i] becomes src[i]: whole pages shared, a partial last page copied."""
        _check(cu().bkPagesFork(C.byref(self.desc), src, dst, n, ok))

    def grow(self, seqs: int, add: int, n: int, ok: int = 0) -> None:
        """Room for add[i] more rows of sequence seqs[i]."""
        _check(cu().bkPagesGrow(C.byref(self.desc), seqs, add, n, ok))

    def free(self, seqs: int, n: int) -> None:
        """The sequences give up their pages."""
        _check(cu().bkPagesFree(C.byref(self.desc), seqs, n))

    def compact(self, table_out: int, ref_out: int, map_out: int, used_out: int) -> None:
        """Used pages move to the front of the pool; table_out and ref_out may be the pool's own."""
        _check(cu().bkPagesCompact(C.byref(self.desc), table_out, ref_out, map_out, used_out))

    def batch(self, seqs: int, n: int, *, T: int = 1, n_new: int = 0, parent: int = 0, table: int = 0, lens: int = 0, pos: int = 0, slot: int = 0, mask: int = 0,
              mask_words: int = 0, ok: int = 0, count: int = 0) -> None:
        """What a step over sequences seqs[0..n) with up to T new tokens each takes: their tables and lengths in the list's order, and of every token (a node of a
        drafted tree) its position, its row in the pool and the nodes on its path (bkPagesBatch).  ok: what ``grow`` said."""
        _check(cu().bkPagesBatch(C.byref(self.desc), C.byref(R.bkPagesBatchArgs(seqs, n_new, parent, table, lens, pos, slot, mask, ok, count, n, T, mask_words))))

    def commit(self, seqs: int, n: int, *, T: int, parent: int, token: int, target: int, n_new: int = 0, path: int = 0, n_path: int = 0, next: int = 0,
               ok: int = 0, history: int = 0, hist_len: int = 0, history_ld: int = 0, values: bool = False) -> None:
        """Of every drafted tree the path that agrees with target stays, the rest of its rows are given up (bkPagesCommit).  values: the targets' logits lie behind
        them, and one of -inf is no target."""
        _check(cu().bkPagesCommit(C.byref(self.desc), C.byref(R.bkPagesCommitArgs(seqs, n_new, parent, token, target, path, n_path, next, ok, history, hist_len,
                                                                                   n, T, history_ld, int(values)))))
