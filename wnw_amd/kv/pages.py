"""The pages of a paged cache: samples forked and reordered, pages reserved for
the next rows and given back, a pool's used pages moved to its front.

A pool's state, beside the pages of each layer that shares it
(``wnw_amd.kv.paged``):

* ``page_table`` int32 [N, M]: the page of each block of each segment, -1 where
  there is none;
* ``seg_len`` int32 [N];
* ``page_refs`` int32 [P]: how many entries name each page (0: free, any other
  number: used).  A program may count pages of its own too, that no entry names.

Every call gives the new table and the new counts, which agree again:
``page_refs`` + the new table's entries - the old one's.  Fresh pages are the
lowest free ones, in the order of (segment, block).  Segments may share pages
that are full; a page that is partly filled is named once.

Nothing is waited for, and what depends on the data is found out on the device: a
call that cannot be done, because the free pages do not suffice or because one
of its lengths, parents or token counts is bad, sets the device error word
(``wnw_amd._lib.device_error()``: DEVERR_CAPACITY, DEVERR_BOUNDS) and changes
nothing.  Entries that are neither a page nor -1 set it too, and are taken for -1.
So does, for ``paged_compact``, an entry whose page the counts call free; the
other calls go by the counts alone, and may hand such a page out again.
"""
from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from .. import _lib
from .paged import E4M3, _PAGE_DTYPES, _refuse_watched, _tensors, _view


def _table(page_table: Tensor, page_refs: Tensor, seg_len: Tensor | None, *others: Tensor | None) -> tuple[int, int, int, int]:
    """Checks a pool's state; (N, M, P, entries from a row to the next)."""
    tensors = [t for t in (page_table, page_refs, seg_len, *others) if t is not None]
    _refuse_watched(tensors)
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise _lib.WnwError("page_table must be int32 [N, M] with contiguous rows")
    N, M = page_table.shape
    if page_refs.dtype != torch.int32 or page_refs.dim() != 1 or not page_refs.is_contiguous():
        raise _lib.WnwError("page_refs must be a contiguous int32 [P]")
    if seg_len is not None and (seg_len.dtype != torch.int32 or seg_len.shape != (N,) or not seg_len.is_contiguous()):
        raise _lib.WnwError(f"seg_len must be a contiguous int32 [{N}]")
    return N, M, page_refs.numel(), page_table.stride(0) if N > 1 else M


def _out(out: tuple[Tensor, Tensor] | None, page_table: Tensor, page_refs: Tensor) -> tuple[Tensor, Tensor, int]:
    """The new table and counts, and the table's stride."""
    N, M = page_table.shape
    if out is None:
        return page_table.new_empty((N, M)), torch.empty_like(page_refs), M
    table, refs = out
    if table.shape != page_table.shape or table.dtype != torch.int32 or (M > 1 and table.stride(1) != 1) \
            or (N > 1 and table.stride(0) < M):
        raise _lib.WnwError(f"out's table must be int32 [{N}, {M}] with contiguous rows")
    if refs.shape != page_refs.shape or refs.dtype != torch.int32 or not refs.is_contiguous():
        raise _lib.WnwError(f"out's counts must be a contiguous int32 [{page_refs.numel()}]")
    return table, refs, table.stride(0) if N > 1 else M


def _workspace(page_table: Tensor, n_seg: int, n_samples: int, n_pages: int) -> Tensor:
    need = int(_lib.lib().wnw_pages_workspace_bytes(n_seg, n_samples, n_pages))
    if need < 0:
        raise _lib.WnwError(f"too many segments or pages: {n_seg}, {n_pages}")
    return torch.empty(need, dtype=torch.uint8, device=page_table.device)


def paged_fork(page_table: Tensor, seg_len: Tensor, page_refs: Tensor, parents: Tensor, page_rows: int, *,
               kv_heads: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Reorders and copies samples, as a beam search does after each step; returns
    (new table, new lengths, new counts, copies).

    New sample i goes on from sample ``parents[i]`` (int32 [B'], of the B = N /
    ``kv_heads`` there are; -1: a sample without rows).  The first child of a
    parent takes its pages over, reserved ones too; each other child shares those
    that are full and gets a fresh page for a block that is partly filled.  Pages
    of samples that no one goes on from are given back.

    ``copies`` int32 [B' * kv_heads, 3] says what is still to be copied, (page,
    fresh page, rows) or (-1, -1, 0): ``paged_copy`` does it, once for each layer
    that shares the table.  Where the call cannot be done the new table has no
    pages and the new lengths are 0; the old ones hold.  At most 8,192 samples."""
    done = (_lib._callpath or _lib.callpath()).paged_fork(page_table, seg_len, page_refs, parents, page_rows, kv_heads)
    if done is not None:  # the plain form: checked and launched natively
        return done
    N, M, P, stride = _table(page_table, page_refs, seg_len, parents)
    if parents.dtype != torch.int32 or parents.dim() != 1 or not parents.is_contiguous():
        raise _lib.WnwError("parents must be a contiguous int32 [B']")
    kv_heads, page_rows = _lib.whole("kv_heads", kv_heads), _lib.whole("page_rows", page_rows)
    if kv_heads < 1 or N % kv_heads:
        raise _lib.WnwError(f"{N} segments are not samples x {kv_heads} KV heads")
    n_new = parents.numel()
    S = n_new * kv_heads
    new_table = page_table.new_empty((S, M))
    new_len, copies, new_refs = seg_len.new_empty(S), seg_len.new_empty((S, 3)), torch.empty_like(page_refs)
    with torch.cuda.device(page_table.device):
        _lib.ensure_init(page_table.device)
        ws = _workspace(page_table, max(N, S), N // kv_heads, P)
        _lib.check(_lib.lib().wnw_paged_fork(
            _lib.ptr(page_table), stride, _lib.ptr(seg_len), _lib.ptr(page_refs), _lib.ptr(parents), N // kv_heads, n_new,
            kv_heads, M, P, page_rows, _lib.ptr(new_table), M, _lib.ptr(new_len), _lib.ptr(new_refs), _lib.ptr(copies),
            _lib.ptr(ws), ws.numel(), _lib.stream_of(page_table.device)), "paged_fork")
    return new_table, new_len, new_refs, copies


def paged_reserve(page_table: Tensor, seg_len: Tensor, page_refs: Tensor, page_rows: int, *, tokens: int = 1,
                  cu_tokens: Tensor | None = None, window: int | Tensor | None = None, sinks: int | Tensor | None = None,
                  out: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor]:
    """Pages for the rows of the next append; returns (new table, new counts).

    Each segment gets a page for every block of its rows [seg_len, seg_len + n)
    that has none: n = ``tokens`` for all, or those of its sample, ``cu_tokens``
    int32 [B + 1] (as ``paged_append`` takes it).

    With ``window`` (and ``sinks``; as ``paged_decode_attn`` takes them) the blocks
    that neither the next row nor a later one sees are given back, for later
    calls to hand out: those behind the sinks that end at or below row seg_len + 1
    - max(window, 1) (the row at seg_len is written, whether it is seen or not).
    ``tokens`` may be 0.

    ``out``: (table, counts) to write to, which may be the given ones themselves,
    for programs and captured graphs that keep them in one place."""
    done = (_lib._callpath or _lib.callpath()).paged_reserve(page_table, seg_len, page_refs, page_rows, tokens, cu_tokens, window,
                                                             sinks, out)
    if done is not None:
        return done
    N, M, P, stride = _table(page_table, page_refs, seg_len, cu_tokens, *(out or ()), *_tensors(window, sinks))
    if cu_tokens is not None:
        if cu_tokens.dtype != torch.int32 or cu_tokens.dim() != 1 or cu_tokens.numel() < 1 or not cu_tokens.is_contiguous():
            raise _lib.WnwError("cu_tokens must be a contiguous int32 [B + 1]")
        B = cu_tokens.numel() - 1
        if (B == 0 and N) or (B and N % B):
            raise _lib.WnwError(f"{N} segments are not {B} samples x KV heads")
    else:
        B = N
    tokens, page_rows = _lib.whole("tokens", tokens), _lib.whole("page_rows", page_rows)
    if tokens < 0:
        raise _lib.WnwError("tokens must not be negative")
    if window is None and sinks is not None:
        raise _lib.WnwError("sinks need a window")
    view = (None, -1, None, 0) if window is None else _view(window, sinks, N)
    new_table, new_refs, new_stride = _out(out, page_table, page_refs)
    with torch.cuda.device(page_table.device):
        _lib.ensure_init(page_table.device)
        ws = _workspace(page_table, N, B, P)
        _lib.check(_lib.lib().wnw_paged_reserve(
            _lib.ptr(page_table), stride, _lib.ptr(seg_len), _lib.ptr(page_refs), N, B, M, P, page_rows, _lib.ptr(cu_tokens),
            tokens, *view, _lib.ptr(new_table), new_stride, _lib.ptr(new_refs), _lib.ptr(ws), ws.numel(),
            _lib.stream_of(page_table.device)), "paged_reserve")
    return new_table, new_refs


def paged_compact(page_table: Tensor, page_refs: Tensor, page_rows: int, *,
                  out: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """The used pages to the front of the pool, so that its end can go; returns
    (new table, new counts, moves, used).

    ``used`` int32 [1]: the pages in use, U.  Each one at U or above moves, in
    order, to the lowest place below U that is free: ``moves`` int32 [P // 2, 3],
    (page, its new place, page_rows), then (-1, -1, 0), for ``paged_copy``.
    ``out`` as for ``paged_reserve``."""
    done = (_lib._callpath or _lib.callpath()).paged_compact(page_table, page_refs, page_rows, out)
    if done is not None:
        return done
    N, M, P, stride = _table(page_table, page_refs, None, *(out or ()))
    page_rows = _lib.whole("page_rows", page_rows)
    new_table, new_refs, new_stride = _out(out, page_table, page_refs)
    moves, used = page_refs.new_empty((P // 2, 3)), page_refs.new_empty(1)
    with torch.cuda.device(page_table.device):
        _lib.ensure_init(page_table.device)
        ws = _workspace(page_table, N, 0, P)
        _lib.check(_lib.lib().wnw_paged_compact(
            _lib.ptr(page_table), stride, _lib.ptr(page_refs), N, M, P, page_rows, _lib.ptr(new_table), new_stride,
            _lib.ptr(new_refs), _lib.ptr(moves), _lib.ptr(used), _lib.ptr(ws), ws.numel(), _lib.stream_of(page_table.device)),
            "paged_compact")
    return new_table, new_refs, moves, used


def paged_copy(k_pages: Tensor, v_pages: Tensor, copies: Tensor, *, k_scale: Tensor | None = None,
               v_scale: Tensor | None = None) -> None:
    """Copies rows from page to page, in place: the first n rows of page src to
    page dst, of K and V, and the pages' scales, for each (src, dst, n) of
    ``copies`` int32 [C, 3].  Entries with src -1 are none; one outside the pool
    or the page sets the device error word and is left out.  No page may be dst
    twice, or both src and dst (``paged_fork``'s and ``paged_compact``'s are
    not)."""
    if (_lib._callpath or _lib.callpath()).paged_copy(k_pages, v_pages, copies, k_scale, v_scale) is not None:
        return
    tensors = [t for t in (k_pages, v_pages, copies, k_scale, v_scale) if t is not None]
    _refuse_watched(tensors)
    if k_pages.dim() != 3 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype \
            or k_pages.dtype not in _PAGE_DTYPES:
        raise _lib.WnwError(f"k_pages / v_pages must be equal [P, R, D] of bf16, f16 or e4m3: {tuple(k_pages.shape)} "
                            f"{k_pages.dtype} / {tuple(v_pages.shape)} {v_pages.dtype}")
    P, R, D = k_pages.shape
    if any(t.numel() and (t.stride(2) != 1 or t.stride(1) != D) for t in (k_pages, v_pages)):
        raise _lib.WnwError("the rows of a page must be contiguous")
    if copies.dtype != torch.int32 or copies.dim() != 2 or copies.shape[1] != 3 or not copies.is_contiguous():
        raise _lib.WnwError("copies must be a contiguous int32 [C, 3]")
    if k_pages.dtype == E4M3:
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t is None or t.dtype != torch.float32 or t.shape != (P,) or not t.is_contiguous():
                raise _lib.WnwError(f"e4m3 pages need {name}, a contiguous float32 [{P}]")
    elif k_scale is not None or v_scale is not None:
        raise _lib.WnwError("16-bit pages have no scales")
    strides = [t.stride(0) if P > 1 else R * D for t in (k_pages, v_pages)]
    cache = _lib.PagedCache(k_pages.data_ptr(), v_pages.data_ptr(), None if k_scale is None else k_scale.data_ptr(),
                            None if v_scale is None else v_scale.data_ptr(), None, 0, P, 0, R, D, *strides, 0,
                            _PAGE_DTYPES[k_pages.dtype])
    with torch.cuda.device(k_pages.device):
        _lib.ensure_init(k_pages.device)
        _lib.check(_lib.lib().wnw_paged_copy(ctypes.byref(cache), _lib.ptr(copies), copies.shape[0],
                                             _lib.stream_of(k_pages.device)), "paged_copy")
