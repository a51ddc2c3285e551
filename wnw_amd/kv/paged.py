"""A K/V cache in pages of 16 or 8 bits: append with rotation, decode
attention and prompt attention over it.

The segments are the flat cache's (segment s = b * Hkv + h holds the rows of
sequence b and KV head h; src/common/kv/flat_cache.py:46-54 of the reference,
which has no paged form), but a segment's rows lie in pages that need not be
neighbours, so it grows without being moved:

* ``k_pages`` / ``v_pages`` [P, R, D]: R = 16, 32, 64, 128 or 256 rows of D =
  64, 128 or 256 elements; bf16 / f16, or e4m3 (``torch.float8_e4m3fn``) codes;
* ``k_scale`` / ``v_scale`` float32 [P], with e4m3 pages: a code stands for
  code * scale, one positive scale (V's from 2^-80 up) for each block of R
  tokens of one head;
* ``page_table`` int32 [N, M]: row i of segment s is row i % R of page
  ``page_table[s, i // R]``; entries past a segment's rows are not read;
* ``seg_len`` int32 [N]: rows of each segment.

An append writes the pages in place and returns the new lengths in a tensor of
their own.  A page that an append writes belongs to one segment; segments that
are only read may share pages.  Lengths, table entries and token offsets live
on the device, so launches captured in a HIP graph follow them; bad ones set
the device error word (``wnw_amd._lib.device_error()``) and nothing outside the
arrays is touched.  The kernels write behind autograd's back: inputs that
require a gradient or carry a tangent are refused, and so are calls that are
being traced.
"""
from __future__ import annotations

import ctypes
from collections.abc import Sequence

import torch
from torch import Tensor
from torch.autograd import forward_ad

from .. import _lib

E4M3 = torch.float8_e4m3fn
_PAGE_DTYPES = {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16, E4M3: _lib.DT_E4M3}

# Attention workspaces of eager calls, one per (device, stream): [buffer, bytes of its counters].  The counters at
# its front are cleared once and left at zero by every launch.  A captured call gets a buffer of its own from the
# graph's memory and clears it in the graph, so graphs and eager calls on other streams never share one.
_workspaces: dict[tuple[int, int], list] = {}


_is_capturing = torch.cuda.is_current_stream_capturing


class PagedWorkspace:
    """The workspace of decode attention calls (and of prompt attention calls
    of up to 16 query rows per segment) that a program keeps itself: room for
    ``n_seg`` segments of ``rows`` query rows (heads of a group times tokens),
    cleared once, here, on the current stream.  A captured call that is given
    one needs no launch to clear its own (about 3 us).  Launches that use one
    must not overlap: give graphs or streams that run at the same time one
    each."""

    def __init__(self, n_seg: int, rows: int, head_dim: int, device: torch.device | str | int | None = None):
        if _is_capturing():
            raise _lib.WnwError("make the workspace before the capture")
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise _lib.WnwError(f"the workspace must be on a GPU, not {dev}")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        need = int(_lib.lib().wnw_paged_decode_workspace_bytes(n_seg, rows, head_dim))
        if need < 0:
            raise _lib.WnwError(f"bad workspace sizes: {n_seg} segments, {rows} rows, head_dim {head_dim}")
        self.counters = int(_lib.lib().wnw_paged_counter_bytes(n_seg))
        with torch.cuda.device(dev):
            _lib.ensure_init(dev)
            self.buf = torch.zeros(need, dtype=torch.uint8, device=dev)

    def get(self, device: torch.device, n_seg: int, need: int) -> Tensor:
        if self.buf.device != device:
            raise _lib.WnwError("the workspace is on another device")
        if self.buf.numel() < need or self.counters != int(_lib.lib().wnw_paged_counter_bytes(n_seg)):
            raise _lib.WnwError(f"the workspace is too small, or for other segment counts: {self.buf.numel()} bytes, {need} "
                                "needed")
        return self.buf


def call_workspace(idx: int, stream: int, n_seg: int, need: int) -> Tensor:
    """The workspace of an attention call on ``stream`` of device ``idx`` (the
    current one), its counters zero."""
    _lib.ensure_init_index(idx)
    counters = (n_seg + 4095) // 4096 * 16384  # wnw_paged_counter_bytes
    capturing = _is_capturing()
    held = _workspaces.get((idx, stream))
    if not capturing and held is not None and held[1] == counters and held[0].numel() >= need:
        return held[0]
    size = need if capturing or held is None else max(need, held[0].numel())
    buf = torch.empty(size, dtype=torch.uint8, device=torch.device("cuda", idx))
    _lib.check(_lib.lib().wnw_workspace_init(_lib.ptr(buf), counters, ctypes.c_void_p(stream)), "workspace init")
    if not capturing:
        _workspaces[(idx, stream)] = [buf, counters]
    return buf


def _workspace(dev: torch.device, n_seg: int, need: int, given: PagedWorkspace | None) -> Tensor | None:
    if need < 0:  # a cache that the library does not take: the call itself says why
        return None
    if given is not None:
        return given.get(dev, n_seg, need)
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    return call_workspace(idx, _lib.raw_stream(dev), n_seg, need)


def _refuse_watched(tensors: list[Tensor]) -> None:
    """Refuses tensors on the host or on several devices, and calls that autograd or a trace would have to follow."""
    _lib.require_gpu(*tensors)
    if any(t.device != tensors[0].device for t in tensors):
        raise _lib.WnwError("all tensors of a call must be on one device")
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise _lib.WnwError("the paged cache's operators have no gradient: call them under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise _lib.WnwError("the paged cache's operators have no forward-mode gradient either")
    if torch._C._get_tracing_state() is not None \
            or torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        raise _lib.WnwError("the paged cache's operators cannot be traced: a trace would hold outputs that nothing writes")


def _cache(k_pages: Tensor, v_pages: Tensor, page_table: Tensor, seg_len: Tensor, k_scale: Tensor | None,
           v_scale: Tensor | None, *others: Tensor | None) -> _lib.PagedCache:
    """The checked cache as the library takes it; ``others``: tensors of the call that share its device."""
    tensors = [t for t in (k_pages, v_pages, page_table, seg_len, k_scale, v_scale, *others) if t is not None]
    _refuse_watched(tensors)
    if k_pages.dim() != 3 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype \
            or k_pages.dtype not in _PAGE_DTYPES:
        raise _lib.WnwError(f"k_pages / v_pages must be equal [P, R, D] of bf16, f16 or e4m3: {tuple(k_pages.shape)} "
                            f"{k_pages.dtype} / {tuple(v_pages.shape)} {v_pages.dtype}")
    P, R, D = k_pages.shape
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.numel() and (t.stride(2) != 1 or t.stride(1) != D):
            raise _lib.WnwError(f"the rows of a page must be contiguous ({name})")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise _lib.WnwError("page_table must be int32 [N, M] with contiguous rows")
    N, M = page_table.shape
    if seg_len.dtype != torch.int32 or seg_len.shape != (N,) or not seg_len.is_contiguous():
        raise _lib.WnwError(f"seg_len must be a contiguous int32 [{N}]")
    if k_pages.dtype == E4M3:
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t is None or t.dtype != torch.float32 or t.shape != (P,) or not t.is_contiguous():
                raise _lib.WnwError(f"e4m3 pages need {name}, a contiguous float32 [{P}]")
    elif k_scale is not None or v_scale is not None:
        raise _lib.WnwError("16-bit pages have no scales")
    stride = [t.stride(0) if P > 1 else R * D for t in (k_pages, v_pages)]
    return _lib.PagedCache(
        k_pages.data_ptr(), v_pages.data_ptr(), None if k_scale is None else k_scale.data_ptr(),
        None if v_scale is None else v_scale.data_ptr(), page_table.data_ptr(), N, P, M, R, D, *stride,
        page_table.stride(0) if N > 1 else M, _PAGE_DTYPES[k_pages.dtype])


def _heads(name: str, t: Tensor, tokens: int | None, dim: int) -> Tensor:
    """[tokens, heads, dim] with contiguous, 16-byte aligned heads (copied where they are not)."""
    if t.dim() != 3 or t.shape[2] != dim or (tokens is not None and t.shape[0] != tokens):
        raise _lib.WnwError(f"{name} must be [{'T' if tokens is None else tokens}, heads, {dim}], got {tuple(t.shape)}")
    if t.stride(2) != 1 or t.data_ptr() % 16 or any(t.stride(i) < 0 or t.stride(i) % 8 for i in range(2)):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _tokens(cu_tokens: Tensor | None, tokens: int, n_seg: int, max_tokens: int | None) -> tuple[int, int]:
    """Samples, and the most tokens of one."""
    if cu_tokens is None:
        if max_tokens not in (None, 1):
            raise _lib.WnwError("without cu_tokens every sample has one token")
        return tokens, 1
    if cu_tokens.dtype != torch.int32 or cu_tokens.dim() != 1 or cu_tokens.numel() < 1 or not cu_tokens.is_contiguous():
        raise _lib.WnwError("cu_tokens must be a contiguous int32 [B + 1]")
    B = cu_tokens.numel() - 1
    if (B == 0 and n_seg) or (B and n_seg % B):
        raise _lib.WnwError(f"{n_seg} segments are not {B} samples x KV heads")
    if max_tokens is not None and max_tokens < 0:
        raise _lib.WnwError("max_tokens must not be negative")
    return B, tokens if max_tokens is None else min(int(max_tokens), tokens)


def paged_append(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, seg_len: Tensor, *,
                 q: Tensor | None = None, positions: Tensor | None = None, inv_freq: Tensor | None = None,
                 sections: Sequence[int] | None = None, interleaved: bool = False, cu_tokens: Tensor | None = None,
                 max_tokens: int | None = None, k_scale: Tensor | None = None, v_scale: Tensor | None = None,
                 new_len: Tensor | None = None) -> tuple[Tensor | None, Tensor]:
    """Append tokens to the pages in place, with the rotation of q and K on the
    way, in one launch; returns (q rotated, new lengths int32 [N]).

    ``k`` / ``v`` [T, Hkv, D] and ``q`` [T, Hq, D] in bf16 or f16 (any strides;
    the views of one projection need no copy).  Sample b has the tokens
    [cu_tokens[b], cu_tokens[b + 1]) (int32 [B + 1], B = N / Hkv), one each
    without ``cu_tokens``.  ``max_tokens``, the most tokens of a sample, sizes
    the grid (default T); a sample with more sets the device error word and is
    not appended.  Rows of the rotated q that belong to no such sample (tokens
    behind the last) are not written.

    ``positions`` (int64 or int32, [T] or [axes, T]) and ``inv_freq`` (float64 or
    float32, [rot / 2], rot a multiple of 16 up to D) rotate q and K: pair j by
    the angle positions[axis(j)] * inv_freq[j] (a product in 64 bits).
    ``sections``, pairs per axis, deals the pairs to up to four axes in order
    (time, height, width; default: all to one).  A pair is the elements (j,
    j + rot / 2), or (2 j, 2 j + 1) with ``interleaved``; elements from rot on
    stay as they are.  Without ``positions`` nothing is rotated and q comes back
    as it is.

    e4m3 pages: a page's scale is the least power of two that holds its rows
    (|x| <= 448 * scale, at least 2^-64), each code its value rounded once.  The
    scale only rises while a page fills; the rows already in it are rescaled
    then.  Infinities and NaN are stored as NaN and do not count.

    ``new_len``: where to put the new lengths (not ``seg_len`` itself).  16-bit
    pages must have the type of ``k``."""
    if new_len is None:  # the plain form (tensors that need no copy): checked and launched natively
        done = (_lib._callpath or _lib.callpath()).paged_append(
            k, v, k_pages, v_pages, page_table, seg_len, q, positions, inv_freq, sections, interleaved, cu_tokens, max_tokens,
            k_scale, v_scale)
        if done is not None:
            return done
    cache = _cache(k_pages, v_pages, page_table, seg_len, k_scale, v_scale, k, v, q, positions, inv_freq, cu_tokens, new_len)
    N, D = cache.n_seg, cache.head_dim
    if k.dtype not in (torch.bfloat16, torch.float16) or v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise _lib.WnwError("q, k and v must share a type, bf16 or f16")
    if k_pages.dtype not in (E4M3, k.dtype):
        raise _lib.WnwError("16-bit pages must have the type of k and v")
    k, v = _heads("k", k, None, D), _heads("v", v, k.shape[0], D)  # bound to names: must outlive the launch
    T, H = k.shape[:2]
    B, most = _tokens(cu_tokens, T, N, max_tokens)
    if v.shape[1] != H or N != B * H:
        raise _lib.WnwError(f"{N} segments are not {B} samples x {H} KV heads ({v.shape[1]} of v)")
    group = 1
    if q is not None:
        group = q.shape[1] // max(H, 1) if q.dim() == 3 else 0
        if group < 1 or q.shape[1] != group * H:
            raise _lib.WnwError(f"q must be [{T}, heads, {D}] with a multiple of {H} heads, got {tuple(q.shape)}")
    secs, rot = [], 0
    if positions is not None:
        if inv_freq is None:
            raise _lib.WnwError("positions need inv_freq")
        if inv_freq.dim() != 1 or inv_freq.dtype not in (torch.float64, torch.float32) or not inv_freq.is_contiguous():
            raise _lib.WnwError("inv_freq must be a contiguous float64 or float32 [rot / 2]")
        rot = 2 * inv_freq.numel()
        if rot % 16 or not 16 <= rot <= D:
            raise _lib.WnwError(f"the rotated part must be a multiple of 16 elements up to {D}, got {rot}")
        secs = [rot // 2] if sections is None else [int(x) for x in sections]
        if not 1 <= len(secs) <= 4 or min(secs) < 0 or sum(secs) != rot // 2:
            raise _lib.WnwError(f"sections must be one to four counts of pairs that add up to {rot // 2}, got {secs}")
        if positions.dtype not in (torch.int64, torch.int32) or positions.shape not in (
                ((T,), (1, T)) if len(secs) == 1 else ((len(secs), T),)):
            raise _lib.WnwError(f"positions must be int64 or int32 [{len(secs)}, {T}], got {positions.dtype} "
                                f"{tuple(positions.shape)}")
        if T > 1 and positions.stride(-1) != 1 or (positions.dim() == 2 and positions.stride(0) < T):
            positions = positions.clone(memory_format=torch.contiguous_format)
    elif inv_freq is not None or sections is not None:
        raise _lib.WnwError("inv_freq and sections need positions")
    q_out = None
    if q is not None and positions is not None:
        q = _heads("q", q, T, D)
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if new_len is None:
        new_len = torch.empty_like(seg_len)
    elif new_len.dtype != torch.int32 or new_len.shape != (N,) or not new_len.is_contiguous() \
            or new_len.data_ptr() == seg_len.data_ptr():
        raise _lib.WnwError(f"new_len must be a contiguous int32 [{N}] of its own")
    strides = (ctypes.c_int64 * 6)(*(x for t in (q if q_out is not None else k, k, v) for x in (t.stride(0), t.stride(1))))
    with torch.cuda.device(k.device):
        _lib.ensure_init(k.device)
        _lib.check(_lib.lib().wnw_paged_append(
            ctypes.byref(cache), _lib.ptr(seg_len), _lib.ptr(new_len), None if q_out is None else _lib.ptr(q), _lib.ptr(k),
            _lib.ptr(v), _lib.ptr(q_out), strides, T, B, group, _lib.ptr(cu_tokens), most, _lib.ptr(positions),
            0 if positions is None else 8 * positions.element_size(),
            0 if positions is None or positions.dim() == 1 else positions.stride(0), _lib.ptr(inv_freq),
            0 if inv_freq is None else 8 * inv_freq.element_size(), rot, (ctypes.c_int32 * 4)(*secs), len(secs),
            int(interleaved), _lib.dtype_code(k.dtype), _lib.stream_of(k.device)), "paged_append")
    return (q_out if q_out is not None else q), new_len


def _out(out: Tensor | None, q: Tensor) -> Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(2) != 1 or out.data_ptr() % 16 \
            or any(out.stride(i) < 0 or out.stride(i) % 8 for i in range(2)):
        raise _lib.WnwError("out must be q's shape, type and device, with contiguous, 16-byte aligned heads")
    return out


def _check_q(q: Tensor, k_pages: Tensor, scale: float) -> None:
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise _lib.WnwError(f"q must be bf16 or f16, got {q.dtype}")
    if k_pages.dtype not in (E4M3, q.dtype):
        raise _lib.WnwError("16-bit pages must have the type of q")
    if not 0 < scale < float("inf"):
        raise _lib.WnwError(f"the scale must be positive, got {scale}")


def _tensors(*args) -> list[Tensor]:
    return [x for x in args if isinstance(x, Tensor)]


def _view(window: int | Tensor, sinks: int | Tensor | None, n_seg: int) -> tuple:
    """The checked window and sinks as the library takes them: (pointer, number) each."""
    args = []
    for name, x in (("window", window), ("sinks", 0 if sinks is None else sinks)):
        if isinstance(x, Tensor):
            if x.dtype != torch.int32 or x.shape != (n_seg,) or not x.is_contiguous():
                raise _lib.WnwError(f"{name} must be a contiguous int32 [{n_seg}], or a number")
            args += [_lib.ptr(x), 0]
        else:
            if isinstance(x, bool) or not isinstance(x, int) or x < 0:
                raise _lib.WnwError(f"{name} must be a whole number, not negative, or int32 [{n_seg}], got {x!r}")
            args += [None, min(x, 1 << 30)]
    return tuple(args)


def paged_decode_attn(q_flat: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, seg_len: Tensor, scale: float, *,
                      window: int | Tensor | None = None, sinks: int | Tensor | None = None,
                      k_scale: Tensor | None = None, v_scale: Tensor | None = None, out: Tensor | None = None,
                      workspace: PagedWorkspace | None = None) -> Tensor:
    """Decode attention over the pages: ``decode_attn`` for a paged cache.

    ``q_flat`` [N, G, D] in bf16 or f16, G up to 16; returns [N, G, D].  A
    segment without rows gives zeros.  ``out``: a contiguous tensor for the
    result.  The lengths are read on the device; ``page_table.shape[1]`` bounds
    them and sizes the grid.  ``workspace``: the caller's own.

    ``window``: each segment's query rows see its last ``window`` rows and its
    first ``sinks`` (default none) alone; a number for all segments, or int32 [N],
    one for each (class-A heads a window as long as the cache, class-B heads a
    short one, in one launch).  0 leaves the sinks; a segment that shows no row
    gives zeros.  Table entries of blocks that are not seen are not read: their
    pages may have gone (``wnw_amd.kv.pages``).  Negative entries set the device
    error word and give zeros."""
    if workspace is None:
        native = _lib._callpath or _lib.callpath()
        args = (q_flat, k_pages, v_pages, page_table, seg_len, scale, k_scale, v_scale, out)
        done = native.paged_decode(*args) if window is None and sinks is None else \
            native.paged_decode_window(*args, window, sinks)
        if done is not None:
            return done
    cache = _cache(k_pages, v_pages, page_table, seg_len, k_scale, v_scale, q_flat, out, *_tensors(window, sinks))
    _check_q(q_flat, k_pages, scale)
    N, D = cache.n_seg, cache.head_dim
    if q_flat.dim() != 3 or q_flat.shape[0] != N or q_flat.shape[2] != D or not 1 <= q_flat.shape[1] <= 16:
        raise _lib.WnwError(f"q_flat must be [{N}, 1 to 16, {D}], got {tuple(q_flat.shape)}")
    q = q_flat.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    if out is not None and not out.is_contiguous():
        raise _lib.WnwError("out must be contiguous")
    if window is None and sinks is not None:
        raise _lib.WnwError("sinks need a window")
    view = () if window is None else _view(window, sinks, N)
    o = _out(out, q)
    G = q.shape[1]
    if N == 0:
        return o
    call = _lib.lib().wnw_paged_decode_attn_window if view else _lib.lib().wnw_paged_decode_attn
    with torch.cuda.device(q.device):
        _lib.ensure_init(q.device)
        ws = _workspace(q.device, N, int(_lib.lib().wnw_paged_decode_workspace_bytes(N, G, D)), workspace)
        _lib.check(call(
            ctypes.byref(cache), _lib.ptr(seg_len), _lib.ptr(q), _lib.ptr(o), G, *view, float(scale), _lib.dtype_code(q.dtype),
            _lib.ptr(ws), 0 if ws is None else ws.numel(), _lib.stream_of(q.device)), "paged_decode_attn")
    return o


def paged_prompt_attn(q: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, seg_len: Tensor, cu_tokens: Tensor,
                      scale: float, *, max_tokens: int | None = None, window: int | Tensor | None = None,
                      sinks: int | Tensor | None = None, k_scale: Tensor | None = None,
                      v_scale: Tensor | None = None, out: Tensor | None = None,
                      workspace: PagedWorkspace | None = None) -> Tensor:
    """Causal attention of prompts, or of chunks of them, over the pages that
    hold their K and V already (``paged_append`` comes first).

    ``q`` [T, Hq, D] in bf16 or f16: sample b's n tokens [cu_tokens[b],
    cu_tokens[b + 1]) are the last of its segments' ``seg_len`` rows, and token
    i of them sees the first seg_len - n + i + 1 (none: zeros).  Returns
    [T, Hq, D].  ``max_tokens``, the most tokens of a sample, sizes the grid
    (default T); a sample with more sets the device error word and its rows of
    the result are not written.  ``workspace``: the caller's own, used by calls
    of up to 16 query rows per segment (max_tokens times heads of a group).

    ``window`` and ``sinks`` as for ``paged_decode_attn``: a token at row r sees
    the rows j <= r with j < sinks or j > r - window."""
    if workspace is None:
        native = _lib._callpath or _lib.callpath()
        args = (q, k_pages, v_pages, page_table, seg_len, cu_tokens, scale, max_tokens, k_scale, v_scale, out)
        done = native.paged_prompt(*args) if window is None and sinks is None else \
            native.paged_prompt_window(*args, window, sinks)
        if done is not None:
            return done
    cache = _cache(k_pages, v_pages, page_table, seg_len, k_scale, v_scale, q, cu_tokens, out, *_tensors(window, sinks))
    _check_q(q, k_pages, scale)
    N, D = cache.n_seg, cache.head_dim
    q = _heads("q", q, None, D)
    T = q.shape[0]
    B, most = _tokens(cu_tokens, T, N, max_tokens)
    H = N // max(B, 1)
    if N and (q.shape[1] < 1 or q.shape[1] % H):
        raise _lib.WnwError(f"{q.shape[1]} query heads are not a multiple of {H} KV heads")
    if window is None and sinks is not None:
        raise _lib.WnwError("sinks need a window")
    view = () if window is None else _view(window, sinks, N)
    o = _out(out, q)
    if N == 0 or T == 0:
        return o
    if most == 0:
        raise _lib.WnwError("max_tokens is zero and there are tokens")
    G = q.shape[1] // H
    strides = (ctypes.c_int64 * 4)(q.stride(0), q.stride(1), o.stride(0), o.stride(1))
    lib = _lib.lib()
    call, size = (lib.wnw_paged_prompt_attn_window, lib.wnw_paged_prompt_window_workspace_bytes) if view else \
        (lib.wnw_paged_prompt_attn, lib.wnw_paged_prompt_workspace_bytes)
    with torch.cuda.device(q.device):
        _lib.ensure_init(q.device)
        need = int(size(ctypes.byref(cache), G, most, *view))
        if G * most <= 16:
            ws = _workspace(q.device, N, need, workspace)
        else:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
        _lib.check(call(
            ctypes.byref(cache), _lib.ptr(seg_len), _lib.ptr(q), _lib.ptr(o), strides, T, B, G, _lib.ptr(cu_tokens), most,
            *view, float(scale), _lib.dtype_code(q.dtype), _lib.ptr(ws), max(need, 0), _lib.stream_of(q.device)),
            "paged_prompt_attn")
    return o
