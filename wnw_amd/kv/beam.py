"""Beam search's selection: the k best continuations of each sample, over all of
its beams and the vocabulary.  The flat caches cannot be reordered
(src/common/kv/flat_cache.py:134-135 of the reference raises); a paged one is
forked by the parents found here (``wnw_amd.kv.pages.paged_fork``)."""
from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from .. import _lib
from .paged import _refuse_watched


def beam_select(logits: Tensor, scores: Tensor, k: int | None = None, *, done: Tensor | None = None,
                end: int = 0) -> tuple[Tensor, Tensor, Tensor]:
    """The k best of each sample's candidates (beam w, token v), best first, equal
    ones by the lower (w, v); returns (scores float32 [B, k], parents int32 [B, k],
    tokens int64 [B, k]).

    ``logits`` [B, W, V] in float32, bf16 or f16 (rows at any stride, their tokens
    contiguous; not normalised), ``scores`` float32 [B, W].  A candidate's score is
    scores[b, w] + logits[b, w, v] - log sum exp logits[b, w], formed and compared
    in 64 bits and rounded once at the end.  The log-sum is off by less than 2^-18
    (up to 2^20 tokens): the order within a beam is exact, between beams up to that.
    ``k`` is W unless given; W and k up to 64.

    ``done`` bool [B, W]: finished beams offer (their score, ``end``) alone; their
    logits are not looked at.  Logits of -inf, and beams with a score of -inf,
    offer nothing.  NaN or +inf among a beam's logits, or as its score, set the
    device error word (DEVERR_VALUES), and the beam offers nothing.

    ``parents`` are rows of a [B * W] batch, b * W + w, as ``paged_fork`` takes
    them.  Where a sample has fewer than k candidates the rest have the score
    -inf, the sample's first beam and the token ``end``."""
    native = (_lib._callpath or _lib.callpath()).beam_select(logits, scores, k, done, end)
    if native is not None:  # the plain form: checked and launched natively
        return native
    tensors = [t for t in (logits, scores, done) if t is not None]
    _refuse_watched(tensors)
    if logits.dim() != 3 or logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise _lib.WnwError(f"logits must be [B, W, V] of float32, f16 or bf16, got {tuple(logits.shape)} {logits.dtype}")
    B, W, V = logits.shape
    if scores.dtype != torch.float32 or scores.shape != (B, W):
        raise _lib.WnwError(f"scores must be float32 [{B}, {W}], got {scores.dtype} {tuple(scores.shape)}")
    if done is not None and (done.dtype != torch.bool or done.shape != (B, W)):
        raise _lib.WnwError(f"done must be bool [{B}, {W}], got {done.dtype} {tuple(done.shape)}")
    k, end = W if k is None else _lib.whole("k", k), _lib.whole("end", end)
    if logits.numel() and logits.stride(2) != 1 or any(logits.stride(i) < 0 for i in range(2)):
        logits = logits.clone(memory_format=torch.contiguous_format)
    scores = scores.contiguous()
    done = None if done is None else done.contiguous()
    need = int(_lib.lib().wnw_beam_workspace_bytes(B, W, V, _lib.dtype_code(logits.dtype)))
    if need < 0:
        raise _lib.WnwError(f"{B} samples of {W} beams over {V} tokens: below 2^20 samples, 1 to 64 beams, 1 to 2^25 - 1 tokens")
    if not 1 <= k <= 64:
        raise _lib.WnwError(f"k must be 1 to 64, got {k}")
    dev = logits.device
    out_scores = torch.empty((B, k), dtype=torch.float32, device=dev)
    parents = torch.empty((B, k), dtype=torch.int32, device=dev)
    tokens = torch.empty((B, k), dtype=torch.int64, device=dev)
    if B == 0:
        return out_scores, parents, tokens
    with torch.cuda.device(dev):
        _lib.ensure_init(dev)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.check(_lib.lib().wnw_beam_select(
            _lib.ptr(logits), (ctypes.c_int64 * 2)(logits.stride(0), logits.stride(1)), B, W, V, _lib.ptr(scores), _lib.ptr(done),
            end, k, _lib.dtype_code(logits.dtype), _lib.ptr(out_scores), _lib.ptr(parents), _lib.ptr(tokens), _lib.ptr(ws),
            ws.numel(), _lib.stream_of(dev)), "beam_select")
    return out_scores, parents, tokens
