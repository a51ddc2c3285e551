"""Refusals of the windowed attention's entry points that need no device."""
import ctypes

import pytest
import torch

from tests.test_paged_cpu import BAD_CACHES, PTR, _cache
from wnw_amd import _lib
from wnw_amd.kv.paged import paged_decode_attn, paged_prompt_attn


def _decode(cache, **change):
    c = dict(seg_len=PTR, q=PTR, out=PTR, group=4, window=None, window_all=100, sinks=None, sinks_all=4, scale=0.1,
             dtype=_lib.DT_BF16, ws=PTR, bytes=1 << 40)
    c.update(change)
    return _lib.lib().wnw_paged_decode_attn_window(
        ctypes.byref(cache), c["seg_len"], c["q"], c["out"], c["group"], c["window"], c["window_all"], c["sinks"],
        c["sinks_all"], c["scale"], c["dtype"], c["ws"], c["bytes"], None)


def _prompt(cache, **change):
    c = dict(seg_len=PTR, q=PTR, out=PTR, strides=[4096, 128, 4096, 128], T=600, B=2, group=4, cu=PTR, most=300, window=None,
             window_all=100, sinks=None, sinks_all=4, scale=0.1, dtype=_lib.DT_BF16, ws=PTR, bytes=1 << 40)
    c.update(change)
    return _lib.lib().wnw_paged_prompt_attn_window(
        ctypes.byref(cache), c["seg_len"], c["q"], c["out"], (ctypes.c_int64 * 4)(*c["strides"]), c["T"], c["B"], c["group"],
        c["cu"], c["most"], c["window"], c["window_all"], c["sinks"], c["sinks_all"], c["scale"], c["dtype"], c["ws"],
        c["bytes"], None)


@pytest.mark.parametrize("call", [_decode, _prompt])
def test_refused(call):
    for bad in BAD_CACHES:
        assert call(_cache(**bad)) == _lib.WNW_EINVAL, bad
    for bad in (dict(window_all=-1), dict(sinks_all=-1), dict(window=PTR, sinks_all=-5), dict(sinks=PTR, window_all=-5),
                dict(dtype=_lib.DT_F32), dict(group=0), dict(scale=0.0), dict(seg_len=None), dict(q=None), dict(out=PTR + 2),
                dict(out=PTR + 256), dict(ws=PTR + 16)):
        assert call(_cache(), **bad) == _lib.WNW_EINVAL, bad
    assert _decode(_cache(), group=17) == _lib.WNW_EINVAL and _decode(_cache(), bytes=100) == _lib.WNW_EINVAL
    assert _decode(_cache(n_seg=0)) == _lib.WNW_OK
    assert _prompt(_cache(), T=0) == _lib.WNW_OK and _prompt(_cache(), cu=None) == _lib.WNW_EINVAL
    assert _prompt(_cache(), most=1, bytes=8) == _lib.WNW_EINVAL


def test_workspace_sizes():
    lib, c = _lib.lib(), _cache(max_blocks=1000, table_stride=1000)

    def size(cache, group, most, window=None, window_all=100, sinks=None, sinks_all=4):
        return lib.wnw_paged_prompt_window_workspace_bytes(ctypes.byref(cache), group, most, window, window_all, sinks, sinks_all)

    assert size(c, 4, 2) == lib.wnw_paged_decode_workspace_bytes(8, 8, 128)
    assert size(c, 4, 100) == 0  # a short walk is not cut
    assert size(c, 4, 100, window_all=1 << 40) == size(c, 4, 100, window=PTR) > 0  # shared out
    assert size(c, 4, 100, window_all=-1) == size(c, 0, 100) == size(_cache(head_dim=96), 4, 100) == -1


def test_host_tensors_are_refused():
    pages = torch.zeros(4, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(_lib.WnwError):
        paged_decode_attn(x, pages, pages, table, lens, 0.1, window=4)
    with pytest.raises(_lib.WnwError):
        paged_prompt_attn(x, pages, pages, table, lens, torch.tensor([0, 1, 2], dtype=torch.int32), 0.1, window=4, sinks=1)
