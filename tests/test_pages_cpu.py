"""Refusals of the pools' operators and of beam selection that need no device."""
import ctypes

import pytest
import torch

from tests.test_paged_cpu import PTR, _cache
from wnw_amd import _lib
from wnw_amd.kv.beam import beam_select
from wnw_amd.kv.pages import paged_compact, paged_copy, paged_fork, paged_reserve

FAR = PTR << 6  # arrays of a MiB's distance: FAR * i
BAD = [dict(R=24), dict(R=512), dict(M=-1), dict(M=1 << 27), dict(stride=9), dict(nstride=9), dict(P=-1), dict(P=1 << 30),
       dict(table=None), dict(new=None), dict(refs=None), dict(nrefs=None), dict(ws=None), dict(ws=PTR + 4), dict(bytes=100),
       dict(new=FAR + 4), dict(nrefs=FAR * 3 + 4), dict(nrefs=FAR), dict(new=FAR * 3)]


def _args(change):
    c = dict(table=FAR, stride=10, lens=FAR * 2, refs=FAR * 3, parents=FAR * 4, B=4, new_B=6, H=2, M=10, P=100, R=64, new=FAR * 5,
             nstride=10, nlen=FAR * 6, nrefs=FAR * 7, copies=FAR * 8, ws=FAR * 9, bytes=1 << 20, cu=None, tokens=1, window=None, w=-1,
             sinks=None, z=0, moves=FAR * 8, used=FAR * 10)
    c.update(change)
    return c


def _fork(**change):
    c = _args(change)
    return _lib.lib().wnw_paged_fork(c["table"], c["stride"], c["lens"], c["refs"], c["parents"], c["B"], c["new_B"], c["H"], c["M"],
                                     c["P"], c["R"], c["new"], c["nstride"], c["nlen"], c["nrefs"], c["copies"], c["ws"], c["bytes"],
                                     None)


def _reserve(**change):
    c = _args(change)
    return _lib.lib().wnw_paged_reserve(c["table"], c["stride"], c["lens"], c["refs"], c["B"] * c["H"], c["B"], c["M"], c["P"], c["R"],
                                        c["cu"], c["tokens"], c["window"], c["w"], c["sinks"], c["z"], c["new"], c["nstride"],
                                        c["nrefs"], c["ws"], c["bytes"], None)


def _compact(**change):
    c = _args(change)
    return _lib.lib().wnw_paged_compact(c["table"], c["stride"], c["refs"], c["B"] * c["H"], c["M"], c["P"], c["R"], c["new"],
                                        c["nstride"], c["nrefs"], c["moves"], c["used"], c["ws"], c["bytes"], None)


@pytest.mark.parametrize("call", [_fork, _reserve, _compact])
def test_bad_pools(call):
    for bad in BAD:
        assert call(**bad) == _lib.WNW_EINVAL, bad


def test_bad_calls():
    for bad in (dict(B=-1), dict(B=8193), dict(new_B=8193), dict(new_B=-1), dict(H=0), dict(H=2000), dict(lens=None), dict(parents=None),
                dict(nlen=None), dict(copies=None), dict(nlen=FAR * 2), dict(new=FAR), dict(nrefs=FAR * 3), dict(nrefs=FAR * 2)):
        assert _fork(**bad) == _lib.WNW_EINVAL, bad
    for bad in (dict(tokens=-1), dict(tokens=(1 << 30) + 1), dict(lens=None), dict(w=5, z=-1), dict(window=PTR, z=-1),
                dict(new=FAR, nstride=11), dict(new=FAR * 2)):
        assert _reserve(**bad) == _lib.WNW_EINVAL, bad
    for bad in (dict(moves=None), dict(used=None)):
        assert _compact(**bad) == _lib.WNW_EINVAL, bad


def test_bad_copies():
    def copy(cache, at=PTR, n=3):
        return _lib.lib().wnw_paged_copy(ctypes.byref(cache), at, n, None)

    for bad in (dict(page_rows=48), dict(head_dim=96), dict(page_dtype=9), dict(k_scale=None), dict(n_pages=-1),
                dict(k_stride=64 * 128 - 16), dict(v_pages=PTR + 8)):
        assert copy(_cache(**bad)) == _lib.WNW_EINVAL, bad
    assert copy(_cache(), None) == _lib.WNW_EINVAL and copy(_cache(), n=-1) == _lib.WNW_EINVAL
    assert copy(_cache(), None, 0) == _lib.WNW_OK
    assert _lib.lib().wnw_paged_copy(None, PTR, 1, None) == _lib.WNW_EINVAL


def test_bad_selections():
    def select(**change):
        c = dict(x=FAR, strides=[400, 100], B=2, W=4, V=100, s=FAR * 2, done=None, end=0, k=4, dtype=_lib.DT_BF16, out=FAR * 3,
                 p=FAR * 4, t=FAR * 5, ws=FAR * 6, bytes=1 << 30)
        c.update(change)
        return _lib.lib().wnw_beam_select(c["x"], (ctypes.c_int64 * 2)(*c["strides"]), c["B"], c["W"], c["V"], c["s"], c["done"],
                                          c["end"], c["k"], c["dtype"], c["out"], c["p"], c["t"], c["ws"], c["bytes"], None)

    for bad in (dict(dtype=_lib.DT_E4M3), dict(dtype=7), dict(B=-1), dict(B=1 << 20), dict(W=0), dict(W=65), dict(V=0), dict(V=1 << 25),
                dict(k=0), dict(k=65), dict(end=-1), dict(end=100), dict(x=None), dict(s=None),
                dict(out=None), dict(p=None), dict(t=None), dict(ws=None), dict(ws=FAR + 4), dict(bytes=100), dict(x=FAR + 1),
                dict(strides=[-1, 100]), dict(strides=[400, 1 << 41])):
        assert select(**bad) == _lib.WNW_EINVAL, bad
    assert select(B=0) == _lib.WNW_OK
    size = _lib.lib().wnw_beam_workspace_bytes
    assert size(2, 4, 100, _lib.DT_BF16) > 0 and size(2, 4, 100, _lib.DT_E4M3) == size(2, 65, 100, 0) == size(2, 4, 0, 0) == -1


def test_host_tensors_are_refused():
    i32 = dict(dtype=torch.int32)
    table, lens, refs = torch.zeros(2, 2, **i32), torch.zeros(2, **i32), torch.zeros(4, **i32)
    pages = torch.zeros(4, 16, 64, dtype=torch.bfloat16)
    for call in (lambda: paged_fork(table, lens, refs, lens, 16, kv_heads=1), lambda: paged_reserve(table, lens, refs, 16),
                 lambda: paged_compact(table, refs, 16), lambda: paged_copy(pages, pages.clone(), torch.zeros(1, 3, **i32)),
                 lambda: beam_select(torch.zeros(1, 2, 10), torch.zeros(1, 2))):
        with pytest.raises(_lib.WnwError, match="GPU tensors"):
            call()
