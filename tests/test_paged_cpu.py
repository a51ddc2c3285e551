"""Refusals of the paged cache's entry points that need no device: nothing is
launched, and no pointer is looked at."""
import ctypes

import pytest
import torch

from wnw_amd import _lib
from wnw_amd.kv.paged import paged_append, paged_decode_attn, paged_prompt_attn

PTR = 1 << 20


def _cache(**change):
    f = dict(k_pages=PTR, v_pages=PTR * 4, k_scale=PTR, v_scale=PTR * 8, page_table=PTR, n_seg=8, n_pages=100, max_blocks=10,
             page_rows=64, head_dim=128, k_stride=64 * 128, v_stride=64 * 128, table_stride=10, page_dtype=_lib.DT_E4M3)
    f.update(change)
    return _lib.PagedCache(*(f[n] for n, _ in _lib.PagedCache._fields_))


BAD_CACHES = [dict(page_rows=48), dict(page_rows=512), dict(head_dim=96), dict(page_dtype=_lib.DT_F32), dict(page_dtype=9),
              dict(k_scale=None), dict(v_scale=None), dict(page_dtype=_lib.DT_BF16), dict(n_seg=-1), dict(n_pages=-1),
              dict(max_blocks=-1), dict(max_blocks=1 << 30), dict(table_stride=9), dict(k_stride=64 * 128 - 16),
              dict(v_stride=64 * 128 + 8), dict(k_stride=-64 * 128), dict(page_table=None), dict(k_pages=None),
              dict(v_pages=PTR + 8), dict(n_pages=1 << 31)]


def _append(cache, **change):
    c = dict(seg_len=PTR, new_len=PTR * 2, q=PTR, k=PTR, v=PTR, q_out=PTR, strides=[4096, 128, 1024, 128, 1024, 128], T=6, B=2,
             group=4, cu=PTR, most=4, pos=PTR, pos_bits=64, pos_stride=6, freq=PTR, freq_bits=64, rot=128,
             sections=[16, 24, 24], n_sections=3, dtype=_lib.DT_BF16)
    c.update(change)
    return _lib.lib().wnw_paged_append(
        ctypes.byref(cache), c["seg_len"], c["new_len"], c["q"], c["k"], c["v"], c["q_out"], (ctypes.c_int64 * 6)(*c["strides"]),
        c["T"], c["B"], c["group"], c["cu"], c["most"], c["pos"], c["pos_bits"], c["pos_stride"], c["freq"], c["freq_bits"],
        c["rot"], (ctypes.c_int32 * 4)(*c["sections"]), c["n_sections"], 0, c["dtype"], None)


def _decode(cache, **change):
    c = dict(seg_len=PTR, q=PTR, out=PTR, group=4, scale=0.1, dtype=_lib.DT_BF16, ws=PTR, bytes=1 << 40)
    c.update(change)
    return _lib.lib().wnw_paged_decode_attn(ctypes.byref(cache), c["seg_len"], c["q"], c["out"], c["group"], c["scale"],
                                            c["dtype"], c["ws"], c["bytes"], None)


def _prompt(cache, **change):
    c = dict(seg_len=PTR, q=PTR, out=PTR, strides=[4096, 128, 4096, 128], T=600, B=2, group=4, cu=PTR, most=300, scale=0.1,
             dtype=_lib.DT_BF16, ws=PTR, bytes=1 << 40)
    c.update(change)
    return _lib.lib().wnw_paged_prompt_attn(
        ctypes.byref(cache), c["seg_len"], c["q"], c["out"], (ctypes.c_int64 * 4)(*c["strides"]), c["T"], c["B"], c["group"],
        c["cu"], c["most"], c["scale"], c["dtype"], c["ws"], c["bytes"], None)


@pytest.mark.parametrize("call", [_append, _decode, _prompt])
def test_bad_caches(call):
    for bad in BAD_CACHES:
        assert call(_cache(**bad)) == _lib.WNW_EINVAL, bad


def test_bad_appends():
    for bad in (dict(dtype=_lib.DT_F32), dict(B=3), dict(B=0), dict(T=-1), dict(T=1 << 30), dict(most=-1), dict(group=0),
                dict(seg_len=None), dict(new_len=None), dict(new_len=PTR), dict(k=None), dict(v=PTR + 2), dict(q_out=None),
                dict(strides=[4096, 128, 1024, 128, 1023, 128]), dict(strides=[-4096, 128, 1024, 128, 1024, 128]),
                dict(freq=None), dict(pos_bits=16), dict(freq_bits=16), dict(rot=24), dict(rot=0), dict(rot=256),
                dict(sections=[16, 24, 23]), dict(sections=[-16, 40, 40]), dict(n_sections=5), dict(n_sections=0),
                dict(pos_stride=5), dict(cu=None)):
        assert _append(_cache(), **bad) == _lib.WNW_EINVAL, bad
    half = dict(page_dtype=_lib.DT_F16, k_scale=None, v_scale=None)
    assert _append(_cache(**half)) == _lib.WNW_EINVAL  # bf16 rows
    assert _append(_cache(n_seg=0), B=0, T=0, cu=None) == _lib.WNW_OK


def test_bad_attention_calls():
    for call in (_decode, _prompt):
        for bad in (dict(dtype=_lib.DT_F32), dict(group=0), dict(group=2000), dict(scale=0.0), dict(scale=-1.0),
                    dict(scale=float("nan")), dict(scale=float("inf")), dict(seg_len=None), dict(q=None), dict(out=None),
                    dict(q=PTR + 8), dict(out=PTR + 2), dict(ws=PTR + 16)):
            assert call(_cache(), **bad) == _lib.WNW_EINVAL, (call, bad)
        assert call(_cache(page_dtype=_lib.DT_F16, k_scale=None, v_scale=None)) == _lib.WNW_EINVAL
    assert _decode(_cache(), group=17) == _lib.WNW_EINVAL
    assert _decode(_cache(), bytes=100) == _lib.WNW_EINVAL and _decode(_cache(), ws=None) == _lib.WNW_EINVAL
    assert _decode(_cache(n_seg=(1 << 24) - 1, max_blocks=1 << 23, table_stride=1 << 23)) == _lib.WNW_EINVAL
    assert _decode(_cache(n_seg=0)) == _lib.WNW_OK
    for bad in (dict(B=3), dict(B=0), dict(T=-1), dict(T=1 << 24), dict(most=0), dict(most=-1), dict(cu=None),
                dict(strides=[4096, 128, 4096, 127]), dict(strides=[4096, -128, 4096, 128])):
        assert _prompt(_cache(), **bad) == _lib.WNW_EINVAL, bad
    assert _prompt(_cache(), most=1, group=4, bytes=8) == _lib.WNW_EINVAL  # the decode kernel's workspace
    assert _prompt(_cache(), T=0) == _lib.WNW_OK and _prompt(_cache(n_seg=0), B=0) == _lib.WNW_OK


def test_workspace_sizes():
    l = _lib.lib()
    a = l.wnw_paged_decode_workspace_bytes(64, 4, 128)
    assert a > 0 and a % 256 == 0 and l.wnw_paged_counter_bytes(64) == l.wnw_paged_counter_bytes(4096)
    assert l.wnw_paged_decode_workspace_bytes(64, 16, 256) > a and l.wnw_paged_counter_bytes(4097) > l.wnw_paged_counter_bytes(1)
    for bad in ((-1, 4, 128), (64, 0, 128), (64, 17, 128), (64, 4, 0), (64, 4, 512)):
        assert l.wnw_paged_decode_workspace_bytes(*bad) == -1
    c = _cache()
    assert l.wnw_paged_prompt_workspace_bytes(ctypes.byref(c), 4, 2) == l.wnw_paged_decode_workspace_bytes(8, 8, 128)
    assert l.wnw_paged_prompt_workspace_bytes(ctypes.byref(c), 4, 100000) == 0  # one split: nothing to add up
    assert l.wnw_paged_prompt_workspace_bytes(ctypes.byref(c), 0, 100) == -1
    assert l.wnw_paged_prompt_workspace_bytes(ctypes.byref(_cache(head_dim=96)), 4, 100) == -1


def test_host_tensors_are_refused():
    pages = torch.zeros(4, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(_lib.WnwError):
        paged_append(x, x, pages, pages, table, lens)
    with pytest.raises(_lib.WnwError):
        paged_decode_attn(x, pages, pages, table, lens, 0.1)
    with pytest.raises(_lib.WnwError):
        paged_prompt_attn(x, pages, pages, table, lens, torch.tensor([0, 1, 2], dtype=torch.int32), 0.1)


def test_grids_past_the_launch_limit_are_refused():
    many = _cache(n_seg=1 << 23, n_pages=1 << 20)
    assert _append(many, T=1 << 24, B=1 << 20, most=64) == _lib.WNW_EINVAL
    assert _prompt(many, T=1 << 23, B=1 << 20, most=4096) == _lib.WNW_EINVAL
