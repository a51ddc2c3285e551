"""Which sizes of windowed prompts a call takes, without a device: a workspace that is not aligned is looked at after them."""
from tests.test_paged_cpu import PTR, _cache
from tests.test_paged_window_cpu import _prompt
from wnw_amd import _lib


def _why(n_seg, samples, most, **kw):
    cache = _cache(n_seg=n_seg, max_blocks=1000, table_stride=1000)
    kw |= dict(T=1 << 23, B=samples, most=most, ws=PTR + 16)
    assert _prompt(cache, **kw) == _lib.WNW_EINVAL
    return _lib.lib().wnw_last_error().decode()


def test_many_segments_and_tokens():
    """8,192 samples of 8 KV heads, the longest of 4,096 tokens: 2^30 query rows in the grid; 255 blocks of 128 rows a
    segment, the most that 2^32 threads allow; twice and four times as many."""
    for kw in (dict(window=PTR), dict(window_all=100), dict(window_all=1 << 30)):
        assert "aligned" in _why(1 << 16, 1 << 13, 4096, **kw)
        assert "aligned" in _why(1 << 16, 1 << 13, 8160, **kw)
        assert "too many" in _why(1 << 16, 1 << 13, 8192, **kw)
        assert "too many" in _why(1 << 16, 1 << 13, 16384, **kw)
