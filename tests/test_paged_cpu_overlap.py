"""Results that would overwrite queries other workgroups may yet read: refused
before anything is launched."""
from tests.test_paged_cpu import PTR, _cache, _decode, _prompt
from wnw_amd import _lib


def test_results_over_a_part_of_q_are_refused():
    """q itself, or rows between q's, are fine (here: up to the workspace's check)."""
    def why(call, cache, **change):
        assert call(cache, **change) == _lib.WNW_EINVAL
        return "covers" in _lib.lib().wnw_last_error().decode()

    c = _cache()  # 8 segments, groups of 4: 4,096 elements
    for apart, refused in ((0, False), (16, True), (-16, True), (256, True), (8176, True), (8192, False), (-8176, True), (-8192, False)):
        assert why(_decode, c, out=PTR + apart, bytes=0) is refused, apart
    dense = [16 * 128, 128, 16 * 128, 128]
    wide = [16 * 256, 256, 16 * 256, 256]  # 256 elements a head, of which 128 are the row
    two = [2 * 16 * 128, 128, 2 * 16 * 128, 128]  # q and out side by side in one token's row
    few = dict(T=6, B=2, group=4, most=2, bytes=0)
    for strides, apart, refused in (
            (dense, 0, False), (dense, 256, True), (dense, 16 * 256, True), (dense, 6 * 16 * 256, False), (dense, 6 * 16 * 256 - 16, True),
            (wide, 256, False), (wide, 240, True), (wide, 512, True), (wide, -256, False), (wide, 16 * 512 + 256, False),
            (two, 16 * 256, False), (two, -16 * 256, False), (two, 16 * 256 - 16, True), (two, 2 * 16 * 256, True),
            (two, 15 * 256, True), ([16 * 128, 128, 128, 6 * 128], 0, True), ([16 * 128, 128, 128, 6 * 128], 6 * 16 * 256, False)):
        assert why(_prompt, c, out=PTR + apart, strides=strides, **few) is refused, (strides, apart)
