"""The paged cache's attention over numbers that a query must not feel: scales of
pages that no segment names, infinities in one of a segment's pieces, rows
without weight.  Tolerances as in test_gpu_paged.py, from the same bounds."""
import pytest
import torch

from tests.paged_ref import HALF, Cache, attend
from tests.test_gpu_paged import BF, FP, _check, _clean, _cu, _decode_check, _q
from wnw_amd import _lib
from wnw_amd.kv.paged import paged_decode_attn, paged_prompt_attn

pytestmark = pytest.mark.gpu


def _free_page_0(c):
    """Moves page 0's rows to a page that no segment names, if one does; True where pages are named."""
    ids = [(s, i) for s, n in enumerate(c.lens) for i in range(-(-n // c.page))]
    named = torch.zeros(c.P, dtype=torch.bool, device=c.dev)
    for s, i in ids:
        named[c.table[s, i].item()] = True
    spare = int((~named).nonzero()[-1])
    if bool(named[0]):
        for t in (c.k, c.v):
            b = t.view(torch.uint8) if c.q8 else t
            b[spare] = b[0]
        for t in (c.k_scale, c.v_scale):
            if t is not None:
                t[spare] = t[0]
        for s, i in ids:
            if c.table[s, i].item() == 0:
                c.table[s, i] = spare
        named[0], named[spare] = False, True
    return named


@pytest.mark.parametrize("dtype,D,G,page", [(BF, 128, 4, 64), (FP, 64, 2, 16), (FP, 256, 16, 32), (BF, 64, 1, 256)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -1.0])
def test_scales_of_pages_that_nobody_names(gpu, dtype, D, G, page, value):
    """A pool whose scales nobody has written yet, page 0's among them."""
    lens = [1, 16, 33, 48, 15, 32, 17, 500, 0, 2000, 9, 9]
    c = Cache(gpu, lens, page, D, dtype, True, seed=D + page)
    named = _free_page_0(c)
    q = _q(gpu, len(lens), G, D, dtype)
    few = _q(gpu, 6 * 3, 2, D, dtype)  # 3 tokens a sample of 2 heads: the decode kernel's rows
    long = _q(gpu, 6 * 30, 2 * G, D, dtype)
    calls = (lambda: paged_decode_attn(q, *c.args(), D ** -0.5, **c.scales()),
             lambda: paged_prompt_attn(few, *c.args(), _cu([3] * 6, gpu), D ** -0.5, max_tokens=3, **c.scales()),
             lambda: paged_prompt_attn(long, *c.args(), _cu([30] * 6, gpu), D ** -0.5, max_tokens=30, **c.scales()))
    c.k_scale[~named] = c.v_scale[~named] = 1.0
    want = [f() for f in calls]
    c.k_scale[~named] = c.v_scale[~named] = value
    got = [f() for f in calls]
    _clean()
    _decode_check(c, q, got[0], D ** -0.5)
    for a, b in zip(got, want):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)
    # entries that are no page: rows of zeros, whatever page 0's scale is
    c.table[9, 0], c.table[7, 0] = -1, c.P
    c.k_scale[~named] = c.v_scale[~named] = 1.0
    want = [f() for f in calls]
    c.k_scale[~named] = c.v_scale[~named] = value
    got = [f() for f in calls]
    torch.cuda.synchronize()
    assert _lib.device_error() == _lib.DEVERR_BOUNDS
    for a, b in zip(got, want):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D,G", [(BF, 128, 4), (FP, 64, 4), (BF, 256, 16), (FP, 128, 4), (BF, 64, 1)])
@pytest.mark.parametrize("n", [1, 33, 600, 9000])
def test_decode_infinities_stay_infinities(gpu, q8, dtype, D, G, n):
    """An infinity of V, with the largest weight and with small ones; 8 bits have NaN in its place."""
    c = Cache(gpu, [n], 64, D, dtype, q8, seed=n + D)
    u = torch.randn(D, device=gpu, generator=torch.Generator(device=gpu).manual_seed(5))
    u = u / u.norm() * D ** 0.5
    q = (u + 0.2 * _q(gpu, 1, G, D, dtype).float()).to(dtype)
    for d, (r, size) in enumerate([(n // 2, 3.0), (n - 1, -2.0), (0, 0.0)][:3 if n > 1 else 1]):
        p, at = c.table[0, r // 64].item(), r % 64
        if q8:
            c.k[p, at] = (u * size / c.k_scale[p]).clamp(-448, 448).to(c.k.dtype)
            c.v.view(torch.uint8)[p, at, 7 * d + 3] = 0xff
        else:
            c.k[p, at] = (u * size).to(dtype)
            c.v[p, at, 7 * d + 3] = float("-inf")
    out = paged_decode_attn(q, *c.args(), 3.0 / D, **c.scales())
    _clean()
    odd = [3, 10, 17][:3 if n > 1 else 1]
    assert bool((out[..., odd].isnan() if q8 else out[..., odd] == float("-inf")).all())
    keep = [d for d in range(D) if d not in odd]
    k, v = c.rows(0)
    ref, A = attend(q[0].double(), k, v[:, keep], torch.full((G,), n, device=gpu), 3.0 / D)
    _check(out[0][:, keep], ref, HALF[dtype] * ref.abs() + 2.0 ** -13 * A, n)


@pytest.mark.parametrize("dtype,D,G", [(BF, 128, 4), (BF, 64, 1), (BF, 256, 16), (FP, 128, 4), (FP, 256, 2)])
@pytest.mark.parametrize("n", [2, 33, 100, 1500, 20000])
def test_decode_largest_values_without_weight(gpu, dtype, D, G, n):
    """V at the type's largest number in rows whose weight is 0 in 32 bits: they add nothing."""
    c = Cache(gpu, [n, 40], 64, D, dtype, False, seed=n + D)
    u = torch.randn(D, device=gpu, generator=torch.Generator(device=gpu).manual_seed(5))
    u = u / u.norm() * D ** 0.5
    q = (u + 0.2 * _q(gpu, 2, G, D, dtype).float()).to(dtype)
    for r in {0, n // 2, n // 3} if n > 2 else {0}:
        p, at = c.table[0, r // 64].item(), r % 64
        c.k[p, at] = (u * -30).to(dtype)
        c.v[p, at] = torch.finfo(dtype).max
    out = paged_decode_attn(q, *c.args(), 10.0 / D)
    _clean()
    _decode_check(c, q, out, 10.0 / D)
