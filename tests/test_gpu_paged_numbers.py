"""The paged cache's attention over numbers that a query must not feel: scales of
pages that no segment names, V scales of pages that a causal mask hides or that
have no weight, values of such rows; and of infinities and the type's largest
values that it does see.  Tolerances
per element, h = half a step of the result's type, A = sum of |weight * value|
over the rows that the query sees:
* decode attention: h |ref| + 2^-13 A, as in test_gpu_paged.py;
* prompt attention: h |ref| + (h + 2^-13) A, and nothing for rows that the query
  does not see; f16 results below 2^-14 are whole multiples of 2^-24: 2^-25.
"""
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

def _rows_check(c, q, out, new, scale, tokens):
    """The first ``tokens`` tokens of one sample with one KV head, against the rows that each sees alone."""
    n, G, D = new, q.shape[1], q.shape[2]
    k, v = c.rows(0)
    lim = c.lens[0] - n + torch.arange(tokens, device=q.device).repeat_interleave(G) + 1
    most = int(lim[-1])
    ref, A = attend(q[:tokens].reshape(-1, D).double(), k[:most], v[:most], lim, scale)
    h = HALF[q.dtype]
    bound = h * ref.abs() + (h + 2.0 ** -13) * A + (2.0 ** -25 if q.dtype == FP else 0)
    _check(out[:tokens].reshape(-1, D), ref, bound, (new, tokens))


# new tokens after old rows: one tile, several, splits of a long segment, the few rows of the decode kernel
SHAPES = [(90, 0), (70, 400), (300, 700), (40, 6000), (3, 110)]
HIDDEN = [(FP, r) for r in (20, 24, 26, 30, 35, 60)] + [(BF, r) for r in (30, 60, 100, 116)]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new,old", SHAPES, ids=lambda x: str(x))
@pytest.mark.parametrize("dtype,ratio", HIDDEN, ids=lambda x: str(x).replace("torch.", ""))
def test_hidden_pages_have_no_say_in_the_scale(gpu, dtype, ratio, new, old, D):
    """V pages of later tokens 2^ratio above the others: the tokens before them give what they gave."""
    page, G = 16, 4
    c = Cache(gpu, [old + new], page, D, dtype, True, seed=D + new + ratio, room=1)
    q = _q(gpu, new, G, D, dtype)
    first = (old + new - 1) // page  # the block of the last rows
    before = first * page - old      # tokens that do not see it
    want = paged_prompt_attn(q, *c.args(), _cu([new], gpu), 0.1, **c.scales())
    c.v_scale[c.table[0, first].item()] *= 2.0 ** ratio
    got = paged_prompt_attn(q, *c.args(), _cu([new], gpu), 0.1, **c.scales())
    _clean()
    assert torch.equal(got[:before], want[:before])
    _rows_check(c, q, got, new, 0.1, before)
    if dtype == BF:  # the others see it: its values fit the result's type
        _rows_check(c, q, got, new, 0.1, new)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new,old", SHAPES, ids=lambda x: str(x))
@pytest.mark.parametrize("dtype,ratio", HIDDEN, ids=lambda x: str(x).replace("torch.", ""))
def test_pages_without_weight_have_no_say_in_the_scale(gpu, dtype, ratio, new, old, D):
    """The first block's V 2^ratio above the others' and its K against every query: seen, and of no weight."""
    page, G = 16, 4
    c = Cache(gpu, [old + new + page], page, D, dtype, True, seed=D + new + ratio)
    u = torch.randn(D, device=gpu, generator=torch.Generator(device=gpu).manual_seed(5))
    u = u / u.norm() * D ** 0.5
    q = (u + 0.2 * _q(gpu, new, G, D, dtype).float()).to(dtype)
    p = c.table[0, 0].item()
    c.k[p] = (u * -30).clamp(-448, 448).to(c.k.dtype)
    c.k_scale[p] = 1.0
    c.v_scale[p] *= 2.0 ** ratio
    scale = 10.0 / D  # the block's scores: -300 of base e
    out = paged_prompt_attn(q, *c.args(), _cu([new], gpu), scale, **c.scales())
    _clean()
    _rows_check(c, q, out, new, scale, new)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new,old", SHAPES, ids=lambda x: str(x))
@pytest.mark.parametrize("dtype,low,high", [(FP, -13, 12), (FP, -10, 10), (BF, -70, 10), (BF, -60, 118), (BF, -30, 30)],
                         ids=lambda x: str(x).replace("torch.", ""))
def test_prompt_scales_far_apart(gpu, dtype, low, high, new, old, D):
    """Every third block's V at 2^high and the others' at 2^low, all of them seen: each element to its own sum's bound."""
    page, G = 16, 4
    c = Cache(gpu, [old + new], page, D, dtype, True, seed=D + new - low)
    for i in range(-(-(old + new) // page)):
        c.v_scale[c.table[0, i].item()] *= 2.0 ** (high if i % 3 == 2 else low)
    q = _q(gpu, new, G, D, dtype)
    out = paged_prompt_attn(q, *c.args(), _cu([new], gpu), 0.1, **c.scales())
    _clean()
    _rows_check(c, q, out, new, 0.1, new)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("D,G,new,old", [(128, 4, 1, 3), (128, 4, 1, 9000), (64, 1, 3, 300), (128, 4, 90, 0), (64, 4, 300, 700),
                                         (256, 4, 60, 100), (128, 4, 40, 6000), (128, 8, 2, 20)])
def test_sums_of_the_largest_values(gpu, q8, D, G, new, old):
    """V near bf16's largest number in every row: the mean of such rows is no infinity, though their sum is."""
    c = Cache(gpu, [old + new], 64, D, BF, q8, seed=D + new + old)
    sign = torch.where(torch.arange(D, device=gpu) % 3 == 0, -1.0, 1.0)
    if q8:
        c.v.copy_((sign * 416).to(c.v.dtype).expand(c.v.shape))
        c.v_scale.fill_(2.0 ** 119)
    else:
        c.v.copy_((sign * 2.75e38).to(BF).expand(c.v.shape))
    q = _q(gpu, new, G, D, BF)
    out = paged_prompt_attn(q, *c.args(), _cu([new], gpu), 0.1, **c.scales())
    _clean()
    _rows_check(c, q, out, new, 0.1, new)
    if new == 1:
        assert torch.equal(paged_decode_attn(q, *c.args(), 0.1, **c.scales()), out)
