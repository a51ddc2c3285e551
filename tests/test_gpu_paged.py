"""The paged cache's append, decode attention and prompt attention against
64-bit forms.

Tolerances, per element, h = half a step of the result's type (bf16 2^-8, f16
2^-11), A = sum of |weight * value|:
* decode attention: h |ref| (the result's rounding) + 2^-13 A (weights of two
  16-bit parts: 2^-15; scores of D 32-bit additions each: below 2^-14 here).
* prompt attention: h |ref| + h A (16-bit weights) + 2^-13 A, and for f16,
  whose weights are absolute below 2^-14, keys * 2^-25 of the largest |value|.
* rotation: h |ref| + 2^-21 (|a| + |b|) of the pair (four 32-bit roundings of
  products and sums, 2^-24 each, and sines off by 2^-23).
* 8-bit rows: 2^-4 |ref| + 2^-10 scale (half a step, and of subnormal codes).
"""
import pytest
import torch

from tests.paged_ref import E4M3, HALF, Cache, attend, rotate, scale_of
from wnw_amd import _lib
from wnw_amd.kv.paged import paged_append, paged_decode_attn, paged_prompt_attn

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def _check(got, ref, bound, what=""):
    got = got.double()
    bad = ~((got - ref).abs() <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - ref).abs() - bound)[bad].max()) if
                                 bool(torch.isfinite(got[bad]).all()) else "not finite", bad.nonzero()[:4].tolist())


def _decode_check(c, q, out, scale, lens=None):
    for s, n in enumerate(c.lens if lens is None else lens):
        if n == 0:
            assert int(torch.count_nonzero(out[s])) == 0, s
            continue
        k, v = c.rows(s, n)
        ref, A = attend(q[s].double(), k, v, torch.full((q.shape[1],), n, device=q.device), scale)
        _check(out[s], ref, HALF[q.dtype] * ref.abs() + 2.0 ** -13 * A, (s, n))


def _clean():
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def _q(dev, n, g, d, dtype, seed=1):
    return torch.randn(n, g, d, device=dev, generator=torch.Generator(device=dev).manual_seed(seed)).to(dtype)


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 1000, 0, 2500]


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D,G,page", [(BF, 128, 4, 64), (BF, 128, 7, 16), (FP, 128, 16, 32), (BF, 64, 1, 256),
                                            (FP, 64, 8, 16), (BF, 256, 4, 128), (FP, 256, 16, 16), (FP, 128, 2, 256)])
def test_decode(gpu, q8, dtype, D, G, page):
    c = Cache(gpu, LENS, page, D, dtype, q8, seed=D + G, joined=page == 32)
    q = _q(gpu, len(LENS), G, D, dtype)
    out = paged_decode_attn(q, *c.args(), D ** -0.5, **c.scales())
    _clean()
    assert out.shape == q.shape and out.dtype == dtype
    _decode_check(c, q, out, D ** -0.5)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("lens", [[30011], [5], [0], [0, 0, 9001, 0], [4099, 33, 0, 20000, 1], [1] * 300, list(range(700)),
                                  [i % 4 for i in range(5000)]], ids=lambda x: f"{len(x)}x{max(x)}")
def test_decode_splits(gpu, q8, lens):
    """One long segment over all workgroups, many short ones in each, more segments than threads."""
    c = Cache(gpu, lens, 64, 64, BF, q8, seed=3)
    q = _q(gpu, len(lens), 4, 64, BF)
    out = paged_decode_attn(q, *c.args(), 0.2, **c.scales())
    _clean()
    again = paged_decode_attn(q, *c.args(), 0.2, **c.scales())
    assert torch.equal(out, again)  # the pieces are added in one order
    if len(lens) > 1000:  # the segments' lengths repeat: a sample of them
        keep = list(range(0, 5000, 97)) + [1, 2, 3]
        for s in keep:
            c2 = c.rows(s) if lens[s] else None
            if c2 is None:
                assert int(torch.count_nonzero(out[s])) == 0
                continue
            ref, A = attend(q[s].double(), *c2, torch.full((4,), lens[s], device=gpu), 0.2)
            _check(out[s], ref, HALF[BF] * ref.abs() + 2.0 ** -13 * A, s)
    else:
        _decode_check(c, q, out, 0.2)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_decode_any_scales(gpu, dtype):
    """Scales that are no powers of two and differ from page to page; a page whose scales are zero."""
    lens = [700, 64, 40, 2000]
    c = Cache(gpu, lens, 32, 128, dtype, True, seed=5, scales="any")
    c.v_scale[c.table[0, 3].item()] = 0.0
    c.k_scale[c.table[3, 1].item()] = 0.0
    c.v_scale[c.table[3, 7].item()] *= 1e6
    q = _q(gpu, 4, 4, 128, dtype) * 0.3
    out = paged_decode_attn(q, *c.args(), 0.05, **c.scales())
    _clean()
    if dtype == FP:
        c.lens = lens[:3]  # the last one's values pass f16's range
    _decode_check(c, q, out, 0.05)


@pytest.mark.parametrize("q8,dtype", [(True, BF), (False, BF), (False, FP)])
def test_decode_not_finite(gpu, q8, dtype):
    """What is not finite in a segment's own rows shows in its result and in no other's; an infinity of V stays one."""
    lens = [100, 200, 300, 33]
    c = Cache(gpu, lens, 64, 128, dtype, q8, seed=6)
    q = _q(gpu, 4, 4, 128, dtype)
    where = lambda s, i: (c.table[s, i // 64].item(), i % 64)  # noqa: E731
    p, r = where(1, 150)
    if q8:
        c.v.view(torch.uint8)[p, r, 5] = 0x7f
    else:
        c.v[p, r, 5] = float("inf")
    p, r = where(2, 299)
    (c.k.view(torch.uint8) if q8 else c.k)[p, r, 9] = 0x7f if q8 else float("nan")
    out = paged_decode_attn(q, *c.args(), 0.1, **c.scales())
    _clean()
    assert bool(torch.isfinite(out[[0, 3]]).all()) and bool(out[2].isnan().all())
    assert bool(out[1, :, 5].isnan().all() if q8 else (out[1, :, 5] == float("inf")).all())
    assert bool(torch.isfinite(out[1, :, [i for i in range(128) if i != 5]]).all())


def test_decode_large_scores(gpu):
    """Scores in the thousands, rising and falling along the rows."""
    c = Cache(gpu, [900, 64], 64, 128, BF, False, seed=7)
    q = _q(gpu, 2, 4, 128, BF) * 40
    out = paged_decode_attn(q, *c.args(), 1.0)
    _clean()
    for s, n in enumerate(c.lens):
        k, v = c.rows(s)
        ref, A = attend(q[s].double(), k, v, torch.full((4,), n, device=gpu), 1.0)
        # a score of 2^11 holds 2^-13 absolute in 32 bits, 128 additions of it 2^-6 at most: as weights go
        _check(out[s], ref, HALF[BF] * ref.abs() + 2.0 ** -6 * A)


@pytest.mark.parametrize("bad", ["page", "negative", "past", "length", "below"])
@pytest.mark.parametrize("q8", [True, False])
def test_bad_tables_are_told_and_kept_apart(gpu, bad, q8):
    """A page that is none, a length past the table or below zero: the device error word, the other segments as they are."""
    lens = [200, 300, 100]
    c = Cache(gpu, lens, 32, 64, BF, q8, seed=8)
    q = _q(gpu, 3, 2, 64, BF)
    want = paged_decode_attn(q, *c.args(), 0.1, **c.scales())
    qp = _q(gpu, 60, 2, 64, BF)
    cu = torch.tensor([0, 20, 40, 60], dtype=torch.int32, device=gpu)
    wantp = paged_prompt_attn(qp, *c.args(), cu, 0.1, **c.scales())
    _clean()
    if bad in ("page", "negative"):
        c.table[1, 4] = c.P if bad == "page" else -1
    elif bad == "past":
        c.table[1, 0] = 0x7fffffff
    else:
        c.seg_len[1] = c.M * 32 + 1 if bad == "length" else -5
    out = paged_decode_attn(q, *c.args(), 0.1, **c.scales())
    torch.cuda.synchronize()
    assert _lib.device_error() & _lib.DEVERR_BOUNDS
    assert torch.equal(out[[0, 2]], want[[0, 2]]) and bool(torch.isfinite(out).all())
    if bad in ("length", "below"):
        assert int(torch.count_nonzero(out[1])) == 0
    outp = paged_prompt_attn(qp, *c.args(), cu, 0.1, **c.scales())
    torch.cuda.synchronize()
    assert _lib.device_error() & _lib.DEVERR_BOUNDS
    keep = list(range(20)) + list(range(40, 60))
    assert torch.equal(outp[keep], wantp[keep]) and bool(torch.isfinite(outp).all())


# --------------------------------------------------------------------------
# prompts
# --------------------------------------------------------------------------
def _prompt_check(c, q, out, new, H, scale):
    G = q.shape[1] // H
    start = 0
    for b, n in enumerate(new):
        for h in range(H):
            s = b * H + h
            if n == 0:
                continue
            k, v = c.rows(s)
            lim = c.lens[s] - n + torch.arange(n, device=q.device).repeat_interleave(G) + 1
            rows = q[start:start + n, h * G:(h + 1) * G].reshape(n * G, -1)
            got = out[start:start + n, h * G:(h + 1) * G].reshape(n * G, -1)
            if c.lens[s] == 0:
                assert int(torch.count_nonzero(got)) == 0
                continue
            ref, A = attend(rows.double(), k, v, lim, scale)
            hs = HALF[q.dtype]
            bound = hs * ref.abs() + (hs + 2.0 ** -13) * A
            if q.dtype == FP:
                bound = bound + c.lens[s] * 2.0 ** -25 * v.abs().max()
            _check(got, ref, bound, (b, h, n, c.lens[s]))
            assert int(torch.count_nonzero(got[lim <= 0])) == 0
        start += n


def _cu(new, dev):
    return torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=dev)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D,G,page", [(BF, 128, 4, 64), (FP, 128, 7, 16), (BF, 64, 1, 32), (FP, 64, 16, 256),
                                            (BF, 256, 2, 16), (FP, 256, 4, 64), (BF, 128, 32, 128)])
@pytest.mark.parametrize("new,old", [([1, 2, 3], [0, 70, 1]), ([33, 0, 64, 5], [0, 9, 100, 1000]), ([129, 200], [0, 333]),
                                     ([260], [4000])], ids=["few", "ragged", "longer", "split"])
def test_prompt(gpu, q8, dtype, D, G, page, new, old):
    H = 2
    lens = [o + n for o, n in zip(old, new) for _ in range(H)]
    c = Cache(gpu, lens, page, D, dtype, q8, seed=D + G + len(new), joined=page == 64)
    T = sum(new)
    q = _q(gpu, T, H * G, D, dtype)
    out = paged_prompt_attn(q, *c.args(), _cu(new, gpu), D ** -0.5, max_tokens=max(new), **c.scales())
    _clean()
    _prompt_check(c, q, out, new, H, D ** -0.5)
    wide = paged_prompt_attn(q, *c.args(), _cu(new, gpu), D ** -0.5, **c.scales())  # any grid that holds them
    _clean()
    _prompt_check(c, q, wide, new, H, D ** -0.5)


def test_prompt_longer_than_its_rows(gpu):
    """Segments that hold fewer rows than the sample has tokens (compressed ones): the first tokens see nothing."""
    c = Cache(gpu, [100, 7, 0, 64], 16, 128, BF, True, seed=11)
    for new in ([50, 20], [2, 1]):
        T = sum(new)
        c.lens = [100, 7, 0, 64] if new[0] == 50 else [1, 2, 0, 64]
        c.seg_len = torch.tensor(c.lens, dtype=torch.int32, device=gpu)
        q = _q(gpu, T, 8, 128, BF)
        out = paged_prompt_attn(q, *c.args(), _cu(new, gpu), 0.1, **c.scales())
        _clean()
        _prompt_check(c, q, out, new, 2, 0.1)


def test_prompt_any_scales(gpu):
    for dtype in (BF, FP):
        lens = [500, 400]
        c = Cache(gpu, lens, 16, 128, dtype, True, seed=12, scales="any")
        c.v_scale[c.table[0, 3].item()] = 0.0
        c.k_scale[c.table[1, 1].item()] = 0.0
        if dtype == BF:
            c.v_scale[c.table[1, 7].item()] *= 1e9
            c.v_scale[c.table[0, 0].item()] *= 1e-12
        q = _q(gpu, 90, 8, 128, dtype) * 0.3
        out = paged_prompt_attn(q, *c.args(), _cu([90], gpu), 0.05, **c.scales())
        _clean()
        _prompt_check(c, q, out, [90], 2, 0.05)


def test_prompt_rows_strided_and_left_alone(gpu):
    """q as a view of a wider projection, the result into a view; rows behind the last sample stay as they are."""
    new, H, G, D = [40, 30], 2, 4, 128
    c = Cache(gpu, [140, 140, 30, 30], 64, D, BF, True, seed=13)
    wide = torch.randn(80, (H * G + 4) * D, device=gpu).to(BF)
    q = wide[:, :H * G * D].unflatten(1, (H * G, D))
    room = torch.full((80, H * G, 2 * D), 7.0, device=gpu, dtype=BF)
    out = paged_prompt_attn(q, *c.args(), _cu(new, gpu), 0.1, max_tokens=40, out=room[..., :D], **c.scales())
    _clean()
    assert out.data_ptr() == room.data_ptr()
    _prompt_check(c, q[:70], room[:70, :, :D], new, H, 0.1)
    assert bool((room[70:] == 7).all()) and bool((room[..., D:] == 7).all())


def test_prompt_not_finite_before_its_tile(gpu):
    """A row that is not finite is seen by the tokens from its own on."""
    c = Cache(gpu, [256], 64, 128, BF, False, seed=14)
    c.v[c.table[0, 3].item(), 63, 5] = float("inf")
    q = _q(gpu, 256, 4, 128, BF)
    out = paged_prompt_attn(q, *c.args(), _cu([256], gpu), 0.1)
    _clean()
    assert bool((out[255, :, 5] == float("inf")).all()) and bool(torch.isfinite(out[:192]).all())
    c.v[c.table[0, 3].item(), 63, 5] = 0.0
    c.k[c.table[0, 3].item(), 63, 5] = float("nan")
    out = paged_prompt_attn(q, *c.args(), _cu([256], gpu), 0.1)
    _clean()
    assert bool(out[255].isnan().all()) and bool(torch.isfinite(out[:255]).all())


# --------------------------------------------------------------------------
# append
# --------------------------------------------------------------------------
def _append_case(dev, lens, new, H, G, D, page, dtype, q8, seed, axes=1, interleaved=False, rot=None, far=0, cu=True,
                 joined=False, pos32=False, freq32=False, values=None):
    c = Cache(dev, lens, page, D, dtype, q8, seed=seed, room=1 + -(-max(new) // page), joined=joined, values=values)
    g = torch.Generator(device=dev).manual_seed(seed)
    T = sum(new)
    qkv = torch.randn(T, (G + 2) * H * D, device=dev, generator=g).to(dtype)
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([H * G * D, H * D, H * D], dim=1))
    rot = D if rot is None else rot
    secs = [rot // 2] if axes == 1 else [rot // 8, rot // 4, rot // 2 - rot // 8 - rot // 4]
    pos = torch.randint(0, 2000, (axes, T), device=dev, generator=g) + far
    pos = (pos if axes > 1 else pos[0]).to(torch.int32 if pos32 else torch.int64)
    freq = (1e4 ** (-torch.arange(rot // 2, device=dev, dtype=torch.float64) / (rot // 2)))
    freq = freq.float() if freq32 else freq
    return c, q, k, v, pos, freq, secs


def _append_check(c, old, q, k, v, qo, new_len, new, H, turn):
    """The whole of the cache after an append, against ``old`` = (K, V, their scales) before."""
    dev, page = q.device, c.page
    before = c.lens
    after = [before[s] + new[s // H] for s in range(len(before))]
    assert new_len.tolist() == after
    if turn is None:
        kr, ka, qr, qa = k.double(), k.double().abs(), None, None
        assert torch.equal(qo, q)
    else:
        (kr, ka), (qr, qa) = rotate(k, *turn), rotate(q, *turn)
        _check(qo, qr, HALF[q.dtype] * qr.abs() + 2.0 ** -21 * qa, "q")
    for name, rows, size, now, was, sc, scw in (("k", kr, ka, c.k, old[0], c.k_scale, old[2]),
                                                ("v", v.double(), v.double().abs() * 0, c.v, old[1], c.v_scale, old[3])):
        now_b, was_b = (x.contiguous().view(torch.uint8 if c.q8 else torch.int16) for x in (now, was))
        touched = torch.zeros(c.P, page, dtype=torch.bool, device=dev)
        named = torch.zeros(c.P, dtype=torch.bool, device=dev)
        for s in range(len(before)):
            b, h = divmod(s, H)
            first, at = sum(new[:b]), before[s]
            while at < after[s]:
                pg, r = c.table[s, at // page].item(), at % page
                stop = min(after[s], at - r + page)
                n = stop - at
                x, a = (y[first + at - before[s]:first + at - before[s] + n, h] for y in (rows, size))
                touched[pg, r:r + n], named[pg] = True, True
                if not c.q8:
                    _check(now[pg, r:r + n], x, (HALF[c.dtype] * x.abs() + 2.0 ** -21 * a) * (1 if name == "k" else 0), name)
                else:
                    need = scale_of(x.abs().amax()).item()
                    want = max(need, scw[pg].item()) if r else need
                    big = float(x.abs().amax())
                    edge = [abs(big / (448 * 2.0 ** e) - 1) < 1e-5 for e in range(-70, 130)]
                    got = sc[pg].item()
                    assert got == want or (name == "k" and any(edge) and got in (want / 2, want * 2)), (name, s, got, want)
                    _check(now[pg, r:r + n].double() * got, x, 2.0 ** -4 * x.abs() + 2.0 ** -10 * got + 2.0 ** -21 * a, name)
                    if name == "v":
                        assert torch.equal(now_b[pg, r:r + n], (x / got).float().to(E4M3).view(torch.uint8))
                    if r:
                        moved = (was[pg, :r].float() * (scw[pg].item() / got)).to(E4M3).view(torch.uint8)
                        assert torch.equal(now_b[pg, :r], moved), (name, s)
                        touched[pg, :r] = True
                at = stop
        assert torch.equal(now_b[~touched], was_b[~touched]), name
        if c.q8:
            assert torch.equal(sc[~named], scw[~named]), name


def _snapshot(c):
    return c.k.clone(), c.v.clone(), None if c.k_scale is None else c.k_scale.clone(), \
        None if c.v_scale is None else c.v_scale.clone()


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D,G,page,opt", [
    (BF, 128, 4, 64, dict()), (FP, 128, 7, 16, dict(axes=3, pos32=True)), (BF, 64, 1, 256, dict(interleaved=True, rot=32)),
    (FP, 64, 2, 32, dict(rot=16, freq32=True)), (BF, 256, 3, 256, dict(axes=3, joined=True)),
    (FP, 256, 1, 16, dict(interleaved=True, far=10 ** 6)), (BF, 128, 4, 128, dict(axes=3, rot=64, interleaved=True))])
@pytest.mark.parametrize("new,old", [([1, 1, 1], [0, 15, 64]), ([5, 0, 40], [3, 70, 250]), ([300, 77], [0, 129]),
                                     ([1100], [31])], ids=["one", "few", "ragged", "long"])
def test_append(gpu, q8, dtype, D, G, page, opt, new, old):
    H = 2
    lens = [o + (h if o else 0) for o in old for h in range(H)]  # a sample's segments need not be equally long
    c, q, k, v, pos, freq, secs = _append_case(gpu, lens, new, H, G, D, page, dtype, q8, seed=D + G + len(new), **opt)
    was = _snapshot(c)
    qo, nl = paged_append(k, v, *c.args(), q=q, positions=pos, inv_freq=freq, sections=secs,
                          interleaved=opt.get("interleaved", False), cu_tokens=_cu(new, gpu), max_tokens=max(new), **c.scales())
    _clean()
    _append_check(c, was, q, k, v, qo, nl, new, H, (pos, freq, secs, opt.get("interleaved", False)))


@pytest.mark.parametrize("q8", [True, False])
def test_append_without_rotation_or_offsets(gpu, q8):
    """Keys that the model has rotated itself, one token per sample, no q."""
    lens, H = [0, 1, 63, 64, 65, 200], 2
    c, q, k, v, *_ = _append_case(gpu, lens, [1, 1, 1], H, 1, 128, 64, BF, q8, seed=21)
    was = _snapshot(c)
    qo, nl = paged_append(k, v, *c.args(), **c.scales())
    _clean()
    assert qo is None
    _append_check(c, was, q, k, v, q, nl, [1, 1, 1], H, None)
    c.lens, c.seg_len = nl.tolist(), nl
    was = _snapshot(c)
    room = torch.empty_like(nl)
    qo, nl = paged_append(k, v, *c.args(), q=q, new_len=room, **c.scales())
    _clean()
    assert qo is q and nl is room
    _append_check(c, was, q, k, v, q, nl, [1, 1, 1], H, None)


def test_append_rising_scales(gpu):
    """Rows that grow: the page's scale follows, the rows in it are rescaled; zero rows and tiny ones too."""
    c, q, k, v, *_ = _append_case(gpu, [0, 0], [1], 2, 1, 64, 32, BF, True, seed=22)
    for i, size in enumerate([0.0, 1e-30, 1e-4, 1.0, 0.5, 900.0, 1e4, 3.0, 1e20, 1.0, 448.0, 449.0, 1e36]):
        x, y = (torch.randn_like(t) * size for t in (k, v))
        was = _snapshot(c)
        _, nl = paged_append(x, y, *c.args(), **c.scales())
        _clean()
        _append_check(c, was, q, x, y, q, nl, [1], 2, None)
        c.lens, c.seg_len = nl.tolist(), nl
    assert c.lens == [13, 13]


def test_append_not_finite(gpu):
    """Infinities and NaN become NaN codes; the scale is that of the finite values."""
    c, q, k, v, *_ = _append_case(gpu, [0, 40], [20], 2, 1, 64, 32, BF, True, seed=23)
    v = v.clone()
    v[3, 0, 7], v[5, 1, 9], v[5, 1, 10] = float("inf"), float("nan"), float("-inf")
    clean = v.clone()
    clean[3, 0, 7] = clean[5, 1, 9] = clean[5, 1, 10] = 0.0
    _, nl = paged_append(k, v, *c.args(), cu_tokens=_cu([20], gpu), **c.scales())
    _clean()
    p0, p1 = c.table[0, 0].item(), c.table[1, 1].item()
    assert c.v_scale[p0].item() == scale_of(clean[:20, 0].abs().amax().double()).item()
    assert bool(c.v[p0, 3, 7].float().isnan()) and bool(c.v[p1, 8 + 5, 9:11].float().isnan().all())
    assert int(c.v[p0, :20].float().isnan().sum()) == 1


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("bad", ["room", "page", "length", "order", "more"])
def test_append_refused_on_the_device(gpu, q8, bad):
    """Rows past the table, in no page, of a bad length or of bad token offsets: told, and nothing else is touched."""
    new, H = [20, 20], 1
    c, q, k, v, pos, freq, secs = _append_case(gpu, [30, 30], new, H, 2, 64, 32, BF, q8, seed=24)
    cu, most = _cu(new, gpu), 20
    want = _snapshot(c)
    ref = Cache.__new__(Cache)
    ref.__dict__.update(c.__dict__)
    ref.k, ref.v, ref.k_scale, ref.v_scale = (None if x is None else x.clone() for x in want)
    paged_append(k, v, *ref.args(), cu_tokens=cu, **ref.scales())
    _clean()
    table, seg_len = c.table.clone(), c.seg_len.clone()
    if bad == "room":
        c.table = table[:, :1]
    elif bad == "page":
        c.table = table.clone()
        c.table[1, 0], c.table[1, 1] = -1, c.P
    elif bad == "length":
        c.seg_len = torch.tensor([30, -3], dtype=torch.int32, device=gpu)
    elif bad == "order":
        cu = torch.tensor([0, 20, 10], dtype=torch.int32, device=gpu)
    else:
        cu = torch.tensor([0, 0, 40], dtype=torch.int32, device=gpu)
    qo, nl = paged_append(k, v, *c.args(), q=q, positions=pos, inv_freq=freq, cu_tokens=cu, max_tokens=most, **c.scales())
    torch.cuda.synchronize()
    assert _lib.device_error() & (_lib.DEVERR_CAPACITY if bad in ("room", "length") else _lib.DEVERR_BOUNDS)
    p = table[1, 0].item(), table[1, 1].item()
    for got, old in ((c.v, want[1]), (c.k, want[0])):
        assert torch.equal(got.contiguous().view(torch.uint8)[list(p)], old.contiguous().view(torch.uint8)[list(p)])
    if bad in ("page", "length", "order"):  # the first sample is appended as ever
        p = [table[0, 0].item(), table[0, 1].item()]
        assert torch.equal(c.v.contiguous().view(torch.uint8)[p], ref.v.contiguous().view(torch.uint8)[p])


# --------------------------------------------------------------------------
# together
# --------------------------------------------------------------------------
@pytest.mark.parametrize("q8,page", [(True, 64), (False, 16)])
def test_a_run_of_them(gpu, q8, page):
    """Ragged prompts in two chunks, then steps of one token: what each attention gives is attention over the rows that
    the cache stands for at that point."""
    H, G, D, dtype = 2, 4, 128, BF
    chunks = [[70, 1, 130], [33, 64, 5]] + [[1, 1, 1]] * 5
    lens = [0] * 6
    c = Cache(gpu, [400] * 6, page, D, dtype, q8, seed=31)
    freq = 1e4 ** (-torch.arange(D // 2, device=gpu, dtype=torch.float64) / (D // 2))
    c.seg_len = torch.zeros(6, dtype=torch.int32, device=gpu)
    rows = [[] for _ in range(6)]
    for i, new in enumerate(chunks):
        T = sum(new)
        q, k, v = (torch.randn(T, n, D, device=gpu).to(dtype) for n in (H * G, H, H))
        pos = torch.cat([torch.arange(n, device=gpu) + lens[b * H] for b, n in enumerate(new)])
        qo, nl = paged_append(k, v, *c.args(), q=q, positions=pos, inv_freq=freq, cu_tokens=_cu(new, gpu), max_tokens=max(new),
                              **c.scales())
        kr = rotate(k, pos, freq, [D // 2], False)[0]
        for s in range(6):
            b, h = divmod(s, H)
            rows[s].append((kr[sum(new[:b]):sum(new[:b + 1]), h], v[sum(new[:b]):sum(new[:b + 1]), h].double()))
        lens = [x + new[s // H] for s, x in enumerate(lens)]
        c.seg_len, c.lens = nl, lens
        if max(new) == 1:
            out = paged_decode_attn(qo.view(6, G, D), *c.args(), 0.09, **c.scales())
            _clean()
            _decode_check(c, qo.view(6, G, D), out, 0.09)
            same = paged_prompt_attn(qo, *c.args(), _cu(new, gpu), 0.09, max_tokens=1, **c.scales())
            assert torch.equal(same.view(6, G, D), out)
        else:
            out = paged_prompt_attn(qo, *c.args(), _cu(new, gpu), 0.09, max_tokens=max(new), **c.scales())
            _clean()
            _prompt_check(c, qo, out, new, H, 0.09)
    for s in range(6):  # the cache stands for the rows that were appended
        for got, want in zip(c.rows(s), (torch.cat([x[i] for x in rows[s]]) for i in range(2))):
            step = 2.0 ** -4 if q8 else 2.0 ** -8
            _check(got, want, step * want.abs() + (2.0 ** -9 * 16 / 448 if q8 else 1e-5), s)


def test_graph_replays(gpu):
    """Append and attention of a step captured once: the replays follow the lengths on the device, between eager calls of
    other sizes, and equal the eager step."""
    H, G, D = 4, 4, 128
    c = Cache(gpu, [90, 700, 31, 64, 1, 1500, 255, 256], 64, D, BF, True, seed=41, room=3)
    other = Cache(gpu, [3000, 5], 32, 64, FP, True, seed=42)
    eager = Cache.__new__(Cache)
    eager.__dict__.update(c.__dict__)
    for name in ("k", "v", "k_scale", "v_scale", "seg_len"):
        setattr(eager, name, getattr(c, name).clone())
    freq = 1e4 ** (-torch.arange(D // 2, device=gpu, dtype=torch.float64) / (D // 2))
    q, k, v = (torch.zeros(2, n, D, device=gpu, dtype=BF) for n in (H * G, H, H))
    pos = torch.zeros(2, device=gpu, dtype=torch.int64)
    qo_other = _q(gpu, 2, 2, 64, FP)

    def step(x):
        qo, nl = paged_append(k, v, *x.args(), q=q, positions=pos, inv_freq=freq, **x.scales())
        out = paged_decode_attn(qo.view(2 * H, G, D), x.k, x.v, x.table, nl, 0.1, **x.scales())
        x.seg_len.copy_(nl)
        return out

    state = _snapshot(c) + (c.seg_len.clone(),)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c)
    torch.cuda.current_stream().wait_stream(side)
    for name, x in zip(("k", "v", "k_scale", "v_scale", "seg_len"), state):
        getattr(c, name).copy_(x)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same step, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c))
        graphs.append(g)
    for i in range(6):
        gen = torch.Generator(device=gpu).manual_seed(i)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device=gpu, generator=gen))
        pos.fill_(100 + i)
        graphs[i % 2].replay()
        want = step(eager)
        paged_decode_attn(qo_other, *other.args(), 0.2, **other.scales())
        if i % 3 == 0:
            torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want), i
        assert torch.equal(c.seg_len, eager.seg_len)
    _clean()
    assert torch.equal(c.k.view(torch.uint8), eager.k.view(torch.uint8)) and torch.equal(c.v_scale, eager.v_scale)


def test_streams(gpu):
    """Calls on two streams at once, each with a workspace of its own."""
    cs = [Cache(gpu, [6000 + 500 * i, 100, 3000], 64, 128, BF, True, seed=50 + i) for i in range(2)]
    qs = [_q(gpu, 3, 4, 128, BF, seed=i) for i in range(2)]
    want = [paged_decode_attn(q, *c.args(), 0.1, **c.scales()) for q, c in zip(qs, cs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(paged_decode_attn(qs[i], *cs[i].args(), 0.1, **cs[i].scales()))
    _clean()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_sizes_in_turn(gpu):
    """One workspace for calls of other segment counts, groups and head sizes: its counters stay at zero."""
    cases = [([5000, 40], 4, 128), ([300] * 70, 1, 64), ([9000], 16, 256), (list(range(0, 900, 3)), 8, 128), ([5000, 40], 4, 128)]
    for i, (lens, G, D) in enumerate(cases):
        c = Cache(gpu, lens, 64, D, FP, True, seed=60 + i)
        q = _q(gpu, len(lens), G, D, FP)
        out = paged_decode_attn(q, *c.args(), 0.1, **c.scales())
        _clean()
        _decode_check(c, q, out, 0.1)


def test_refusals(gpu):
    """Arguments that the operators do not take."""
    c = Cache(gpu, [40, 50], 32, 64, BF, True, seed=70)
    q = _q(gpu, 2, 4, 64, BF)
    k = torch.zeros(2, 1, 64, device=gpu, dtype=BF)
    cu = _cu([1, 1], gpu)
    ok = c.scales()
    E = _lib.WnwError
    for fn in (
            lambda: paged_decode_attn(q.float(), *c.args(), 0.1, **ok),
            lambda: paged_decode_attn(q[:1], *c.args(), 0.1, **ok),
            lambda: paged_decode_attn(_q(gpu, 2, 17, 64, BF), *c.args(), 0.1, **ok),
            lambda: paged_decode_attn(q, *c.args(), 0.1),
            lambda: paged_decode_attn(q, *c.args(), -0.1, **ok),
            lambda: paged_decode_attn(q, *c.args(), float("nan"), **ok),
            lambda: paged_decode_attn(q, c.k, c.v, c.table.long(), c.seg_len, 0.1, **ok),
            lambda: paged_decode_attn(q, c.k, c.v, c.table, c.seg_len[:1], 0.1, **ok),
            lambda: paged_decode_attn(q, c.k.float(), c.v.float(), c.table, c.seg_len, 0.1),
            lambda: paged_decode_attn(q, c.k[:, :24], c.v[:, :24], c.table, c.seg_len, 0.1, **ok),
            lambda: paged_decode_attn(q.requires_grad_(), *c.args(), 0.1, **ok),
            lambda: paged_decode_attn(q.detach().cpu(), *c.args(), 0.1, **ok),
            lambda: paged_prompt_attn(q.detach(), *c.args(), cu.long(), 0.1, **ok),
            lambda: paged_prompt_attn(q.detach(), *c.args(), _cu([1, 1, 0], gpu), 0.1, **ok),
            lambda: paged_prompt_attn(q.detach(), *c.args(), cu, 0.1, max_tokens=0, **ok),
            lambda: paged_prompt_attn(q.detach(), *c.args(), cu, 0.1, out=torch.empty(2, 4, 64, device=gpu), **ok),
            lambda: paged_append(k, k, *c.args(), new_len=c.seg_len, **ok),
            lambda: paged_append(k.float(), k.float(), *c.args(), **ok),
            lambda: paged_append(k, k.half(), *c.args(), **ok),
            lambda: paged_append(k[:1], k[:1], *c.args(), **ok),
            lambda: paged_append(k, k, *c.args(), positions=torch.zeros(2, device=gpu), inv_freq=torch.ones(32, device=gpu), **ok),
            lambda: paged_append(k, k, *c.args(), positions=cu[:2], inv_freq=torch.ones(20, device=gpu), **ok),
            lambda: paged_append(k, k, *c.args(), positions=cu[:2], inv_freq=torch.ones(32, device=gpu), sections=[16, 15], **ok),
            lambda: paged_append(k, k, *c.args(), inv_freq=torch.ones(32, device=gpu), **ok),
            lambda: paged_append(k, k, *c.args(), q=torch.zeros(2, 0, 64, device=gpu, dtype=BF), **ok),
    ):
        with pytest.raises(E):
            fn()
    _clean()


def test_nothing_to_do(gpu):
    """No segments, no tokens."""
    c = Cache(gpu, [40, 50], 32, 64, BF, True, seed=71)
    e = torch.zeros(0, dtype=torch.int32, device=gpu)
    t = torch.zeros(0, 3, dtype=torch.int32, device=gpu)
    assert paged_decode_attn(torch.zeros(0, 4, 64, device=gpu, dtype=BF), c.k, c.v, t, e, 0.1, **c.scales()).shape == (0, 4, 64)
    kv = torch.zeros(0, 2, 64, device=gpu, dtype=BF)
    was = _snapshot(c)
    _, nl = paged_append(kv, kv, *c.args(), cu_tokens=_cu([0], gpu), **c.scales())
    assert nl.tolist() == [40, 50] and torch.equal(c.k.view(torch.uint8), was[0].view(torch.uint8))
    _, nl = paged_append(kv, kv, c.k, c.v, t, e, **c.scales())
    assert nl.numel() == 0
    o = paged_prompt_attn(torch.zeros(0, 8, 64, device=gpu, dtype=BF), *c.args(), _cu([0], gpu), 0.1, **c.scales())
    assert o.shape == (0, 8, 64)
    _clean()
