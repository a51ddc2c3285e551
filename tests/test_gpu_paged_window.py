"""Attention over the paged cache through a sliding window with first rows that
stay visible, against its 64-bit form.  Tolerances as in test_gpu_paged.py: the
same sums over the rows that are seen.  Blocks that no row of a call sees hold
entries that are no page, and their pages NaN."""
import pytest
import torch

from tests.paged_ref import HALF, Cache
from tests.test_gpu_paged import BF, FP, _check, _clean, _cu, _q
from tests.test_gpu_paged_edges import _General
from wnw_amd import _lib
from wnw_amd.kv.paged import PagedWorkspace, paged_decode_attn, paged_prompt_attn

pytestmark = pytest.mark.gpu
ALL = 1 << 30


def _seen(n, pos, window, sinks):
    """[len(pos), n]: the rows of n that a row at pos sees."""
    j = torch.arange(n, device=pos.device)
    p = pos.unsqueeze(1)
    return (j <= p) & ((j < sinks) | (j > p - window))


def _each(x, n_seg):
    return [x] * n_seg if isinstance(x, int) else x.tolist()


def _hide(c, new, window, sinks):
    """Gives back the blocks that none of the last new[s // H] rows of segment s sees."""
    N = len(c.lens)
    H = N // len(new)
    named = set()
    for s, (w, z) in enumerate(zip(_each(window, N), _each(sinks, N))):
        n, first = c.lens[s], max(c.lens[s] - new[s // H] + 1 - w, 0)
        for j in range(-(-n // c.page)):
            if j * c.page < z or (j + 1) * c.page > first:
                named.add(int(c.table[s, j]))
            else:
                page = int(c.table[s, j])
                for pages in (c.k, c.v):
                    (pages.view(torch.uint8) if c.q8 else pages)[page] = 0x7f if c.q8 else float("nan")
                for scales in (c.k_scale, c.v_scale):
                    if scales is not None:
                        scales[page] = float("nan")
                c.table[s, j] = (-1, 0x7fffffff, -9)[j % 3]
    return named


def _clean_rows(c, s):
    """K and V of segment s in 64 bits; zeros where no page holds them."""
    keep = c.table.clone()
    c.table[(c.table < 0) | (c.table >= c.P)] = 0
    k, v = c.rows(s)
    c.table.copy_(keep)
    return k, v


def _check_rows(c, s, q, got, pos, window, sinks, scale, weights):
    """Rows q at pos against segment s; weights: 16-bit weights in the value product (prompt)."""
    if c.lens[s] == 0:
        assert int(torch.count_nonzero(got)) == 0
        return
    k, v = _clean_rows(c, s)
    seen = _seen(c.lens[s], pos, window, sinks)
    y = (q.double() @ torch.where(seen.any(0).unsqueeze(1), k, 0.0).t().contiguous() * scale).masked_fill(~seen, -torch.inf)
    e = torch.where(seen, torch.exp(y - y.amax(1, keepdim=True).clamp_min(-1e300)), 0.0)
    p = e / e.sum(1, keepdim=True).clamp_min(1e-300)
    v = torch.where(seen.any(0).unsqueeze(1), v, 0.0)
    ref, A = p @ v, p @ v.abs()
    h = HALF[q.dtype]
    bound = h * ref.abs() + (weights * h + 2.0 ** -13) * A
    if weights and q.dtype == FP:
        bound = bound + seen.sum(1, keepdim=True) * 2.0 ** -25 * v.abs().max()
    _check(got, ref, bound, (s, c.lens[s], window, sinks))
    assert int(torch.count_nonzero(got[~seen.any(1)])) == 0


def _decode_check(c, q, out, window, sinks, scale):
    N, G = q.shape[:2]
    for s, (w, z) in enumerate(zip(_each(window, N), _each(sinks, N))):
        pos = torch.full((G,), c.lens[s] - 1, device=q.device)
        _check_rows(c, s, q[s], out[s], pos, w, z, scale, 0)


def _prompt_check(c, q, out, new, window, sinks, scale):
    N = len(c.lens)
    H = N // len(new)
    G = q.shape[1] // H
    start = 0
    for b, n in enumerate(new):
        for h in range(H if n else 0):
            s = b * H + h
            pos = (c.lens[s] - n + torch.arange(n, device=q.device)).repeat_interleave(G)
            place = (slice(start, start + n), slice(h * G, (h + 1) * G))
            _check_rows(c, s, q[place].reshape(n * G, -1), out[place].reshape(n * G, -1), pos, _each(window, N)[s],
                        _each(sinks, N)[s], scale, 1)
        start += n


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 1000, 0, 2500]
VIEWS = [(1, 0), (0, 3), (0, 0), (16, 1), (31, 33), (64, 4), (124, 4), (700, 130), (5000, 0)]


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D,G,page", [(BF, 128, 4, 64), (BF, 128, 7, 16), (FP, 128, 16, 32), (BF, 64, 1, 256),
                                            (FP, 64, 8, 16), (BF, 256, 4, 128), (FP, 256, 16, 16), (FP, 128, 2, 256)])
def test_decode(gpu, q8, dtype, D, G, page):
    for i, (window, sinks) in enumerate(VIEWS):
        c = Cache(gpu, LENS, page, D, dtype, q8, seed=D + G + i, joined=page == 32)
        _hide(c, [1] * len(LENS), window, sinks)
        q = _q(gpu, len(LENS), G, D, dtype)
        out = paged_decode_attn(q, *c.args(), D ** -0.5, window=window, sinks=sinks, **c.scales())
        _clean()
        _decode_check(c, q, out, window, sinks, D ** -0.5)


def _mixed(gpu, n, seed):
    g = torch.Generator().manual_seed(seed)
    window = torch.randint(0, 300, (n,), generator=g).int()
    window[torch.rand(n, generator=g) < 0.3] = 0x7fffffff
    sinks = torch.randint(0, 70, (n,), generator=g).int()
    sinks[torch.rand(n, generator=g) < 0.1] = 0x7fffffff
    return window.to(gpu), sinks.to(gpu)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("lens", [[30011], [5], [0], [0, 0, 9001, 0], [4099, 33, 0, 20000, 1], [1] * 300, list(range(700)),
                                  [(i * 37) % 200 for i in range(2000)]], ids=lambda x: f"{len(x)}x{max(x)}")
def test_decode_splits(gpu, q8, lens):
    """Windows and sinks of each segment's own; one long segment over all workgroups, many short ones in each, more
    segments than threads."""
    N = len(lens)
    for seed in (1, 2):
        c = Cache(gpu, lens, 64, 64, BF, q8, seed=3)
        window, sinks = _mixed(gpu, N, seed + N)
        if N < 700:
            _hide(c, [1] * N, window, sinks)
        q = _q(gpu, N, 4, 64, BF)
        out = paged_decode_attn(q, *c.args(), 0.2, window=window, sinks=sinks, **c.scales())
        _clean()
        assert torch.equal(out, paged_decode_attn(q, *c.args(), 0.2, window=window, sinks=sinks, **c.scales()))
        for s in range(0, N, 1 if N < 50 else 13):
            pos = torch.full((4,), lens[s] - 1, device=gpu)
            _check_rows(c, s, q[s], out[s], pos, int(window[s]), int(sinks[s]), 0.2, 0)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D,G,page", [(BF, 128, 4, 64), (FP, 128, 7, 16), (BF, 64, 1, 32), (FP, 64, 16, 256),
                                            (BF, 256, 2, 16), (FP, 256, 4, 64), (BF, 128, 32, 128)])
@pytest.mark.parametrize("new,old", [([1, 2, 3], [0, 70, 1]), ([33, 0, 64, 5], [0, 9, 100, 1000]), ([129, 200], [0, 333]),
                                     ([260], [4000])], ids=["few", "ragged", "longer", "split"])
def test_prompt(gpu, q8, dtype, D, G, page, new, old):
    H = 2
    lens = [o + n for o, n in zip(old, new) for _ in range(H)]
    q = _q(gpu, sum(new), H * G, D, dtype)
    views = [(1, 0), (0, 5), (17, 3), (64, 64), (150, 129), (1000, 4), (0, 0), _mixed(gpu, len(lens), D + G)]
    for i, (window, sinks) in enumerate(views):
        c = Cache(gpu, lens, page, D, dtype, q8, seed=D + G + len(new) + i, joined=page == 64)
        _hide(c, new, window, sinks)
        for most in (max(new), None):  # any grid that holds them
            out = paged_prompt_attn(q, *c.args(), _cu(new, gpu), D ** -0.5, max_tokens=most, window=window, sinks=sinks,
                                    **c.scales())
            _clean()
            _prompt_check(c, q, out, new, window, sinks, D ** -0.5)


@pytest.mark.parametrize("q8", [True, False])
def test_prompt_segments_shorter_than_the_sample(gpu, q8):
    """Segments that hold fewer rows than the sample has tokens: the first tokens see nothing."""
    for new, lens in (([50, 20], [100, 7, 0, 64]), ([2, 1], [1, 2, 0, 64]), ([3], [1, 2])):
        c = Cache(gpu, lens, 16, 128, BF, q8, seed=11)
        q = _q(gpu, sum(new), 8, 128, BF)
        for window, sinks in ((5, 0), (1, 1), (0, 2), (40, 30)):
            out = paged_prompt_attn(q, *c.args(), _cu(new, gpu), 0.1, window=window, sinks=sinks, **c.scales())
            _clean()
            _prompt_check(c, q, out, new, window, sinks, 0.1)


@pytest.mark.parametrize("q8,odd", [(True, "nan"), (False, "inf"), (False, "-inf"), (False, "nan")])
@pytest.mark.parametrize("dtype,D,G", [(BF, 128, 4), (FP, 64, 1), (BF, 256, 2), (FP, 128, 16)])
@pytest.mark.parametrize("new,old,window,sinks", [(1, 200, 40, 5), (3, 150, 45, 20), (15, 117, 33, 0), (40, 170, 70, 70),
                                                  (300, 0, 100, 4), (70, 6000, 1000, 9)], ids=lambda x: str(x))
def test_v_not_finite_in_rows_that_some_see(gpu, q8, odd, dtype, D, G, new, old, window, sinks):
    """An infinity or NaN of V reaches the tokens that see its row, in its own element, and no other: rows below the
    windows beside sinks, rows that leave the window between the first token and the last, the last tokens' rows."""
    n = old + new
    c = Cache(gpu, [n, 33], 64, D, dtype, q8, seed=D + G + new)
    q = _q(gpu, new + 1, G, D, dtype)
    lo = old + 1 - window  # the first token's window starts here
    rows = sorted({n - 1, old + new // 2, max(lo + new // 2, 0), max(lo, 0), max(lo - 1, 0), sinks, max(sinks - 1, 0)})
    clean = [x.clone() for x in c.rows(0)]
    for i, r in enumerate(rows):
        p, at = c.table[0, r // 64].item(), r % 64
        if q8:
            c.v.view(torch.uint8)[p, at, 5 + i] = 0x7f if i % 2 else 0xff
        else:
            c.v[p, at, 5 + i] = float(odd)
        clean[1][r, 5 + i] = 0.0
    # what no token sees may hold anything, K too
    pos = (old + torch.arange(new, device=gpu)).repeat_interleave(G)
    seen = _seen(n, pos, window, sinks)
    for r in (~seen.any(0)).nonzero().flatten().tolist()[:40]:
        p, at = c.table[0, r // 64].item(), r % 64
        for pages in (c.k, c.v):
            (pages.view(torch.uint8) if q8 else pages)[p, at, 1] = 0x7f if q8 else float("nan")
        clean[0][r], clean[1][r] = 0.0, 0.0
    out = paged_prompt_attn(q, *c.args(), _cu([new, 1], gpu), D ** -0.5, max_tokens=new, window=window, sinks=sinks,
                            **c.scales())
    _clean()
    assert bool(torch.isfinite(out[new]).all())
    y = (q[:new].reshape(new * G, D).double() @ clean[0].t().contiguous() * D ** -0.5).masked_fill(~seen, -torch.inf)
    w = torch.softmax(y, dim=1)
    ref, A = w @ clean[1], w @ clean[1].abs()
    got = out[:new].reshape(new * G, D).clone()
    for i, r in enumerate(rows):
        x = got[seen[:, r], 5 + i]
        assert bool(x.isnan().all()) if odd == "nan" else torch.equal(x, torch.full_like(x, float(odd))), (i, r)
        got[seen[:, r], 5 + i] = ref[seen[:, r], 5 + i].to(dtype)
    h = HALF[dtype]
    bound = h * ref.abs() + (h + 2.0 ** -13) * A + (n * 2.0 ** -25 * clean[1].abs().max() if dtype == FP else 0)
    _check(got, ref, bound)


def test_bad_windows_of_a_segment(gpu):
    """A negative window, or sinks, sets the error word; the segment's rows are zeros, the others' right."""
    c = Cache(gpu, [100, 200, 300, 40], 32, 64, BF, True, seed=4)
    window = torch.tensor([50, -1, 60, 10], dtype=torch.int32, device=gpu)
    sinks = torch.tensor([4, 4, -2147483648, 0], dtype=torch.int32, device=gpu)
    q = _q(gpu, 4, 4, 64, BF)
    long = _q(gpu, 60, 8, 64, BF)
    for call in (lambda: paged_decode_attn(q, *c.args(), 0.1, window=window, sinks=sinks, **c.scales()),
                 lambda: paged_prompt_attn(long, *c.args(), _cu([30, 30], gpu), 0.1, window=window, sinks=sinks, **c.scales())):
        out = call()
        torch.cuda.synchronize()
        assert _lib.device_error() == _lib.DEVERR_BOUNDS
        if out.shape[0] == 4:
            assert int(torch.count_nonzero(out[1:3])) == 0
            for s in (0, 3):
                _check_rows(c, s, q[s], out[s], torch.full((4,), c.lens[s] - 1, device=gpu), int(window[s]), int(sinks[s]), 0.1, 0)
        else:
            assert int(torch.count_nonzero(out[:30, 4:])) == 0 and int(torch.count_nonzero(out[30:, :4])) == 0
            for s, part in ((0, (slice(0, 30), slice(0, 4))), (3, (slice(30, 60), slice(4, 8)))):
                pos = (c.lens[s] - 30 + torch.arange(30, device=gpu)).repeat_interleave(4)
                _check_rows(c, s, long[part].reshape(120, 64), out[part].reshape(120, 64), pos, int(window[s]), int(sinks[s]),
                            0.1, 1)


@pytest.mark.parametrize("tokens", [1, 60])
def test_a_seen_block_without_a_page(gpu, tokens):
    """An entry that is no page, where a row sees it: the error word, and its rows read as zeros."""
    c = Cache(gpu, [400], 32, 64, BF, False, seed=5)
    c.table[0, 11] = -1  # rows 352 .. 383
    q = _q(gpu, tokens, 4, 64, BF)
    paged_prompt_attn(q, *c.args(), _cu([tokens], gpu), 0.1, window=10, sinks=4) if tokens == 1 else None
    _clean()
    paged_prompt_attn(q, *c.args(), _cu([tokens], gpu), 0.1, window=30, sinks=4)
    torch.cuda.synchronize()
    assert _lib.device_error() == _lib.DEVERR_BOUNDS


@pytest.mark.parametrize("q8", [True, False])
def test_both_ways_into_a_call(gpu, q8, monkeypatch):
    """The native way and the general way give the same bits; a window as long as the cache the plain call's result."""
    new, lens = [3, 40, 1], [30, 30, 500, 500, 90, 90]
    c = Cache(gpu, lens, 32, 128, BF, q8, seed=8)
    q, qd = _q(gpu, 44, 8, 128, BF), _q(gpu, 6, 4, 128, BF)
    window, sinks = _mixed(gpu, 6, 9)
    results = []
    for general in (False, True):
        if general:
            monkeypatch.setattr(_lib, "_callpath", _General())
        ws = PagedWorkspace(6, 16, 128)
        for w, z in ((20, 3), (window, 3), (window, sinks), (ALL, None), (1 << 40, 0)):
            results.append([paged_prompt_attn(q, *c.args(), _cu(new, gpu), 0.1, window=w, sinks=z, **c.scales()),
                            paged_decode_attn(qd, *c.args(), 0.1, window=w, sinks=z, **c.scales()),
                            paged_decode_attn(qd, *c.args(), 0.1, window=w, sinks=z, workspace=ws, **c.scales())])
    _clean()
    for a, b in zip(results[:5], results[5:]):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    monkeypatch.undo()
    _prompt_check(c, q, results[3][0], new, ALL, 0, 0.1)
    _decode_check(c, qd, results[3][1], ALL, 0, 0.1)


def test_captured(gpu):
    """A captured decode and prompt follow lengths, windows and tables that change between replays; a second graph with a
    workspace of its own runs in turn with it."""
    lens = [700, 90, 33, 1500]
    c = Cache(gpu, lens, 32, 64, BF, True, seed=9)
    q, qp = _q(gpu, 4, 4, 64, BF), _q(gpu, 50, 8, 64, BF)
    window, sinks = torch.full((4,), 100, dtype=torch.int32, device=gpu), torch.full((4,), 4, dtype=torch.int32, device=gpu)
    cu, few = _cu([30, 20], gpu), _cu([2, 1], gpu)

    def run():
        return (paged_decode_attn(q, *c.args(), 0.1, window=window, sinks=sinks, **c.scales()),
                paged_prompt_attn(qp, *c.args(), cu, 0.1, window=window, sinks=sinks, **c.scales()),
                paged_prompt_attn(qp[:3], *c.args(), few, 0.1, max_tokens=3, window=64, sinks=2, **c.scales()))
    run()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    for step in range(4):
        c.seg_len.copy_(torch.tensor([n - step for n in lens], dtype=torch.int32))
        window.fill_(100 - 30 * step)
        sinks.fill_(step)
        c.lens = [n - step for n in lens]
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = run()
        for g, out in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, want))
        _decode_check(c, q, graphs[0][1][0], window, sinks, 0.1)
        _prompt_check(c, qp, graphs[0][1][1], [30, 20], window, sinks, 0.1)
    _clean()


def test_rows_strided_and_left_alone(gpu):
    """q as a view of a wider projection, the result into a view; rows behind the last sample stay as they are."""
    new, H, G, D = [40, 30], 2, 4, 128
    c = Cache(gpu, [140, 140, 30, 30], 64, D, BF, True, seed=13)
    wide = torch.randn(80, (H * G + 4) * D, device=gpu).to(BF)
    q = wide[:, :H * G * D].unflatten(1, (H * G, D))
    room = torch.full((80, H * G, 2 * D), 7.0, device=gpu, dtype=BF)
    paged_prompt_attn(q, *c.args(), _cu(new, gpu), 0.1, max_tokens=40, window=25, sinks=2, out=room[..., :D], **c.scales())
    _clean()
    _prompt_check(c, q[:70], room[:70, :, :D], new, 25, 2, 0.1)
    assert bool((room[70:] == 7).all()) and bool((room[..., D:] == 7).all())


def test_another_stream(gpu):
    c = Cache(gpu, [5000, 300, 20, 7000], 64, 64, BF, True, seed=15)
    q = _q(gpu, 4, 4, 64, BF)
    want = paged_decode_attn(q, *c.args(), 0.1, window=2500, sinks=4, **c.scales())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(paged_decode_attn(q, *c.args(), 0.1, window=2500, sinks=4, **c.scales()))
    torch.cuda.synchronize()
    _clean()
    assert all(torch.equal(x, want) for x in outs)


def test_refusals(gpu):
    c = Cache(gpu, [100, 50], 32, 64, BF, False, seed=16)
    q, qp, cu = _q(gpu, 2, 4, 64, BF), _q(gpu, 40, 8, 64, BF), _cu([40], gpu)
    t = torch.tensor([5, 5], dtype=torch.int32, device=gpu)
    for bad in (dict(sinks=4), dict(window=-1), dict(window=5, sinks=-1), dict(window=True), dict(window=5.0), dict(window=t.long()),
                dict(window=t[:1]), dict(window=t.cpu()), dict(window=t, sinks=t.float()), dict(window=5, sinks=t.repeat(2)[::2][:1]),
                dict(window=t.repeat_interleave(2)[::2]), dict(window="5"), dict(window=t.view(1, 2))):
        for call in (lambda: paged_decode_attn(q, *c.args(), 0.1, **bad), lambda: paged_prompt_attn(qp, *c.args(), cu, 0.1, **bad),
                     lambda: paged_prompt_attn(qp[:1], *c.args(), _cu([1], gpu), 0.1, **bad)):
            with pytest.raises(_lib.WnwError):
                call()
    _clean()


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D,G,new,old", [(BF, 128, 4, [300], [9000]), (FP, 64, 1, [70, 200, 0], [6000, 300, 12000]),
                                               (BF, 256, 2, [90, 33], [5000, 7000]), (FP, 128, 16, [64], [8000])])
def test_prompt_blocks_of_different_lengths(gpu, q8, dtype, D, G, new, old):
    """Few blocks, cut into shares by their own tiles: heads that see everything beside heads with short windows."""
    H = 4
    lens = [o + n for o, n in zip(old, new) for _ in range(H)]
    c = Cache(gpu, lens, 64, D, dtype, q8, seed=D + G)
    N = len(lens)
    window = torch.tensor([(ALL, 500, 64, 0)[s % 4] for s in range(N)], dtype=torch.int32, device=gpu)
    sinks = torch.tensor([(0, 4, 130, 0)[s % 4] for s in range(N)], dtype=torch.int32, device=gpu)
    _hide(c, new, window, sinks)
    q = _q(gpu, sum(new), H * G, D, dtype)
    out = paged_prompt_attn(q, *c.args(), _cu(new, gpu), D ** -0.5, max_tokens=max(new), window=window, sinks=sinks, **c.scales())
    _clean()
    _prompt_check(c, q, out, new, window, sinks, D ** -0.5)
    assert torch.equal(out, paged_prompt_attn(q, *c.args(), _cu(new, gpu), D ** -0.5, max_tokens=max(new), window=window,
                                              sinks=sinks, **c.scales()))
    # a sample with more tokens than the call says: the error word, its rows not written, the others' right
    if len(new) > 1:
        most = sorted(new)[-2]
        room = torch.full_like(q, 7.0)
        paged_prompt_attn(q, *c.args(), _cu(new, gpu), D ** -0.5, max_tokens=most, window=window, sinks=sinks, out=room, **c.scales())
        torch.cuda.synchronize()
        assert _lib.device_error() == _lib.DEVERR_BOUNDS
        at = 0
        for b, n in enumerate(new):
            if n > most:
                assert bool((room[at:at + n] == 7).all())
                room[at:at + n] = out[at:at + n]
            at += n
        _prompt_check(c, q, room, new, window, sinks, D ** -0.5)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 128), (BF, 64), (BF, 256)])
def test_prompt_long_walks(gpu, q8, dtype, D):
    """Blocks that walk more tiles than a workgroup keeps the pages of, in a call that is not cut."""
    new, old, H, G = [2100], [6000], 8, 8
    c = Cache(gpu, [8100] * H, 64, D, dtype, q8, seed=D)
    window, sinks = 5003, 37
    _hide(c, new, window, sinks)
    q = _q(gpu, 2100, H * G, D, dtype)
    out = paged_prompt_attn(q, *c.args(), _cu(new, gpu), D ** -0.5, window=window, sinks=sinks, **c.scales())
    _clean()
    for s in (0, 7):
        keep = torch.tensor([0, 1, 63, 64, 65, 1000, 1001, 2036, 2098, 2099], device=gpu)
        pos = (6000 + keep).repeat_interleave(G)
        place = (keep, slice(s * G, (s + 1) * G))
        _check_rows(c, s, q[place].reshape(-1, D), out[place].reshape(-1, D), pos, window, sinks, D ** -0.5, 1)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_offsets_past_32_bits(gpu, q8, D):
    """Pages 3 GiB apart, tokens 2 GiB apart, through a window; calls of few rows, of many, and cut into shares."""
    G, R, pages = 4, 256, 5
    small = Cache(gpu, [R * (pages - 1) + 20], R, D, BF, q8, seed=21, spare=0, room=1)
    assert small.P == pages
    room = torch.empty(pages * (3 << 30) + (1 << 20), dtype=torch.uint8, device=gpu).view(small.k.dtype)
    far = (3 << 30) // (1 if q8 else 2)
    k, v = (room.as_strided((pages, R, D), (far, D, 1), i * R * D) for i in range(2))
    for to, of in ((k, small.k), (v, small.v)):
        (to.view(torch.uint8) if q8 else to).copy_(of.view(torch.uint8) if q8 else of)
    q = _q(gpu, 1, G, D, BF)
    view = dict(window=700, sinks=5)
    args, scales = (k, v, small.table, small.seg_len), small.scales()
    assert torch.equal(paged_decode_attn(q, *small.args(), 0.1, **view, **scales), paged_decode_attn(q, *args, 0.1, **view, **scales))
    for new in (3, 40, 600):
        rows = _q(gpu, new, G, D, BF)
        want = paged_prompt_attn(rows, *small.args(), _cu([new], gpu), 0.1, **view, **scales)
        assert torch.equal(want, paged_prompt_attn(rows, *args, _cu([new], gpu), 0.1, **view, **scales))
        _prompt_check(small, rows, want, [new], 700, 5, 0.1)
    for new in (3, 6):
        wide = torch.empty((new - 1) * (1 << 30) + G * D, dtype=BF, device=gpu).as_strided((new, G, D), (1 << 30, D, 1))
        rows = _q(gpu, new, G, D, BF)
        wide.copy_(rows)
        want = paged_prompt_attn(rows, *small.args(), _cu([new], gpu), 0.1, **view, **scales)
        assert torch.equal(want, paged_prompt_attn(wide, *args, _cu([new], gpu), 0.1, **view, **scales))
        assert torch.equal(want, paged_prompt_attn(wide, *args, _cu([new], gpu), 0.1, out=wide, **view, **scales))
    _clean()


@pytest.mark.parametrize("dtype,D,q8", [(BF, 128, True), (FP, 128, False), (BF, 256, False), (FP, 64, True)])
def test_out_is_q(gpu, dtype, D, q8):
    """The result in q's own memory: few rows, many, cut into shares and not."""
    window = torch.tensor([ALL, 40, 333, 0], dtype=torch.int32, device=gpu)
    for new, old in ([1, 1], [900, 5]), ([2, 3], [900, 5]), ([70, 33], [3000, 900]), ([600, 1], [0, 10]):
        c = Cache(gpu, [n + o for n, o in zip(new, old) for _ in range(2)], 32, D, dtype, q8, seed=sum(new))
        q = _q(gpu, sum(new), 16, D, dtype)
        for w, z in ((64, 3), (window, 2)):
            want = paged_prompt_attn(q, *c.args(), _cu(new, gpu), 0.1, max_tokens=max(new), window=w, sinks=z, **c.scales())
            room = q.clone()
            got = paged_prompt_attn(room, *c.args(), _cu(new, gpu), 0.1, max_tokens=max(new), window=w, sinks=z, out=room, **c.scales())
            assert got is room and torch.equal(got, want)
            _prompt_check(c, q, want, new, w, z, 0.1)
        qd = _q(gpu, 4, 16, D, dtype)
        want = paged_decode_attn(qd, *c.args(), 0.1, window=window, sinks=2, **c.scales())
        room = qd.clone()
        assert torch.equal(paged_decode_attn(room, *c.args(), 0.1, window=window, sinks=2, out=room, **c.scales()), want)
    _clean()


def test_captured_shares(gpu):
    """Captured calls that are cut into shares, two graphs and eager ones in turn, as lengths and windows change."""
    lens = [4000] * 8
    c = Cache(gpu, lens, 64, 128, BF, True, seed=31)
    q, cu = _q(gpu, 100, 32, 128, BF), _cu([100], gpu)
    window = torch.tensor([ALL, 500] * 4, dtype=torch.int32, device=gpu)
    calls = [lambda: paged_prompt_attn(q, *c.args(), cu, 0.1, window=window, sinks=4, **c.scales()),
             lambda: paged_prompt_attn(q, *c.args(), cu, 0.1, window=3000, sinks=4, **c.scales())]
    graphs = []
    for call in calls:
        call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for step in range(5):
        c.lens = [4000 - 700 * step] * 8
        c.seg_len.copy_(torch.tensor(c.lens, dtype=torch.int32))
        window[step] = 900 * step
        for g, _ in graphs:
            g.replay()
        want = [call() for call in calls]
        for g, _ in graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, x) for (_, out), x in zip(graphs, want))
        _prompt_check(c, q, want[0], [100], window, 4, 0.1)
    _clean()


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D,G", [(BF, 128, 4), (FP, 64, 2), (BF, 256, 4), (FP, 128, 8)])
@pytest.mark.parametrize("new,old", [(1, 900), (2, 900), (60, 900), (700, 300), (40, 9000)])
def test_rows_without_a_page_read_as_zeros(gpu, q8, dtype, D, G, new, old):
    """Blocks that are seen and have no page: the error word, and rows of zeros, beside NaN in page 0 and the last."""
    n, R, window, sinks = new + old, 32, 200 + new, 70
    c = Cache(gpu, [n], R, D, dtype, q8, seed=new + D)
    first = max(old + 1 - window, 0)
    gone = sorted({1, first // R + 1, first // R + 2, n // R - 1})
    used = {int(c.table[0, j]) for j in range(-(-n // R)) if j not in gone}
    k, v = c.rows(0)
    for j in gone:
        k[j * R:(j + 1) * R] = 0
        v[j * R:(j + 1) * R] = 0
        c.table[0, j] = (-1, 0x7fffffff, c.P, -5)[j % 4]
    for page in {0, c.P - 1} - used:
        for pages in (c.k, c.v):
            (pages.view(torch.uint8) if q8 else pages)[page] = 0x7f if q8 else float("nan")
    q = _q(gpu, new, G, D, dtype)
    out = paged_prompt_attn(q, *c.args(), _cu([new], gpu), D ** -0.5, window=window, sinks=sinks, **c.scales())
    torch.cuda.synchronize()
    assert _lib.device_error() == _lib.DEVERR_BOUNDS
    pos = (old + torch.arange(new, device=gpu)).repeat_interleave(G)
    seen = _seen(n, pos, window, sinks)
    p = torch.softmax((q.reshape(-1, D).double() @ k.t().contiguous() * D ** -0.5).masked_fill(~seen, -torch.inf), dim=1)
    ref, A, h = p @ v, p @ v.abs(), HALF[dtype]
    bound = h * ref.abs() + (h + 2.0 ** -13) * A
    if dtype == FP:
        bound = bound + seen.sum(1, keepdim=True) * 2.0 ** -25 * v.abs().max()
    _check(out.reshape(-1, D), ref, bound, (new, old))
