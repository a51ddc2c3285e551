"""The pools' operators against tests/pages_ref.py: whole numbers, equal ones."""
import random

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from tests import pages_ref
from tests.test_gpu_paged import _clean
from tests.test_gpu_paged_edges import _General
from wnw_amd import _lib
from wnw_amd.kv.pages import paged_compact, paged_copy, paged_fork, paged_reserve

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _t(x, gpu, shape=None):
    t = torch.tensor(x, dtype=torch.int32, device=gpu)
    return t if shape is None else t.reshape(shape)


def _wide(table, M, gpu):
    """A table whose rows lie M + 3 entries apart."""
    room = torch.full((max(len(table), 1), M + 3), 12345, dtype=torch.int32, device=gpu)
    view = room[:len(table), :M]
    if len(table) and M:
        view.copy_(_t(table, gpu))
    return view, room


def _state(rng, B, H, R, M, P, junk=False, shared=True):
    """A pool in use: samples of random lengths, some sharing full pages, some entries given back; counts that include pages
    that no table names."""
    pages = list(range(P))
    rng.shuffle(pages)
    table, lens = [], []
    for b in range(B):
        for h in range(H):
            n = rng.choice([0, 1, R - 1, R, R + 1, rng.randrange(M * R + 1), M * R])
            n = min(n, M * R)
            row = []
            for j in range(M):
                named = j * R < n or rng.random() < 0.1
                full = (j + 1) * R <= n
                if not named or not pages or (full and rng.random() < 0.1):
                    row.append(-1)
                elif full and shared and table and rng.random() < 0.3 and any(e >= 0 for e in table[-1]):
                    k = rng.randrange(M)
                    e = table[-1][k]
                    row.append(e if e >= 0 and (k + 1) * R <= lens[-1] else -1)
                else:
                    row.append(pages.pop())
            if junk:
                row = [rng.choice([P, -2, 0x7fffffff, -2147483648]) if e < 0 and rng.random() < 0.3 else e for e in row]
            table.append(row)
            lens.append(n)
    pinned = [pages.pop() for _ in range(min(3, len(pages)))]
    return table, lens, pages_ref.counts(table, P, pinned)


SIZES = [(1, 1, 16, 1, 3), (1, 1, 64, 4, 10), (3, 2, 16, 9, 70), (8, 4, 32, 20, 700), (5, 8, 128, 300, 20000), (64, 8, 16, 7, 40000),
         (2, 1, 256, 700, 17001), (300, 1, 16, 3, 2000), (0, 2, 16, 4, 9), (3, 1, 16, 0, 5)]


@pytest.mark.parametrize("B,H,R,M,P", SIZES)
@pytest.mark.parametrize("junk", [False, True])
def test_fork(gpu, B, H, R, M, P, junk):
    rng = random.Random(B * 1000 + M)
    for n_new in (B, 1, 2 * B + 3, 0):
        table, lens, refs = _state(rng, B, H, R, M, P, junk)
        parents = [rng.randrange(-1, B) if rng.random() < 0.9 else -1 for _ in range(n_new)]
        if n_new == 1 and B:
            parents = [B - 1]
        want = pages_ref.fork(table, lens, refs, parents, R, H, M)
        view, room = _wide(table, M, gpu)
        new, new_len, new_refs, copies = paged_fork(view, _t(lens, gpu), _t(refs, gpu), _t(parents, gpu), R, kv_heads=H)
        torch.cuda.synchronize()
        err = _lib.device_error()
        if want is None:
            assert err & _lib.DEVERR_CAPACITY
            assert bool((new == -1).all()) and bool((new_len == 0).all()) and new_refs.tolist() == refs
            assert copies.tolist() == [[-1, -1, 0]] * (n_new * H)
        else:
            assert err in ((0, _lib.DEVERR_BOUNDS) if junk else (0,))
            assert new.tolist() == want[0] and new_len.tolist() == want[1]
            assert new_refs.tolist() == want[2] and copies.tolist() == want[3]
        assert room[:, M:].unique().tolist() in ([12345], []) and view.tolist() == table


@pytest.mark.parametrize("B,H,R,M,P", SIZES)
@pytest.mark.parametrize("junk", [False, True])
def test_reserve(gpu, B, H, R, M, P, junk):
    rng = random.Random(B * 999 + M)
    N = B * H
    for how in ("one", "none", "chunks", "window", "windows"):
        table, lens, refs = _state(rng, B, H, R, M, P, junk)
        cu = view = None
        tokens = [{"one": 1, "none": 0, "window": min(2, R * M)}.get(how, 0)] * N
        kw = dict(tokens=tokens[0] if N else 0)
        if how in ("chunks", "windows"):
            new = [rng.choice([0, 1, rng.randrange(M * R + 1)]) for _ in range(B)]
            cu = [sum(new[:b]) for b in range(B + 1)]
            tokens = [new[s // H] for s in range(N)]
            lens = [max(0, min(n, M * R - t)) for n, t in zip(lens, tokens)]
            kw = dict(cu_tokens=_t(cu, gpu))
        else:
            lens = [max(0, min(n, M * R - t)) for n, t in zip(lens, tokens)]
        if how == "window":
            view = [(R + 3, 5)] * N
            kw |= dict(window=R + 3, sinks=5)
        elif how == "windows":
            view = [(rng.choice([0, 1, R, 3 * R + 1, 0x7fffffff]), rng.choice([0, 1, R, R + 1, 0x7fffffff])) for _ in range(N)]
            kw |= dict(window=_t([w for w, _ in view], gpu), sinks=_t([z for _, z in view], gpu))
        want = pages_ref.reserve(table, lens, refs, R, tokens, view)
        was, room = _wide(table, M, gpu)
        counts = _t(refs, gpu)
        new, new_refs = paged_reserve(was, _t(lens, gpu), counts, R, **kw)
        torch.cuda.synchronize()
        err = _lib.device_error()
        if want is None:
            assert err & _lib.DEVERR_CAPACITY, how
            want = table, refs
        else:
            assert err in ((0, _lib.DEVERR_BOUNDS) if junk else (0,)), how
        assert new.tolist() == want[0] and new_refs.tolist() == want[1], how
        assert was.tolist() == table and counts.tolist() == refs
        paged_reserve(was, _t(lens, gpu), counts, R, out=(was, counts), **kw)  # in place
        torch.cuda.synchronize()
        _lib.device_error()
        assert was.tolist() == want[0] and counts.tolist() == want[1], how
        assert room[:, M:].unique().tolist() in ([12345], [])


@pytest.mark.parametrize("B,H,R,M,P", SIZES + [(20, 4, 16, 40, 50001)])
@pytest.mark.parametrize("junk", [False, True])
def test_compact(gpu, B, H, R, M, P, junk):
    rng = random.Random(B * 77 + M)
    for _ in range(2):
        table, lens, refs = _state(rng, B, H, R, M, P, junk)
        want = pages_ref.compact(table, refs, R)
        was, room = _wide(table, M, gpu)
        counts = _t(refs, gpu)
        new, new_refs, moves, used = paged_compact(was, counts, R)
        torch.cuda.synchronize()
        assert _lib.device_error() in ((0, _lib.DEVERR_BOUNDS) if junk else (0,))
        assert new.tolist() == want[0] and new_refs.tolist() == want[1]
        assert moves.tolist() == want[2] and used.tolist() == [want[3]]
        got = paged_compact(was, counts, R, out=(was, counts))
        torch.cuda.synchronize()
        _lib.device_error()
        assert was.tolist() == want[0] and counts.tolist() == want[1] and got[2].tolist() == want[2]
        again = paged_compact(was, counts, R)  # nothing is left to move
        assert torch.equal(again[0], was) and torch.equal(again[1], counts) and bool((again[2][:, 0] == -1).all())
        assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype,D,R", [(E4M3, 128, 64), (E4M3, 64, 16), (torch.bfloat16, 256, 256), (torch.float16, 64, 32),
                                       (E4M3, 256, 128)])
def test_copy(gpu, dtype, D, R):
    rng = random.Random(R)
    P = 300
    both = torch.randint(0, 256, (P, 2, R, D * (1 if dtype == E4M3 else 2)), dtype=torch.uint8, device=gpu)
    both = both if dtype == E4M3 else both
    k, v = (both[:, i].view(dtype) for i in range(2))  # pages of K and V beside each other
    scales = [torch.rand(P, device=gpu) for _ in range(2)] if dtype == E4M3 else [None, None]
    for n in (1, 7, 100, 0):
        ids = rng.sample(range(P), 2 * n)
        copies = [[ids[2 * i], ids[2 * i + 1], rng.choice([0, 1, R // 2, R - 1, R])] for i in range(n)]
        copies += [[-1, -1, 0], [-5, 3, R]]
        rng.shuffle(copies)
        want, ws = both.clone(), [None if s is None else s.clone() for s in scales]
        for a, b, rows in copies:
            if a >= 0:
                want[b, :, :rows] = want[a, :, :rows]
                for s in ws:
                    if s is not None:
                        s[b] = s[a]
        paged_copy(k, v, _t(copies, gpu), k_scale=scales[0], v_scale=scales[1])
        _clean()
        assert torch.equal(both, want)
        assert all(s is None or torch.equal(s, t) for s, t in zip(scales, ws))
    # entries outside the pool or the page: the error word, and nothing else
    was = both.clone()
    for bad in ([P, 0, R], [0, P, R], [0, -1, R], [4, 4, R], [0, 1, R + 1], [0, 1, -1], [0x7fffffff, 1, 1]):
        paged_copy(k, v, _t([bad], gpu), k_scale=scales[0], v_scale=scales[1])
        torch.cuda.synchronize()
        assert _lib.device_error() == _lib.DEVERR_BOUNDS, bad
    assert torch.equal(both, was)


def test_bad_numbers_change_nothing(gpu):
    """Lengths, parents, token counts and windows that cannot be: the error word, outputs as documented."""
    table, refs, R = [[0, 1, -1, -1], [2, -1, -1, -1]], [1, 1, 1, 0, 0, 0], 16
    bounds, room = _lib.DEVERR_BOUNDS, _lib.DEVERR_CAPACITY

    def fork(lens=(20, 5), parents=(1, 0)):
        return paged_fork(_t(table, gpu), _t(lens, gpu), _t(refs, gpu), _t(parents, gpu), R, kv_heads=1)

    for kw in (dict(lens=(-1, 5)), dict(lens=(20, 65)), dict(parents=(2, 0)), dict(parents=(-2,)), dict(parents=(0, 0x7fffffff))):
        new, new_len, new_refs, copies = fork(**kw)
        torch.cuda.synchronize()
        assert _lib.device_error() == bounds, kw
        assert bool((new == -1).all()) and bool((new_len == 0).all()) and new_refs.tolist() == refs and bool((copies[:, 0] == -1).all())

    def reserve(lens=(20, 5), **kw):
        return paged_reserve(_t(table, gpu), _t(lens, gpu), _t(refs, gpu), R, **kw)

    for want, kw in ((bounds, dict(lens=(-1, 5))), (bounds, dict(lens=(20, 65), tokens=0)), (room, dict(tokens=60)),
                     (room, dict(tokens=44)), (bounds, dict(cu_tokens=_t([0, 5, 3], gpu))), (bounds, dict(cu_tokens=_t([-1, 5, 9], gpu))),
                     (bounds, dict(window=_t([5, -1], gpu))), (bounds, dict(window=5, sinks=_t([-3, 0], gpu))),
                     (room, dict(tokens=1 << 30)), (room, dict(cu_tokens=_t([0, 5, 0x7fffffff], gpu)))):
        new, new_refs = reserve(**kw)
        torch.cuda.synchronize()
        assert _lib.device_error() == want, kw
        assert new.tolist() == table and new_refs.tolist() == refs


def test_captured_in_place(gpu):
    """A captured reserve that keeps its table and counts in place, replayed as segments grow, beside eager calls."""
    rng = random.Random(5)
    B, H, R, M, P = 3, 2, 16, 30, 400
    table, refs = [[-1] * M for _ in range(B * H)], [0] * P
    lens = [0] * (B * H)
    view = [(40, 5)] * (B * H)
    dt, dl, dr = _t(table, gpu), _t(lens, gpu), _t(refs, gpu)
    keep = dt.clone(), dr.clone()
    paged_reserve(dt, dl, dr, R, tokens=7, window=40, sinks=5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_reserve(dt, dl, dr, R, tokens=7, window=40, sinks=5, out=(dt, dr))
    assert torch.equal(dt, keep[0]) and torch.equal(dr, keep[1])  # captured, not run
    for step in range(40):
        graph.replay()
        table, refs = pages_ref.reserve(table, lens, refs, R, [7] * (B * H), view)
        if step % 7 == 3:
            paged_reserve(dt.clone(), dl, dr.clone(), R, tokens=16)
        torch.cuda.synchronize()
        assert dt.tolist() == table and dr.tolist() == refs and refs == pages_ref.counts(table, P)
        lens = [n + rng.choice([7, 3]) for n in lens]
        dl.copy_(_t(lens, gpu))
    _clean()


def test_refusals(gpu):
    table, lens, refs = _t([[0, 1], [2, -1]], gpu), _t([20, 5], gpu), _t([1, 1, 1, 0], gpu)
    parents = _t([0, 1], gpu)
    E = _lib.WnwError
    for bad in (dict(t=table.long()), dict(t=table[0]), dict(t=table.t()), dict(l=lens.long()), dict(l=lens[:1]), dict(r=refs.float()),
                dict(r=refs.view(2, 2)), dict(p=parents.long()), dict(p=parents.view(1, 2)), dict(R=24), dict(R=512), dict(h=0), dict(h=3),
                dict(t=table.cpu()), dict(p=parents.cpu())):
        c = dict(t=table, l=lens, r=refs, p=parents, R=16, h=1)
        c.update(bad)
        with pytest.raises(E):
            paged_fork(c["t"], c["l"], c["r"], c["p"], c["R"], kv_heads=c["h"])
    for kw in (dict(tokens=-1), dict(sinks=3), dict(window=-1), dict(window=3, sinks=-1), dict(cu_tokens=_t([0, 1, 2, 3], gpu)),
               dict(cu_tokens=lens.long()), dict(out=(table[:1], refs)), dict(out=(table, refs[:2])), dict(out=(table.long(), refs)),
               dict(out=(table, refs.clone()[:3])), dict(window=lens.cpu())):
        with pytest.raises(E):
            paged_reserve(table, lens, refs, 16, **kw)
    room = torch.zeros(40, dtype=torch.int32, device=gpu)
    with pytest.raises(E, match="overlaps"):  # one row further on in the same memory
        paged_reserve(room[:20].view(5, 4), torch.zeros(5, dtype=torch.int32, device=gpu), refs, 16,
                      out=(room[4:24].view(5, 4), refs.clone()))
    with pytest.raises(E, match="overlaps"):
        paged_compact(room[:20].view(5, 4), room[20:30], 16, out=(room[:20].view(5, 4), room[21:31]))
    with pytest.raises(E, match="overlaps"):
        paged_reserve(room[:20].view(5, 4), torch.zeros(5, dtype=torch.int32, device=gpu), room[20:30], 16,
                      out=(room[20:40].view(5, 4), refs.new_zeros(10)))
    k = torch.zeros(4, 16, 64, dtype=torch.bfloat16, device=gpu)
    for bad in (dict(c=_t([[0, 1]], gpu)), dict(c=_t([[0, 1, 2]], gpu).long()), dict(v=k[:2]), dict(v=k.half()), dict(s=torch.ones(4, device=gpu)),
                dict(k=k.float(), v=k.float()), dict(k=k.transpose(1, 2), v=k.transpose(1, 2)), dict(c=torch.zeros(1, 3, dtype=torch.int32))):
        c = dict(k=k, v=k.clone(), c=_t([[0, 1, 2]], gpu), s=None)
        c.update(bad)
        with pytest.raises(E):
            paged_copy(c["k"], c["v"], c["c"], k_scale=c["s"])
    _clean()


def test_both_ways_into_a_call(gpu, monkeypatch):
    """The native way of the plain calls and the general way give the same results."""
    rng = random.Random(3)
    B, H, R, M, P = 4, 2, 32, 11, 300
    table, lens, refs = _state(rng, B, H, R, M, P)
    lens = [min(n, M * R - 40) for n in lens]
    k = torch.randn(P, R, 64, device=gpu).to(torch.bfloat16)
    results = []
    for general in (False, True):
        if general:
            monkeypatch.setattr(_lib, "_callpath", _General())
        t, n, r = _t(table, gpu), _t(lens, gpu), _t(refs, gpu)
        kk, vv = k.clone(), -k
        forked = paged_fork(t, n, r, _t([1, 1, 0, -1, 3], gpu), R, kv_heads=H)
        paged_copy(kk, vv, forked[3])
        room = torch.full((B * H, M + 5), 9, dtype=torch.int32, device=gpu)[:, :M], torch.empty_like(r)
        got = [*forked, kk, vv, *paged_reserve(t, n, r, R), *paged_reserve(t, n, r, R, cu_tokens=_t([0, 5, 40, 40, 41], gpu), out=room),
               *paged_reserve(t, n, r, R, tokens=0, window=n + 3, sinks=4), *paged_compact(t, r, R), *paged_compact(t, r, R, out=(t, r))]
        torch.cuda.synchronize()
        results.append((_lib.device_error(), [x.clone() for x in got]))
    assert results[0][0] == results[1][0] == 0
    assert all(torch.equal(a, b) for a, b in zip(results[0][1], results[1][1]))
    want = pages_ref.fork(table, lens, refs, [1, 1, 0, -1, 3], R, H, M)
    assert results[0][1][0].tolist() == want[0]


def test_watched_calls_are_refused(gpu):
    """Pages that require a gradient, and traces."""
    k = torch.zeros(4, 16, 64, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    copies = _t([[0, 1, 2]], gpu)
    with pytest.raises(_lib.WnwError, match="gradient"):
        paged_copy(k, k.detach().clone(), copies)
    with torch.no_grad():
        paged_copy(k, k.detach().clone(), copies)
    table, refs = _t([[0]], gpu), _t([1], gpu)
    with pytest.raises(_lib.WnwError, match="trace"):
        make_fx(lambda r: paged_compact(table, r, 16)[0])(refs)
    _clean()


def test_in_place_of_one_output(gpu):
    """The table written where it is and the counts elsewhere, and the other way round."""
    rng = random.Random(21)
    B, H, R, M, P = 6, 2, 16, 12, 5000
    table, lens, refs = _state(rng, B, H, R, M, P)
    lens = [min(n, M * R - 20) for n in lens]
    reserved, compacted = pages_ref.reserve(table, lens, refs, R, [20] * (B * H)), pages_ref.compact(table, refs, R)
    for mine in (0, 1):
        for call, want in ((lambda t, r, out: paged_reserve(t, _t(lens, gpu), r, R, tokens=20, out=out), reserved),
                           (lambda t, r, out: paged_compact(t, r, R, out=out), compacted)):
            given = _t(table, gpu), _t(refs, gpu)
            out = tuple(x if i == mine else torch.full_like(x, 77) for i, x in enumerate(given))
            got = call(*given, out)
            _clean()
            assert got[0] is out[0] and got[1] is out[1]
            assert out[0].tolist() == want[0] and out[1].tolist() == want[1]
            kept = given[1 - mine].tolist()  # the input that is not written
            assert kept == (refs if mine == 0 else table)


def test_on_another_stream(gpu):
    """Calls on a stream of the caller's, behind work of its own that writes their inputs."""
    rng = random.Random(22)
    B, H, R, M, P = 5, 2, 32, 40, 3000
    table, lens, refs = _state(rng, B, H, R, M, P)
    parents = [4, 4, 0, 1, 1, -1, 2]
    want = pages_ref.fork(table, lens, refs, parents, R, H, M)
    after = pages_ref.compact(want[0], want[2], R)
    ready = [_t(x, gpu) for x in (table, lens, refs, parents)]
    stream = torch.cuda.Stream()
    for _ in range(3):
        late = [torch.zeros_like(x) for x in ready]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(2_000_000)
            for x, y in zip(late, ready):
                x.copy_(y)
            new, new_len, new_refs, copies = paged_fork(*late, R, kv_heads=H)
            packed = paged_compact(new, new_refs, R)
        stream.synchronize()
        assert new.tolist() == want[0] and new_len.tolist() == want[1] and new_refs.tolist() == want[2] and copies.tolist() == want[3]
        assert packed[0].tolist() == after[0] and packed[2].tolist() == after[2]
    _clean()


def test_captured_fork_and_compact(gpu):
    """A captured step that forks, copies and compacts, replayed with other parents; eager calls in between."""
    rng = random.Random(23)
    B, H, R, M, P = 4, 2, 16, 9, 400
    table, lens, refs = _state(rng, B, H, R, M, P)
    dt, dl, dr = _t(table, gpu), _t(lens, gpu), _t(refs, gpu)
    parents = _t([0] * B, gpu)
    k = torch.randn(P, R, 64, device=gpu).to(torch.bfloat16)
    v = k.clone()

    def step():
        forked = paged_fork(dt, dl, dr, parents, R, kv_heads=H)
        return (*forked, *paged_compact(forked[0], forked[2], R))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
        paged_copy(k, v, got[3])
    for _ in range(6):
        now = [rng.randrange(-1, B) for _ in range(B)]
        parents.copy_(_t(now, gpu))
        before = k.clone()
        graph.replay()
        eager = step()
        want = pages_ref.fork(table, lens, refs, now, R, H, M)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        assert got[0].tolist() == want[0] and got[2].tolist() == want[2] and got[3].tolist() == want[3]
        for a, b, n in want[3]:
            if a >= 0:
                before[b, :n] = before[a, :n]
        assert torch.equal(k, before) and torch.equal(v, before)
    _clean()


def test_most_samples(gpu):
    """8,192 samples before and after, all going on from few parents or each from its own; 8,193 are refused."""
    R, M, P = 16, 2, 30000
    rng = random.Random(24)
    table, lens, refs = _state(rng, 8192, 1, R, M, P, shared=False)
    for parents in ([rng.randrange(8192) for _ in range(8192)], [8191] * 8192, list(range(8191, -1, -1))):
        want = pages_ref.fork(table, lens, refs, parents, R, 1, M)
        new, new_len, new_refs, copies = paged_fork(_t(table, gpu), _t(lens, gpu), _t(refs, gpu), _t(parents, gpu), R, kv_heads=1)
        _clean()
        assert new.tolist() == want[0] and new_len.tolist() == want[1] and new_refs.tolist() == want[2] and copies.tolist() == want[3]
    with pytest.raises(_lib.WnwError, match="8192 samples"):
        paged_fork(_t(table, gpu), _t(lens, gpu), _t(refs, gpu), _t([0] * 8193, gpu), R, kv_heads=1)
    _clean()


def test_copy_far_apart(gpu):
    """Pages whose bytes lie past 32 bits of offset."""
    P, R, D = 70001, 256, 128
    k = torch.empty(P, R, D, dtype=torch.bfloat16, device=gpu)
    v = torch.empty(P, R, D, dtype=torch.bfloat16, device=gpu)
    assert k.numel() * 2 > 2 ** 32
    g = torch.Generator(device=gpu).manual_seed(1)
    for at in (0, 3, 69999, 70000):
        k[at] = torch.randn(R, D, device=gpu, generator=g).to(k.dtype)
        v[at] = torch.randn(R, D, device=gpu, generator=g).to(k.dtype)
    far, near = (k[70000].clone(), v[70000].clone()), (k[0].clone(), v[0].clone())
    paged_copy(k, v, _t([[70000, 3, R], [0, 69999, R]], gpu))
    _clean()
    assert torch.equal(k[3], far[0]) and torch.equal(v[3], far[1]) and torch.equal(k[69999], near[0]) and torch.equal(v[69999], near[1])


def test_numbers_that_are_none(gpu):
    """Sizes that are not whole numbers are refused; numpy's are taken."""
    import numpy as np
    table, lens, refs, parents = _t([[0, 1], [2, -1]], gpu), _t([20, 5], gpu), _t([1, 1, 1, 0], gpu), _t([0, 1], gpu)
    for call in (lambda: paged_fork(table, lens, refs, parents, 16, kv_heads=1.0), lambda: paged_fork(table, lens, refs, parents, 16.0, kv_heads=1),
                 lambda: paged_reserve(table, lens, refs, 16, tokens=1.0), lambda: paged_reserve(table, lens, refs, "16"),
                 lambda: paged_compact(table, refs, None)):
        with pytest.raises((_lib.WnwError, TypeError)):
            call()
    a, b = paged_fork(table, lens, refs, parents, np.int64(16), kv_heads=np.int32(1)), paged_fork(table, lens, refs, parents, 16, kv_heads=1)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    _clean()
