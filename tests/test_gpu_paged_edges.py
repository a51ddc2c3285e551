"""The paged cache's operators at their edges: infinities and NaN that a causal
mask hides, few query rows over long segments, offsets past 32 bits, shared
pages, the native and the general way into a call.  Tolerances as in
test_gpu_paged.py, from the same bounds."""
import pytest
import torch

from tests.paged_ref import E4M3, HALF, Cache, attend
from tests.test_gpu_paged import BF, FP, _check, _clean, _cu, _decode_check, _prompt_check, _q, _snapshot
from wnw_amd import _lib
from wnw_amd.kv.paged import PagedWorkspace, paged_append, paged_decode_attn, paged_prompt_attn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q8,odd", [(True, "nan"), (False, "inf"), (False, "-inf"), (False, "nan")])
@pytest.mark.parametrize("dtype,D,G", [(BF, 128, 4), (FP, 64, 1), (BF, 256, 2), (FP, 128, 16)])
@pytest.mark.parametrize("new,old", [(3, 50), (15, 17), (40, 70), (300, 0), (70, 6000)], ids=lambda x: str(x))
def test_v_not_finite_in_masked_rows(gpu, q8, odd, dtype, D, G, new, old):
    """An infinity or NaN of V in a later token's row reaches the tokens from that one on, in its own elements, and no other."""
    c = Cache(gpu, [old + new, 33], 64, D, dtype, q8, seed=D + G + new)
    q = _q(gpu, new + 1, G, D, dtype)
    rows = sorted({old + new - 1, old + new // 2, old + min(1, new - 1)}, reverse=True)
    clean = [x.clone() for x in c.rows(0)]
    for i, r in enumerate(rows):
        p, at = c.table[0, r // 64].item(), r % 64
        for d in (7 + i, D - 2 - 3 * i):
            if q8:
                c.v.view(torch.uint8)[p, at, d] = 0x7f if i % 2 else 0xff
            else:
                c.v[p, at, d] = float(odd)
            clean[1][r, d] = 0.0
    out = paged_prompt_attn(q, *c.args(), _cu([new, 1], gpu), D ** -0.5, max_tokens=new, **c.scales())
    _clean()
    assert bool(torch.isfinite(out[new]).all())
    lim = old + torch.arange(new, device=gpu).repeat_interleave(G) + 1
    ref, A = attend(q[:new].reshape(new * G, D).double(), *clean, lim, D ** -0.5)
    got = out[:new].reshape(new * G, D).clone()
    for i, r in enumerate(rows):
        for d in (7 + i, D - 2 - 3 * i):
            sees = lim > r
            assert bool(torch.equal(got[sees, d], torch.full_like(got[sees, d], float(odd)))) if odd != "nan" \
                else bool(got[sees, d].isnan().all())
            got[sees, d] = ref[sees, d].to(dtype)
    h = HALF[dtype]
    bound = h * ref.abs() + (h + 2.0 ** -13) * A + (c.lens[0] * 2.0 ** -25 * clean[1].abs().max() if dtype == FP else 0)
    _check(got, ref, bound)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D,G,H,new,old", [
    (BF, 128, 4, 2, [5], [8000]), (BF, 128, 1, 1, [17], [20000]), (FP, 64, 8, 2, [64, 3, 0, 9], [3000, 5000, 70, 1]),
    (BF, 256, 4, 1, [33], [5000]), (FP, 128, 32, 1, [1, 1], [4000, 2500]), (BF, 128, 24, 1, [1], [9000])])
def test_prompt_few_rows_long_segments(gpu, q8, dtype, D, G, H, new, old):
    """The splits of a segment's tiles and the launch that joins them, waves without rows beside waves with some."""
    lens = [o + n for o, n in zip(old, new) for _ in range(H)]
    c = Cache(gpu, lens, 64, D, dtype, q8, seed=D + G)
    q = _q(gpu, sum(new), H * G, D, dtype)
    out = paged_prompt_attn(q, *c.args(), _cu(new, gpu), D ** -0.5, max_tokens=max(new), **c.scales())
    _clean()
    _prompt_check(c, q, out, new, H, D ** -0.5)
    assert torch.equal(out, paged_prompt_attn(q, *c.args(), _cu(new, gpu), D ** -0.5, max_tokens=max(new), **c.scales()))


@pytest.mark.parametrize("q8", [True, False])
def test_offsets_past_32_bits(gpu, q8):
    """Pages 3 GiB apart, tokens 2 GiB apart: every offset is a 64-bit one."""
    G, D, R, pages, new = 4, 128, 64, 4, 3
    small = Cache(gpu, [R * (pages - 1) + 20], R, D, BF, q8, seed=21, spare=0, room=1)
    assert small.P == pages
    el = 1 if q8 else 2
    room = torch.empty(pages * (3 << 30) + (1 << 20), dtype=torch.uint8, device=gpu).view(E4M3 if q8 else BF)
    far = (3 << 30) // el
    k = room.as_strided((pages, R, D), (far, D, 1))
    v = room.as_strided((pages, R, D), (far, D, 1), R * D)
    (k.view(torch.uint8) if q8 else k).copy_(small.k.view(torch.uint8) if q8 else small.k)
    (v.view(torch.uint8) if q8 else v).copy_(small.v.view(torch.uint8) if q8 else small.v)
    table, lens = small.table, small.seg_len
    q = _q(gpu, 1, G, D, BF)
    want = paged_decode_attn(q, *small.args(), 0.1, **small.scales())
    assert torch.equal(want, paged_decode_attn(q, k, v, table, lens, 0.1, **small.scales()))
    wide = torch.empty((new - 1) * (1 << 30) + G * D, dtype=BF, device=gpu)
    rows = _q(gpu, 40, G, D, BF)
    want = paged_prompt_attn(rows, *small.args(), _cu([40], gpu), 0.1, **small.scales())
    assert torch.equal(want, paged_prompt_attn(rows, k, v, table, lens, _cu([40], gpu), 0.1, **small.scales()))
    few = wide.as_strided((new, G, D), (1 << 30, D, 1))
    few.copy_(rows[:new])
    want = paged_prompt_attn(rows[:new], *small.args(), _cu([new], gpu), 0.1, **small.scales())
    assert torch.equal(want, paged_prompt_attn(few, k, v, table, lens, _cu([new], gpu), 0.1, **small.scales()))
    # an append into the far pages, from far tokens
    kv = few[:, :1]
    scales = {n: (None if x is None else x.clone()) for n, x in small.scales().items()}
    _, a = paged_append(kv, kv, k, v, table, lens, cu_tokens=_cu([new], gpu), **scales)
    _, b = paged_append(kv.contiguous(), kv.contiguous(), *small.args(), cu_tokens=_cu([new], gpu), **small.scales())
    _clean()
    assert torch.equal(a, b) and torch.equal(k.contiguous().view(torch.uint8), small.k.view(torch.uint8))
    assert torch.equal(v.contiguous().view(torch.uint8), small.v.view(torch.uint8))
    assert not q8 or (torch.equal(scales["k_scale"], small.k_scale) and torch.equal(scales["v_scale"], small.v_scale))


def test_shared_pages_are_read(gpu):
    """Segments that share pages, and a page twice in one segment."""
    c = Cache(gpu, [200, 200, 200], 64, 128, BF, True, seed=22)
    c.table[1, :2] = c.table[0, :2]
    c.table[2, 1] = c.table[2, 0]
    q = _q(gpu, 3, 4, 128, BF)
    out = paged_decode_attn(q, *c.args(), 0.1, **c.scales())
    _clean()
    _decode_check(c, q, out, 0.1)
    q = _q(gpu, 60, 12, 128, BF)
    out = paged_prompt_attn(q, *c.args(), _cu([60], gpu), 0.1, **c.scales())
    _clean()
    _prompt_check(c, q, out, [60], 3, 0.1)


def test_result_in_place_of_the_query(gpu):
    """The result may go where q was: a row's query is read before its result is written."""
    c = Cache(gpu, [900, 4000], 64, 128, BF, True, seed=23)
    q = _q(gpu, 2, 4, 128, BF)
    want = paged_decode_attn(q, *c.args(), 0.1, **c.scales())
    assert torch.equal(paged_decode_attn(q, *c.args(), 0.1, out=q, **c.scales()), want)
    for n in (3, 100, 700):
        q = _q(gpu, n, 8, 128, BF)
        want = paged_prompt_attn(q, *c.args(), _cu([n], gpu), 0.1, **c.scales())
        assert torch.equal(paged_prompt_attn(q, *c.args(), _cu([n], gpu), 0.1, out=q, **c.scales()), want)
    _clean()


class _General:
    """A call path that takes nothing: every call goes the general way."""

    def __getattr__(self, name):
        return lambda *a: None


@pytest.mark.parametrize("q8", [True, False])
def test_both_ways_into_a_call(gpu, q8, monkeypatch):
    """The native way of the plain calls and the general way give the same results."""
    new, H, G, D = [3, 40, 0], 2, 4, 128
    results = []
    for general in (False, True):
        with monkeypatch.context() as m:
            if general:
                m.setattr(_lib, "_callpath", _General())
            c = Cache(gpu, [70, 70, 5, 5, 64, 64], 64, D, BF, q8, seed=24, room=3)
            gen = torch.Generator(device=gpu).manual_seed(1)
            proj = torch.randn(sum(new), (G + 2) * H * D, device=gpu, generator=gen).to(BF).unflatten(1, (-1, D))
            q, k, v = proj.split([G * H, H, H], 1)
            pos = torch.arange(sum(new), device=gpu).expand(3, -1).contiguous() * 7
            freq = 1e4 ** (-torch.arange(D // 2, device=gpu, dtype=torch.float64) / (D // 2))
            qo, nl = paged_append(k, v, *c.args(), q=q, positions=pos, inv_freq=freq, sections=[24, 20, 20],
                                  cu_tokens=_cu(new, gpu), max_tokens=40, **c.scales())
            a = paged_prompt_attn(qo, c.k, c.v, c.table, nl, _cu(new, gpu), 0.1, max_tokens=40, **c.scales())
            few = paged_prompt_attn(qo[:3], c.k, c.v, c.table, nl, _cu([3, 0, 0], gpu), 0.1, max_tokens=4, **c.scales())
            d = paged_decode_attn(_q(gpu, 6, G, D, BF), c.k, c.v, c.table, nl, 0.1, **c.scales())
            _clean()
            results.append((qo, nl, a, few, d) + _snapshot(c))
    for x, y in zip(*results):
        assert (x is None and y is None) or torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


def test_overlapping_outputs_are_refused(gpu):
    c = Cache(gpu, [40, 50], 32, 64, BF, True, seed=25)
    q = _q(gpu, 20, 4, 64, BF)
    cu, ok = _cu([20, 0], gpu), c.scales()
    row = torch.zeros(1, 4, 64, device=gpu, dtype=BF)
    close = torch.zeros(1024, device=gpu, dtype=BF).as_strided((20, 4, 64), (8, 64, 1))
    both = torch.zeros(3, device=gpu, dtype=torch.int32)
    both[:2] = c.seg_len
    kv = torch.zeros(2, 1, 64, device=gpu, dtype=BF)
    for fn in (lambda: paged_prompt_attn(q, *c.args(), cu, 0.1, out=row.expand(20, 4, 64), **ok),
               lambda: paged_prompt_attn(q, *c.args(), cu, 0.1, out=row[:, :1].expand(20, 4, 64), **ok),
               lambda: paged_prompt_attn(q, *c.args(), cu, 0.1, out=close, **ok),
               lambda: paged_append(kv, kv, c.k, c.v, c.table, both[:2], new_len=both[1:], **ok),
               lambda: paged_append(kv, kv, c.k, c.k, c.table, c.seg_len, **ok)):
        with pytest.raises(_lib.WnwError):
            fn()
    # heads before tokens, and rows apart, are fine
    out = torch.zeros(4, 20, 128, device=gpu, dtype=BF).transpose(0, 1)[..., :64]
    got = paged_prompt_attn(q, *c.args(), cu, 0.1, out=out, **ok)
    assert torch.equal(got, paged_prompt_attn(q, *c.args(), cu, 0.1, **ok))
    _clean()


@pytest.mark.parametrize("dtype,D,G", [(BF, 128, 4), (FP, 64, 1), (BF, 256, 2), (FP, 128, 16)])
@pytest.mark.parametrize("new,old", [(3, 50), (15, 17), (40, 70)], ids=lambda x: str(x))
def test_huge_values_in_masked_rows(gpu, dtype, D, G, new, old):
    """K and V of a later token at the type's largest number: the earlier tokens' results do not move."""
    c = Cache(gpu, [old + new], 64, D, dtype, False, seed=D + new)
    q = _q(gpu, new, G, D, dtype)
    want = paged_prompt_attn(q, *c.args(), _cu([new], gpu), D ** -0.5)
    p, at = c.table[0, (old + new - 1) // 64].item(), (old + new - 1) % 64
    c.k[p, at] = c.v[p, at] = torch.finfo(dtype).max
    got = paged_prompt_attn(q, *c.args(), _cu([new], gpu), D ** -0.5)
    _clean()
    assert torch.equal(got[:-1], want[:-1])  # a weight of 0 times any finite number is 0


def test_table_without_blocks(gpu):
    """A page table of no columns: no rows to see, no room to append to."""
    c = Cache(gpu, [5, 9], 32, 64, BF, True, seed=26)
    table, lens = c.table[:, :0], torch.zeros(2, dtype=torch.int32, device=gpu)
    q, ok = _q(gpu, 2, 4, 64, BF), c.scales()
    assert int(torch.count_nonzero(paged_decode_attn(q, c.k, c.v, table, lens, 0.1, **ok))) == 0
    long = _q(gpu, 90, 8, 64, BF)
    assert int(torch.count_nonzero(paged_prompt_attn(long, c.k, c.v, table, lens, _cu([90], gpu), 0.1, **ok))) == 0
    _clean()
    kv, was = torch.ones(2, 1, 64, device=gpu, dtype=BF), _snapshot(c)
    _, nl = paged_append(kv, kv, c.k, c.v, table, lens, **ok)
    torch.cuda.synchronize()
    assert _lib.device_error() == _lib.DEVERR_CAPACITY and nl.tolist() == [1, 1]
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(_snapshot(c), was))


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("new,room", [(3, 1), (60, 1), (60, 60), (700, 1)], ids=lambda x: str(x))
def test_prompts_captured(gpu, q8, new, room):
    """An append and its prompt attention captured, each form of the attention; replays follow the lengths between eager
    calls, and equal them."""
    H, G, D = 2, 4, 128
    c = Cache(gpu, [90, 333], 64, D, BF, q8, seed=27, room=room + 4 * new // 64 + 2)
    eager = Cache.__new__(Cache)
    eager.__dict__.update(c.__dict__)
    for name in ("k", "v", "k_scale", "v_scale", "seg_len"):
        if getattr(c, name) is not None:
            setattr(eager, name, getattr(c, name).clone())
    cu = _cu([new], gpu)
    q, k, v = (torch.zeros(new, n, D, device=gpu, dtype=BF) for n in (H * G, H, H))

    def step(x):
        _, nl = paged_append(k, v, *x.args(), cu_tokens=cu, max_tokens=new, **x.scales())
        out = paged_prompt_attn(q, x.k, x.v, x.table, nl, cu, 0.1, max_tokens=new, **x.scales())
        x.seg_len.copy_(nl)
        return out

    state = [x.clone() for x in (*_snapshot(c), c.seg_len) if x is not None]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip([t for t in (c.k, c.v, c.k_scale, c.v_scale, c.seg_len) if t is not None], state):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(c)
    for i in range(3):
        gen = torch.Generator(device=gpu).manual_seed(i)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device=gpu, generator=gen))
        graph.replay()
        want = step(eager)
        assert torch.equal(out, want), i
        if i == 1:
            torch.cuda.synchronize()
    _clean()
    assert torch.equal(c.seg_len, eager.seg_len) and c.seg_len.tolist() == [90 + 3 * new, 333 + 3 * new]
    assert torch.equal(c.k.view(torch.uint8), eager.k.view(torch.uint8))


def test_own_workspace(gpu):
    """Calls with a workspace of the caller's: eager and captured, two graphs of different sizes replayed in turn on it."""
    cs = [Cache(gpu, lens, 64, 128, BF, True, seed=28 + i) for i, lens in enumerate(([6000, 90, 2500], [3000] * 70))]
    qs = [_q(gpu, len(c.lens), 4, 128, BF) for c in cs]
    few = [_q(gpu, 3, 4 * len(c.lens), 128, BF) for c in cs]
    cu = _cu([3], gpu)
    ws = PagedWorkspace(70, 12, 128)
    assert ws.buf.device == cs[0].k.device

    def step(i, **kw):
        return (paged_decode_attn(qs[i], *cs[i].args(), 0.1, **cs[i].scales(), **kw),
                paged_prompt_attn(few[i], *cs[i].args(), cu, 0.1, **cs[i].scales(), **kw))

    want = [step(i) for i in range(2)]
    graphs, outs = [], []
    for i in range(2):
        got = step(i, workspace=ws)
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i, workspace=ws))
        graphs.append(g)
    for i in (0, 1, 1, 0, 0, 1):
        for o in outs[i]:
            o.zero_()
        graphs[i].replay()
        step(1 - i, workspace=ws)
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i])), i
    _clean()
    assert int(torch.count_nonzero(ws.buf[:ws.counters])) == 0
    E = _lib.WnwError
    for fn in (lambda: step(1, workspace=PagedWorkspace(70, 11, 128)), lambda: step(1, workspace=PagedWorkspace(5000, 16, 128)),
               lambda: PagedWorkspace(70, 17, 128), lambda: PagedWorkspace(-1, 1, 128), lambda: PagedWorkspace(4, 4, 128, "cpu")):
        with pytest.raises(E):
            fn()
    _clean()


@pytest.mark.parametrize("q8,dtype,D,G", [(True, BF, 128, 4), (False, FP, 64, 8), (True, FP, 256, 2)])
@pytest.mark.parametrize("new,old", [([300], [0]), ([64, 90], [500, 0]), ([200, 30, 80, 1], [300, 2000, 10, 0]), ([700], [0])],
                         ids=lambda x: "-".join(map(str, x)))
def test_prompts_in_a_wide_table(gpu, q8, dtype, D, G, new, old):
    """A table for far more rows than the segments have: each block of queries is cut by the rows that it sees."""
    c = Cache(gpu, [o + n for o, n in zip(old, new) for _ in range(2)], 64, D, dtype, q8, seed=30)
    wide = torch.full((c.table.shape[0], c.table.shape[1] + 500), -1, dtype=torch.int32, device=gpu)
    wide[:, :c.table.shape[1]] = c.table
    q = _q(gpu, sum(new), 2 * G, D, dtype)
    out = paged_prompt_attn(q, c.k, c.v, wide, c.seg_len, _cu(new, gpu), D ** -0.5, max_tokens=max(new), **c.scales())
    _clean()
    _prompt_check(c, q, out, new, 2, D ** -0.5)
