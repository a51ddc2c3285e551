"""Windowed attention over the paged cache where a segment's window shows no row:
what is not seen is neither looked up nor read.  Which blocks are seen is taken
from the rows that each token sees, one by one; every other block's entry is no
page, and the page that it had holds NaN.  Tolerances as in
test_gpu_paged_window.py."""
import pytest
import torch

from tests.paged_ref import Cache
from tests.test_gpu_paged import BF, FP, _clean, _cu, _q
from tests.test_gpu_paged_window import _decode_check, _each, _prompt_check, _seen
from wnw_amd.kv.paged import paged_append, paged_decode_attn, paged_prompt_attn
from wnw_amd.kv.pages import paged_reserve

pytestmark = pytest.mark.gpu


def _hide_unseen(c, new, window, sinks):
    N = len(c.lens)
    H = N // len(new)
    for s, (w, z) in enumerate(zip(_each(window, N), _each(sinks, N))):
        n = c.lens[s]
        seen = _seen(n, torch.arange(n - new[s // H], n), w, z).any(0).tolist()
        for j in range(-(-n // c.page)):
            if any(seen[j * c.page:(j + 1) * c.page]):
                continue
            page = int(c.table[s, j])
            for pages in (c.k, c.v):
                (pages.view(torch.uint8) if c.q8 else pages)[page] = 0x7f if c.q8 else float("nan")
            for scales in (c.k_scale, c.v_scale):
                if scales is not None:
                    scales[page] = float("nan")
            c.table[s, j] = (-1, 0x7fffffff, -9)[j % 3]


LENS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 129, 300, 2500]


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D,G,page", [(BF, 128, 4, 16), (FP, 64, 8, 64), (BF, 256, 7, 32)])
def test_decode_of_sinks_alone(gpu, q8, dtype, D, G, page):
    for sinks in (0, 4, 16, 33, 64):
        c = Cache(gpu, LENS, page, D, dtype, q8, seed=sinks)
        _hide_unseen(c, [1] * len(LENS), 0, sinks)
        q = _q(gpu, len(LENS), G, D, dtype)
        out = paged_decode_attn(q, *c.args(), D ** -0.5, window=0, sinks=sinks, **c.scales())
        _clean()
        _decode_check(c, q, out, 0, sinks, D ** -0.5)


def _some_zero(gpu, n):
    """Windows and sinks of n segments: every other window 0."""
    window = torch.tensor([0 if i % 2 else (1, 17, 200, 1 << 30)[i // 2 % 4] for i in range(n)], dtype=torch.int32)
    sinks = torch.tensor([(4, 0, 70, 16, 1)[i % 5] for i in range(n)], dtype=torch.int32)
    return window.to(gpu), sinks.to(gpu)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("lens", [[9000, 12000, 300, 20000], [i % 211 for i in range(400)]], ids=["long", "many"])
def test_decode_of_some_windows_zero(gpu, q8, lens):
    c = Cache(gpu, lens, 16, 64, BF, q8, seed=2)
    window, sinks = _some_zero(gpu, len(lens))
    _hide_unseen(c, [1] * len(lens), window, sinks)
    q = _q(gpu, len(lens), 4, 64, BF)
    out = paged_decode_attn(q, *c.args(), 0.2, window=window, sinks=sinks, **c.scales())
    _clean()
    _decode_check(c, q, out, window, sinks, 0.2)


# few: the decode kernel's; the others the prompt kernel's, blocks shared out where windows are on the device
PROMPTS = [([1, 2, 3], [0, 70, 1]), ([33, 5, 64, 7], [0, 9, 100, 1000]), ([129, 200], [0, 333]), ([300], [9000])]


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,D,G,page", [(BF, 128, 4, 64), (FP, 128, 7, 16), (FP, 64, 4, 32), (BF, 256, 2, 16)])
@pytest.mark.parametrize("new,old", PROMPTS, ids=["few", "ragged", "longer", "split"])
def test_prompt_of_sinks_alone(gpu, q8, dtype, D, G, page, new, old):
    H = 2
    lens = [a + b for a, b in zip(new, old) for _ in range(H)]
    mixed = _some_zero(gpu, len(lens))
    for window, sinks in ((0, 0), (0, 4), (0, 64), (0, 90), mixed):
        c = Cache(gpu, lens, page, D, dtype, q8, seed=3)
        _hide_unseen(c, new, window, sinks)
        q = _q(gpu, sum(new), H * G, D, dtype)
        out = paged_prompt_attn(q, *c.args(), _cu(new, gpu), D ** -0.5, max_tokens=max(new), window=window, sinks=sinks,
                                **c.scales())
        _clean()
        _prompt_check(c, q, out, new, window, sinks, D ** -0.5)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("new", [[2, 0, 1, 0], [60, 0, 7, 0]], ids=["few", "long"])
@pytest.mark.parametrize("window,sinks", [(40, 4), (0, 20), (1 << 30, 0)])
def test_samples_without_tokens(gpu, q8, new, window, sinks):
    """No row of a sample without tokens is seen: none of its blocks is looked up, whatever its length."""
    H, G, D = 2, 4, 64
    lens = [n for n in (90, 500, 33, 16) for _ in range(H)]
    c = Cache(gpu, lens, 16, D, BF, q8, seed=5)
    _hide_unseen(c, new, window, sinks)
    for b, n in enumerate(new):
        assert n or int(c.table[b * H:(b + 1) * H, 0].max()) == -1
    q = _q(gpu, sum(new), H * G, D, BF)
    out = paged_prompt_attn(q, *c.args(), _cu(new, gpu), 0.2, max_tokens=max(new), window=window, sinks=sinks, **c.scales())
    _clean()
    _prompt_check(c, q, out, new, window, sinks, 0.2)


@pytest.mark.parametrize("sinks", [0, 4, 16])
def test_a_loop_of_sinks_alone(gpu, sinks):
    """Pages reserved, a row appended, attention through a window of 0: a segment keeps its sinks' block and the one of the row
    that is written, the last of a block too (row + 1 a multiple of the page's rows)."""
    N, G, D, R = 2, 4, 64, 16
    P = 3 * N  # pages that a call gives back serve the next one
    g = torch.Generator(device=gpu).manual_seed(7)
    table = torch.full((N, 6), -1, dtype=torch.int32, device=gpu)
    refs, lens = torch.zeros(P, dtype=torch.int32, device=gpu), torch.zeros(N, dtype=torch.int32, device=gpu)
    k_pages, v_pages = (torch.zeros(P, R, D, device=gpu, dtype=BF) for _ in range(2))
    rows = torch.randn(2, 90, N, D, device=gpu, generator=g).to(BF)
    for i in range(90):
        paged_reserve(table, lens, refs, R, window=0, sinks=sinks, out=(table, refs))
        assert int(table[0, i // R]) >= 0 and int((table[0] >= 0).sum()) == (2 if sinks and i >= R else 1)
        _, lens = paged_append(rows[0, i].unsqueeze(0), rows[1, i].unsqueeze(0), k_pages, v_pages, table, lens)
        q = torch.randn(N, G, D, device=gpu, generator=g).to(BF)
        out = paged_decode_attn(q, k_pages, v_pages, table, lens, 0.2, window=0, sinks=sinks)
        _clean()
        n = min(i + 1, sinks)
        for s in range(N):
            k, v = rows[0, :n, s].double(), rows[1, :n, s].double()
            w = torch.softmax(q[s].double() @ k.t().contiguous() * 0.2, dim=1)
            ref, A = w @ v, w @ v.abs()
            assert bool(((out[s].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -13 * A).all()), (i, s)
