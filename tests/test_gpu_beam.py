"""Beam selection against 64-bit totals.

Scores: float32 of a total whose log-sum is off by at most 2^-20 (each exponential
and its argument's product off by 2^-22 of the term where it counts, a term in
32 additions of 2^-24, log and the rest in 64 bits) plus the rounding, 2^-24 of
its size.  Tokens and parents are equal where no two totals are nearer than that."""
import pytest
import torch

from tests.test_gpu_paged import _clean
from tests.test_gpu_paged_edges import _General
from wnw_amd import _lib
from wnw_amd.kv.beam import beam_select

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _totals(logits, scores, done, end):
    x = logits.double()
    t = scores.double().unsqueeze(2) + torch.log_softmax(x, dim=2)
    bad = ~torch.isfinite(t).any(2) | ~(x < float("inf")).all(2) | ~torch.isfinite(scores)
    t = torch.where(bad.unsqueeze(2) | ~torch.isfinite(t), -torch.inf, t)
    if done is not None:
        lone = torch.full_like(t, -torch.inf)
        lone[:, :, end] = torch.where(torch.isfinite(scores), scores.double(), -torch.inf)
        t = torch.where(done.unsqueeze(2), lone, t)
    return t.cpu()


def _check(logits, scores, k, got, done=None, end=0, exact_order=True):
    out, parents, tokens = (x.cpu() for x in got)
    B, W, V = logits.shape
    assert out.shape == parents.shape == tokens.shape == (B, k)
    assert out.dtype == F32 and parents.dtype == torch.int32 and tokens.dtype == torch.int64
    t = _totals(logits, scores, done, end).flatten(1)
    for b in range(B):
        value, at = torch.sort(t[b], descending=True, stable=True)
        m = min(k, int((value > -torch.inf).sum()))
        tol = 2.0 ** -20 + 2.0 ** -24 * value[:m].abs()
        assert bool(((out[b, :m].double() - value[:m]).abs() <= tol).all()), b
        assert bool((out[b, m:] == -torch.inf).all()) and parents[b, m:].tolist() == [b * W] * (k - m)
        assert tokens[b, m:].tolist() == [end] * (k - m)
        if m == 0:
            continue
        pick = (parents[b, :m] - b * W) * V + tokens[b, :m]
        assert pick.unique().numel() == m and int(parents[b, :m].min()) >= b * W and int(parents[b, :m].max()) < (b + 1) * W
        mine = t[b][pick]
        assert bool(((mine - value[:m]).abs() <= tol).all()), b  # as good, up to what the sums may be off
        same = pick == at[:m]
        if exact_order:
            gap = (value[:m] - mine).abs()
            assert bool((same | (gap > 0)).all()), (b, pick.tolist(), at[:m].tolist())


def _logits(gpu, B, W, V, dtype, seed, pad=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.randn(B * W, V + pad, device=gpu, generator=g) * 3
    return x.to(dtype)[:, :V].unflatten(0, (B, W)), -torch.rand(B, W, device=gpu, generator=g) * 5


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("B,W,V,k,pad", [(1, 1, 1, 1, 0), (1, 1, 1, 5, 3), (2, 3, 5, 4, 0), (1, 5, 7, 64, 1), (3, 2, 8, 16, 0),
                                         (2, 4, 127, 4, 2), (2, 64, 129, 64, 0), (1, 1, 2047, 1, 1), (1, 2, 2048, 7, 0),
                                         (4, 3, 2049, 6, 5), (1, 8, 32000, 16, 0), (2, 24, 51865, 48, 3), (1, 1, 262144, 64, 0),
                                         (40, 2, 1000, 2, 0)])
def test_select(gpu, dtype, B, W, V, k, pad):
    x, s = _logits(gpu, B, W, V, dtype, B * 100 + V, pad)
    got = beam_select(x, s, k)
    _clean()
    _check(x, s, k, got)
    assert all(torch.equal(a, b) for a, b in zip(got, beam_select(x, s, k)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [3, 100, 5000, 70001])
def test_equal_totals(gpu, dtype, V):
    """Ties go to the lower beam and token: constant rows, equal beams, many candidates at the border."""
    B, W, k = 3, 4, 8
    x = torch.zeros(B, W, V, device=gpu, dtype=dtype)
    s = torch.zeros(B, W, device=gpu)
    s[1, :2] = -1.0  # sample 1: beams 2 and 3 first
    x[2, :, 1::3] = 2.0
    got = beam_select(x, s, k)
    _clean()
    n = min(k, V)
    assert got[1][0, :n].tolist() == [0] * n and got[2][0, :n].tolist() == list(range(n))
    assert got[1][1, :n].tolist() == [6] * n and got[2][1, :n].tolist() == list(range(n))
    high = [i for i in range(V) if i % 3 == 1]
    want = [(w, t) for w in range(W) for t in high][:k]
    assert [(int(p) - 8, int(t)) for p, t in zip(got[1][2], got[2][2])][:len(want)] == want
    _check(x, s, k, got, exact_order=False)


def test_near_ties_at_many_places(gpu):
    """bf16 logits of few values: hundreds of candidates at the k-th total, in every group."""
    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.randint(0, 3, (2, 6, 40000), device=gpu, generator=g).to(BF)
    s = torch.zeros(2, 6, device=gpu)
    for k in (1, 6, 64):
        got = beam_select(x, s, k)
        _clean()
        _check(x, s, k, got, exact_order=False)
        for b in range(2):
            t = got[2][b][got[1][b] == got[1][b, 0]]
            assert torch.equal(t, t.sort().values)
            w = int(got[1][b, 0]) - 6 * b
            assert t.tolist() == (x[b, w] == 2).nonzero().flatten()[:t.numel()].tolist()


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_masked(gpu, dtype):
    """-inf among the logits, rows of nothing else, beams that offer nothing, fewer candidates than k."""
    x, s = _logits(gpu, 5, 4, 3001, dtype, 3)
    x = x.clone()
    x[0, :, 5:] = -torch.inf
    x[1, 1] = -torch.inf
    x[1, 2, 1:] = -torch.inf
    s[1, 3] = -torch.inf
    x[2] = -torch.inf
    x[2, 3, 3000] = 1.0
    s[3] = -torch.inf
    x[4, :, ::2] = torch.finfo(dtype).min
    for k in (4, 8, 64):
        got = beam_select(x, s, k, end=7)
        _clean()
        _check(x, s, k, got, end=7)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_not_finite(gpu, dtype):
    """NaN or +inf in a beam's logits or score: the error word, and no candidate of that beam; the others' as they are."""
    for what in (float("nan"), float("inf"), -float("nan")):
        for at in (0, 17, 4999):
            x, s = _logits(gpu, 2, 3, 5000, dtype, 4)
            x = x.clone()
            x[1, 1, at] = what
            got = beam_select(x, s, 6)
            torch.cuda.synchronize()
            assert _lib.device_error() == _lib.DEVERR_VALUES
            _check(x, s, 6, got)
    for what in (float("nan"), float("inf")):
        x, s = _logits(gpu, 2, 3, 5000, dtype, 5)
        s[0, 2] = what
        got = beam_select(x, s, 6)
        torch.cuda.synchronize()
        assert _lib.device_error() == _lib.DEVERR_VALUES
        _check(x, s, 6, got)


def test_finished(gpu):
    """Finished beams offer their score and `end` alone; their logits are not looked at."""
    x, s = _logits(gpu, 6, 5, 4001, BF, 6)
    done = torch.tensor([[i >> w & 1 for w in range(5)] for i in (0, 1, 31, 6, 9, 16)], dtype=torch.bool, device=gpu)
    s[3, 1] = -torch.inf
    x = x.clone()
    x[done] = float("nan")
    for k in (1, 5, 10, 64):
        got = beam_select(x, s, k, done=done, end=4000)
        _clean()
        _check(x, s, k, got, done, 4000)


def test_extreme_values(gpu):
    """Logits and scores of the types' range; -0 and 0 are equal."""
    x = torch.zeros(2, 2, 600, device=gpu)
    x[0, 0, 7], x[0, 1, 9] = 3.4e38, -3.4e38
    x[1] = -3.4e38
    x[1, :, 300] = -3.39e38
    s = torch.tensor([[-1e30, -2.0], [-3.0, -3.0]], device=gpu)
    got = beam_select(x, s, 4)
    _clean()
    _check(x, s, 4, got, exact_order=False)
    z = torch.zeros(1, 2, 50, device=gpu, dtype=BF)
    z[:, :, ::2] = -0.0
    got = beam_select(z, torch.zeros(1, 2, device=gpu), 5)
    _clean()
    assert got[2].tolist() == [[0, 1, 2, 3, 4]] and got[1].tolist() == [[0] * 5]


def test_strides(gpu):
    """Rows of a longer tensor, beams and samples at strides of their own, an expanded first step."""
    g = torch.Generator(device=gpu).manual_seed(8)
    big = torch.randn(4, 3, 7, 1003, device=gpu, generator=g).to(FP)
    s = -torch.rand(4, 7, device=gpu, generator=g)
    for x in (big[:, 1], big[:, 2, :, 3:1001], big[:, 0].transpose(0, 1), big[0, 0, :1].expand(4, 7, 1003), big[:, :, 0, ::2][:, [0] * 7]):
        ss = s if x.shape[:2] == s.shape else s.t()
        got = beam_select(x, ss, 9)
        _clean()
        _check(x, ss, 9, got, exact_order=False)


def test_captured(gpu):
    """A captured selection follows its inputs; two graphs and eager calls in turn."""
    x, s = _logits(gpu, 4, 4, 9001, BF, 9)
    x = x.clone()
    done = torch.zeros(4, 4, dtype=torch.bool, device=gpu)
    beam_select(x, s, 8, done=done, end=2)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = beam_select(x, s, 8, done=done, end=2)
        graphs.append((g, out))
    for step in range(4):
        y, t = _logits(gpu, 4, 4, 9001, BF, 20 + step)
        x.copy_(y)
        s.copy_(t)
        done[step] = True
        for g, _ in graphs:
            g.replay()
        want = beam_select(x, s, 8, done=done, end=2)
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        _check(x, s, 8, want, done, 2)
    _clean()


def test_refusals(gpu):
    x, s = _logits(gpu, 2, 3, 50, BF, 1)
    done = torch.zeros(2, 3, dtype=torch.bool, device=gpu)
    for bad in (dict(x=x[0]), dict(x=x.double()), dict(x=x.long()), dict(s=s.half()), dict(s=s[:1]), dict(s=s.flatten()), dict(k=0),
                dict(k=65), dict(k=-1), dict(done=done.int()), dict(done=done[0]), dict(end=-1), dict(end=50), dict(x=x.cpu()),
                dict(s=s.cpu()), dict(x=x[:, :0], s=s[:, :0]), dict(x=x[:, :, :0]), dict(s=s.clone().requires_grad_(True)),
                dict(x=x[:, :1].expand(2, 65, 50), s=s[:, :1].expand(2, 65))):
        c = dict(x=x, s=s, k=3, done=None, end=0)
        c.update(bad)
        with pytest.raises(_lib.WnwError):
            beam_select(c["x"], c["s"], c["k"], done=c["done"], end=c["end"])
    assert beam_select(x[:0], s[:0], 3)[0].shape == (0, 3)
    _clean()


def test_both_ways_into_a_call(gpu, monkeypatch):
    """The native way of the plain calls and the general way give the same bits."""
    x, s = _logits(gpu, 3, 4, 5001, FP, 11, 3)
    done = torch.rand(3, 4, device=gpu) < 0.3
    native = [beam_select(x, s), beam_select(x, s, 9, done=done, end=7), beam_select(x.float(), s, 1)]
    monkeypatch.setattr(_lib, "_callpath", _General())
    general = [beam_select(x, s), beam_select(x, s, 9, done=done, end=7), beam_select(x.float(), s, 1)]
    _clean()
    assert all(torch.equal(a, b) for n, g in zip(native, general) for a, b in zip(n, g))


def test_on_another_stream(gpu):
    """A selection on a stream of the caller's, behind work there that writes its logits."""
    x, s = _logits(gpu, 3, 5, 12001, BF, 12)
    want = beam_select(x, s, 7)
    stream = torch.cuda.Stream()
    for _ in range(3):
        late = torch.zeros_like(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(2_000_000)
            late.copy_(x)
            got = beam_select(late, s, 7)
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    _clean()


def test_rows_far_apart(gpu):
    """Samples and beams whose elements lie past 32 bits of offset."""
    room = torch.empty(2 ** 32 + 2 ** 21, dtype=FP, device=gpu)
    for strides in ((2 ** 32, 5001), (5001, 2 ** 32)):
        x = room.as_strided((2, 2, 5000), (*strides, 1))
        y, s = _logits(gpu, 2, 2, 5000, FP, 13)
        x.copy_(y)
        got = beam_select(x, s, 6)
        _clean()
        _check(y, s, 6, got)


def test_numbers_that_are_none(gpu):
    """k and end that are not whole numbers are refused; numpy's are taken."""
    import numpy as np
    x, s = _logits(gpu, 2, 3, 50, BF, 1)
    for kw in (dict(k=3.0), dict(k="3"), dict(end=1.5), dict(end=None)):
        with pytest.raises((_lib.WnwError, TypeError)):
            beam_select(x, s, **kw)
    assert all(torch.equal(a, b) for a, b in zip(beam_select(x, s, np.int64(3)), beam_select(x, s, 3)))
    _clean()
