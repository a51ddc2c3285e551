"""The order of a selection.  Within a beam the log-sum cancels: its picks are its
best logits, equal ones by the lower token, however near to each other.  Between
beams totals are in order up to what their log-sums are off, 2^-18:

an exponential's argument d = x - max, |d| times log2 e, is off by 2.3 * 2^-24 of
its size, its value by twice 2^-24 more; eight terms add up in seven roundings;
the factor that joins tasks likewise, twice 2^-24 more.  Over n = 2^17 terms the
mean of |d| under the softmax is at most 8.7 (t - 1 for t = 1 + n exp(-t)): 2.3 *
8.7 + 11 = 31 times 2^-24."""
import pytest
import torch

from tests.test_gpu_paged import _clean
from wnw_amd.kv.beam import beam_select

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
LOG_SUM = 2.0 ** -18


def _check_order(logits, scores, k, got):
    out, parents, tokens = (x.cpu() for x in got)
    B, W, V = logits.shape
    total = (scores.double().unsqueeze(2) + torch.log_softmax(logits.double(), dim=2)).cpu()
    for b in range(B):
        assert k <= W * V
        taken = []
        for w in range(W):
            mine = tokens[b][parents[b] == b * W + w].tolist()
            best = torch.sort(logits[b, w].double(), descending=True, stable=True).indices[:len(mine)].tolist()
            assert mine == best, (b, w)
            taken += [(w, t) for t in mine]
        assert len(taken) == k
        t = total[b][(parents[b] - b * W).long(), tokens[b]]
        assert bool((t[1:] <= t[:-1] + 2 * LOG_SUM).all()), b
        left = total[b].clone()
        for w, v in taken:
            left[w, v] = -torch.inf
        assert float(left.max()) <= float(t[-1]) + 2 * LOG_SUM, b
        assert bool(((out[b].double() - t).abs() <= LOG_SUM + 2.0 ** -24 * t.abs()).all()), b


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("B,W,V,k", [(1, 1, 64, 64), (2, 3, 129, 20), (3, 4, 2049, 64), (1, 8, 32000, 16), (2, 5, 131072, 10)])
def test_order_within_a_beam(gpu, dtype, B, W, V, k):
    g = torch.Generator(device=gpu).manual_seed(V)
    x = (torch.randn(B, W, V, device=gpu, generator=g) * 3).to(dtype)
    s = -torch.rand(B, W, device=gpu, generator=g)
    got = beam_select(x, s, k)
    _clean()
    _check_order(x, s, k, got)


@pytest.mark.parametrize("score", [-1000.0, -1.0e6])
@pytest.mark.parametrize("V", [200, 5000, 40000])
def test_totals_that_32_bits_would_make_equal(gpu, score, V):
    """Logits one and two steps of 2^-21 apart, the better ones behind: totals near -1000 lie 2^-14 apart in 32 bits."""
    B, W, k = 2, 2, 12
    g = torch.Generator(device=gpu).manual_seed(3)
    x = torch.randn(B, W, V, device=gpu, generator=g).clamp(-3, 3)
    for b in range(B):
        for w in range(W):
            at = torch.randperm(V, generator=g, device=gpu)[:24].sort().values
            steps = torch.tensor([i + (i > 7) + (i > 15) for i in range(24)], device=gpu)  # ascending: a lower token is worse
            x[b, w, at] = 4.0 + steps * 2.0 ** -21
    s = torch.tensor([[score, score], [score, score - 0.25]], device=gpu)
    got = beam_select(x, s, k)
    _clean()
    assert bool((got[0].diff(dim=1) == 0).any())  # (equal once they are rounded)
    _check_order(x, s, k, got)


def test_far_spread_logits(gpu):
    """Log-sums of many small terms, where the exponentials' arguments are largest: still within the bound."""
    B, W, V, k = 2, 4, 131072, 8
    g = torch.Generator(device=gpu).manual_seed(4)
    x = torch.rand(B, W, V, device=gpu, generator=g) * 1e-3 - 10.6  # one logit of 0 against all others together
    x[:, :, 77777] = torch.arange(W, device=gpu) * 0.37
    s = torch.zeros(B, W, device=gpu)
    for y in (x, x + 3000.0, x - 3000.0):
        got = beam_select(y, s, k)
        _clean()
        _check_order(y, s, k, got)
