"""Numbers past 64 bits are refused, not taken modulo 2^64."""
import pytest
import torch

from tests.test_gpu_paged import _clean
from wnw_amd import _lib
from wnw_amd.kv.beam import beam_select
from wnw_amd.kv.pages import paged_compact, paged_fork, paged_reserve

pytestmark = pytest.mark.gpu


def test_refused(gpu):
    def t(x):
        return torch.tensor(x, dtype=torch.int32, device=gpu)

    table, lens, refs, parents = t([[0, 1], [2, -1]]), t([20, 5]), t([1, 1, 1, 0]), t([0, 1])
    x, s = torch.zeros(1, 2, 50, device=gpu), torch.zeros(1, 2, device=gpu)
    for wrap in (1 << 64, -(1 << 64), 3 << 64):
        for call in (lambda: paged_reserve(table, lens, refs, 16, tokens=wrap + 1), lambda: paged_reserve(table, lens, refs, wrap + 16),
                     lambda: paged_fork(table, lens, refs, parents, wrap + 16, kv_heads=1),
                     lambda: paged_fork(table[:0], lens[:0], refs, parents[:0], 16, kv_heads=wrap + 1),
                     lambda: paged_compact(table, refs, wrap + 16), lambda: beam_select(x, s, 2, end=wrap + 3),
                     lambda: beam_select(x, s, wrap + 2)):
            with pytest.raises(_lib.WnwError):
                call()
    _clean()
