"""Counts that do not agree with the table.  A page is free where its count is 0,
for every call alike; a compaction takes an entry that names a free page for -1
and sets the device error word, so that no page that moves lands under it."""
import random

import pytest
import torch

from tests import pages_ref
from tests.test_gpu_pages import _state, _t, _wide
from wnw_amd import _lib
from wnw_amd.kv.pages import paged_compact, paged_fork, paged_reserve

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,H,R,M,P", [(1, 1, 64, 4, 10), (3, 2, 16, 9, 70), (8, 4, 32, 20, 700), (20, 4, 16, 40, 5001)])
@pytest.mark.parametrize("negative", [False, True])
def test_compact_of_named_pages_without_a_count(gpu, B, H, R, M, P, negative):
    rng = random.Random(P)
    for _ in range(3):
        table, _, refs = _state(rng, B, H, R, M, P)
        named = sorted({e for row in table for e in row if e >= 0})
        gone = [p for p in named if rng.random() < 0.3] or named[:1]
        for p in gone:
            refs[p] = 0
        if negative:  # counts that are used, though no number of entries
            for p in named:
                if refs[p] and rng.random() < 0.3:
                    refs[p] = -refs[p]
        kept = [[-1 if e in set(gone) else e for e in row] for row in table]
        want, after, moves, used = pages_ref.compact(kept, [abs(c) for c in refs], R)
        after = list(refs)
        for a, b, _ in moves:
            if a >= 0:
                after[b], after[a] = refs[a], 0
        was, _ = _wide(table, M, gpu)
        counts = _t(refs, gpu)
        for out in (None, (was, counts)):
            got = paged_compact(was, counts, R, out=out)
            torch.cuda.synchronize()
            assert _lib.device_error() == (_lib.DEVERR_BOUNDS if gone else 0)
            assert got[0].tolist() == want and got[1].tolist() == after
            assert got[2].tolist() == moves and got[3].tolist() == [used]
        paged_compact(was, counts, R)  # what it gives agrees again
        torch.cuda.synchronize()
        assert _lib.device_error() == 0


def test_negative_counts_are_not_free(gpu):
    table, lens = _t([[1, -1], [3, -1]], gpu), _t([16, 5], gpu)
    refs = _t([-1, 1, -7, 1, 0, 0], gpu)
    new, after = paged_reserve(table, lens, refs, 16, tokens=1)
    assert new.tolist() == [[1, 4], [3, -1]] and after.tolist() == [-1, 1, -7, 1, 1, 0]
    new, _, after, _ = paged_fork(table, lens, refs, _t([1, 1], gpu), 16, kv_heads=1)
    assert new.tolist() == [[3, -1], [4, -1]] and after.tolist() == [-1, 0, -7, 1, 1, 0]
    new, after, moves, used = paged_compact(table, refs, 16)
    assert used.tolist() == [4] and new.tolist() == table.tolist() and after.tolist() == refs.tolist()
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
