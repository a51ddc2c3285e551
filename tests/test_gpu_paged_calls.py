"""Calls of the paged cache's operators that are refused: with the library's own
reason, whatever ran before on the stream; traced ones, and inputs with tangents."""
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from tests.paged_ref import Cache
from tests.test_gpu_paged import BF, _clean, _cu, _q
from tests.test_gpu_paged_edges import _General
from wnw_amd import _lib
from wnw_amd.kv import paged
from wnw_amd.kv.paged import paged_append, paged_decode_attn, paged_prompt_attn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("tokens", [2, 40])
def test_caches_that_the_library_refuses(gpu, tokens, captured):
    """Page sizes and head sizes that the library does not take: its own refusal, on a stream without a workspace too."""
    for R, D in ((24, 64), (16, 96), (512, 64), (16, 512)):
        pages = torch.zeros(3, R, D, device=gpu, dtype=BF)
        table, lens = torch.zeros(1, 2, dtype=torch.int32, device=gpu), torch.full((1,), 8, dtype=torch.int32, device=gpu)
        q, cu = torch.zeros(tokens, 1, D, device=gpu, dtype=BF), _cu([tokens], gpu)
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        paged._workspaces.pop((0, stream.cuda_stream), None)
        with torch.cuda.stream(stream):
            calls = [lambda: paged_prompt_attn(q, pages, pages, table, lens, cu, 0.1),
                     lambda: paged_decode_attn(q[:1], pages, pages, table, lens, 0.1)]
            graph = torch.cuda.CUDAGraph()
            if captured:
                graph.capture_begin()
            try:
                for fn in calls:
                    with pytest.raises(_lib.WnwError, match="page_rows|head_dim"):
                        fn()
            finally:
                if captured:
                    torch.zeros(1, device=gpu)  # a graph of something
                    graph.capture_end()
    _clean()


def test_traced_and_dual_calls_are_refused(gpu):
    """A trace would record outputs that nothing writes, and a tangent would be lost: both are refused, on both ways in."""
    c = Cache(gpu, [40, 50], 32, 64, BF, False, seed=70)
    q, kv, cu = _q(gpu, 2, 4, 64, BF), _q(gpu, 2, 1, 64, BF), _cu([1, 1], gpu)
    long, cu_long = _q(gpu, 60, 4, 64, BF), _cu([30, 30], gpu)
    pos, freq = torch.arange(2, device=gpu), torch.ones(32, device=gpu)
    was = c.k.clone(), c.v.clone()
    calls = {"decode": (lambda x: paged_decode_attn(x, *c.args(), 0.1), q),
             "few": (lambda x: paged_prompt_attn(x, *c.args(), cu, 0.1), q),
             "prompt": (lambda x: paged_prompt_attn(x, *c.args(), cu_long, 0.1), long),
             "append k": (lambda x: paged_append(x, kv, *c.args())[1], kv),
             "append v": (lambda x: paged_append(kv, x, *c.args())[1], kv),
             "append q": (lambda x: paged_append(kv, kv, *c.args(), q=x, positions=pos, inv_freq=freq)[0], q),
             "append freq": (lambda x: paged_append(kv, kv, *c.args(), q=q, positions=pos, inv_freq=x)[0], freq),
             "pages": (lambda x: paged_decode_attn(q, c.k, x, c.table, c.seg_len, 0.1), c.v)}
    for name, (fn, x) in calls.items():
        with pytest.raises(_lib.WnwError, match="trace"):
            torch.jit.trace(fn, (x,), check_trace=False)
        with pytest.raises(_lib.WnwError, match="trace"):
            make_fx(fn)(x)
        with forward_ad.dual_level(), pytest.raises(_lib.WnwError, match="gradient"):
            fn(forward_ad.make_dual(x, torch.ones_like(x)))
        for general in (False, True):
            with torch.no_grad(), forward_ad.dual_level(), pytest.MonkeyPatch.context() as m:
                if general:
                    m.setattr(_lib, "_callpath", _General())
                with pytest.raises(_lib.WnwError, match="gradient"):
                    fn(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises((_lib.WnwError, RuntimeError)):
            torch.func.jvp(fn, (x,), (torch.ones_like(x),))
    _clean()
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip((c.k, c.v), was))  # rows past the lengths: NaN
    with forward_ad.dual_level(), torch.no_grad():  # plain tensors beside someone else's tangents
        assert bool(torch.isfinite(paged_decode_attn(q, *c.args(), 0.1)).all())
