"""Calls of the paged cache's operators that are refused with the library's own
reason, whatever ran before on the stream."""
import pytest
import torch

from tests.test_gpu_paged import BF, _clean, _cu
from wnw_amd import _lib
from wnw_amd.kv import paged
from wnw_amd.kv.paged import paged_decode_attn, paged_prompt_attn

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
