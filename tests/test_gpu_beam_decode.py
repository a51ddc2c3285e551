"""A beam search over the paged cache, as a decoder runs it: prompts appended and
attended through a window, then in each step pages reserved and given back, a
token appended, attention through the window, the beams selected, samples
forked; now and then the pool is compacted.  A toy model: a token's q, k and v are
rows of a table, its logits a product with the attention's result."""
import pytest
import torch

from tests import pages_ref
from tests.paged_ref import E4M3, HALF
from tests.test_gpu_beam import _check as check_selection
from tests.test_gpu_paged import BF, _check, _clean, _cu
from wnw_amd.kv.beam import beam_select
from wnw_amd.kv.paged import paged_append, paged_decode_attn, paged_prompt_attn
from wnw_amd.kv.pages import paged_compact, paged_copy, paged_fork, paged_reserve

pytestmark = pytest.mark.gpu
H, G, D, R, V, W = 2, 2, 64, 16, 523, 3


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("window,sinks", [(40, 4), (25, 0), (1000, 4)])
def test_beam_decoding(gpu, q8, window, sinks):
    g = torch.Generator(device=gpu).manual_seed(window)
    qkv = torch.randn(V, H * (G + 2) * D, device=gpu, generator=g).to(BF)
    head = (torch.randn(H * G * D, V, device=gpu, generator=g) * 0.3).to(BF)
    prompts = [37, 50]
    B, P, M = len(prompts), 220, 12
    k_pages, v_pages = (torch.zeros(P, R, D, device=gpu).to(E4M3 if q8 else BF) for _ in range(2))
    scales = dict(k_scale=torch.ones(P, device=gpu), v_scale=torch.ones(P, device=gpu)) if q8 else {}
    table = torch.full((B * H, M), -1, dtype=torch.int32, device=gpu)
    refs, lens = torch.zeros(P, dtype=torch.int32, device=gpu), torch.zeros(B * H, dtype=torch.int32, device=gpu)
    view = dict(window=window, sinks=sinks)
    scale = D ** -0.5

    def split(tokens):
        return (x.unflatten(1, (-1, D)) for x in qkv[tokens].split([H * G * D, H * D, H * D], dim=1))

    def seen_rows(pages, sc, s, n):
        """The rows of segment s that its last one sees, in 64 bits, and their places."""
        at = [j for j in range(n) if j < sinks or j > n - 1 - window]
        ids = table[s, torch.tensor(at, device=gpu) // R].long()
        assert bool((ids >= 0).all())
        x = pages.view(torch.uint8)[ids, torch.tensor(at) % R].view(E4M3).double() * sc[ids].double().unsqueeze(1) if q8 \
            else pages[ids, torch.tensor(at) % R].double()
        return x, at

    def check_attention(q, out, history):
        """Each sample's last token against the cache's rows, and these against what was appended."""
        for b, tokens in enumerate(history):
            n = len(tokens)
            _, k, v = split(torch.tensor(tokens, device=gpu))
            for h in range(H):
                kk, at = seen_rows(k_pages, scales.get("k_scale"), b * H + h, n)
                vv, _ = seen_rows(v_pages, scales.get("v_scale"), b * H + h, n)
                for got, want in ((kk, k[at, h].double()), (vv, v[at, h].double())):
                    if q8:  # 2^-4 of the value, or half a subnormal code's step, twice: a page is rescaled as it fills
                        assert bool(((got - want).abs() <= 2.0 ** -3 * want.abs() + 2.0 ** -9 * want.abs().max()).all())
                    else:
                        assert torch.equal(got, want)
                x = q[b, h * G:(h + 1) * G].double()
                w = torch.softmax(x @ kk.t().contiguous() * scale, dim=1)
                ref, A = w @ vv, w @ vv.abs()
                _check(out[b, h * G:(h + 1) * G], ref, HALF[BF] * ref.abs() + (HALF[BF] + 2.0 ** -13) * A, (b, h, n))

    with torch.no_grad():
        # the prompts
        history = [torch.randint(V, (n,), generator=g, device=gpu).tolist() for n in prompts]
        cu = _cu(prompts, gpu)
        table, refs = paged_reserve(table, lens, refs, R, cu_tokens=cu)
        q, k, v = split(torch.tensor(sum(history, []), device=gpu))
        _, lens = paged_append(k, v, k_pages, v_pages, table, lens, cu_tokens=cu, max_tokens=max(prompts), **scales)
        out = paged_prompt_attn(q, k_pages, v_pages, table, lens, cu, scale, max_tokens=max(prompts), **view, **scales)
        last = cu[1:].long() - 1
        check_attention(q[last], out[last], history)
        # the first selection: one beam a sample, W of its candidates; the samples become B * W
        logits = out[last].flatten(1) @ head
        total, parents, tokens = beam_select(logits.view(B, 1, V), torch.zeros(B, 1, device=gpu), W)
        check_selection(logits.view(B, 1, V), torch.zeros(B, 1, device=gpu), W, (total, parents, tokens))
        for step in range(45):
            # go on from the parents
            table, lens, refs, copies = paged_fork(table, lens, refs, parents.flatten(), R, kv_heads=H)
            paged_copy(k_pages, v_pages, copies, **scales)
            history = [history[p] + [t] for p, t in zip(parents.flatten().tolist(), tokens.flatten().tolist())]
            # a page for the next row, those behind the window back
            table, refs = paged_reserve(table, lens, refs, R, **view)
            if step % 11 == 10:
                table, refs, moves, used = paged_compact(table, refs, R)
                paged_copy(k_pages, v_pages, moves, **scales)
                assert int(refs[:int(used)].min()) > 0 and int(refs[int(used):].sum()) == 0
            q, k, v = split(tokens.flatten())
            _, lens = paged_append(k, v, k_pages, v_pages, table, lens, **scales)
            o = paged_decode_attn(q.reshape(B * W * H, G, D), k_pages, v_pages, table, lens, scale, **view, **scales)
            logits = (o.view(B * W, H * G * D) @ head).view(B, W, V)
            done = (torch.rand(B, W, device=gpu, generator=g) < 0.1) if step % 5 == 4 else None
            before = total
            total, parents, tokens = beam_select(logits, before, W, done=done, end=3)
            if step % 4 == 0 or step > 40:
                _clean()
                check_attention(q, o.view(B * W, H * G, D), history)
                check_selection(logits, before, W, (total, parents, tokens), done, 3)
                assert refs.tolist() == pages_ref.counts(table.tolist(), P)
                assert lens.tolist() == [len(x) for x in history for _ in range(H)]
    _clean()
    # nothing stays behind: samples that no one goes on from
    none = torch.full((1,), -1, dtype=torch.int32, device=gpu)
    _, _, refs, _ = paged_fork(table, lens, refs, none, R, kv_heads=H)
    assert int(refs.abs().sum()) == 0
