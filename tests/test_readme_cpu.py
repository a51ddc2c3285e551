"""README's step of beam search, run as it stands with operators that are plain
Python: which beams have finished is carried along."""
import os
import random
import types

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _snippet():
    path = os.path.join(ROOT, "README.md")
    if not os.path.isfile(path):
        pytest.skip("no README here")
    text = open(path, encoding="utf-8").read()
    lines = text[text.index("A step of beam search"):].splitlines()[2:]
    block = []
    for line in lines:
        if line and not line.startswith("    "):
            break
        block.append(line[4:])
    return "\n".join(x for x in block if not x.startswith("from "))


def test_beam_search_step():
    samples, beams, V, end = 3, 4, 6, 2
    rng = random.Random(1)
    code = compile(_snippet(), "README.md", "exec")
    ended = [[False] * beams for _ in range(samples)]  # of each beam, kept by hand
    log = []

    def beam_select(logits, scores, *, done, end):
        assert done.dtype == torch.bool and done.tolist() == ended
        parents = torch.tensor([[b * beams + rng.randrange(beams) for _ in range(beams)] for b in range(samples)])
        tokens = torch.tensor([[end if ended[b][int(p) - b * beams] else rng.randrange(V) for p in row]
                               for b, row in enumerate(parents)])
        log.append((parents, tokens))
        return scores, parents.int(), tokens

    names = types.SimpleNamespace(**{x: None for x in "page_table seg_len page_refs R k_pages v_pages scale k_scale v_scale".split()})
    scope = dict(vars(names), samples=samples, beams=beams, V=V, end_token=end, B=samples * beams, Hkv=1, G=1, D=1, torch=torch,
                 q=torch.zeros(samples * beams, 1, 1), logits=torch.zeros(samples * beams, V), scores=torch.zeros(samples, beams),
                 done=torch.zeros(samples, beams, dtype=torch.bool), beam_select=beam_select,
                 paged_reserve=lambda *a, **k: (None, None), paged_decode_attn=lambda *a, **k: None,
                 paged_fork=lambda *a, **k: (None,) * 4, paged_copy=lambda *a, **k: None)
    for _ in range(30):
        exec(code, scope)
        parents, tokens = log[-1]
        ended = [[ended[b][int(p) - b * beams] or int(t) == end for p, t in zip(parents[b], tokens[b])] for b in range(samples)]
    assert any(map(any, ended))
