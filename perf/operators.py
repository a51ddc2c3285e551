"""Measured cases of the paged cache's operators: the append that rotates,
decode attention and prompt attention over pages of 16 or 8 bits.

Each case is one call for one layer, as a decoder makes it.  The shapes are
those of ``wnw_amd/workloads.py``, ``wnw_amd/offload_bench.py`` and
``perf/cases.py`` (32 / 8 and 28 / 4 heads at head_dim 128, long audio, short
class-B segments beside long class-A ones), the head sizes, groups and types
that the tests hold the attention to, and sizes between and around them.  With
``own`` the calls are the package's, otherwise the same mathematics in
elementary torch operations.

A cache: K and V pages [P, R, D], a page table [N, M] of page indices (-1: no
page) and the lengths [N] of the N = B * Hkv segments.  Pages of 8 bits hold
e4m3 codes that stand for code * scale, one scale per page of K and of V.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # One user's decode step: one token appended in 8 bits.  The smallest call.
        dict(name="append_b1_token", kind="append", dtype="bf16", q8=True, batch=1, hkv=8, group=4, dim=128, page=64,
             rot=128, axes=1, interleaved=False, tokens=1, cached=813, ragged=False, layout=1),
        # A serving batch's step: 28 / 4 heads, positions of three axes, 16-bit pages of 16 rows.
        dict(name="append_b64_axes", kind="append", dtype="bf16", q8=False, batch=64, hkv=4, group=7, dim=128, page=16,
             rot=128, axes=3, interleaved=False, tokens=1, cached=3001, ragged=True, layout=2),
        # A whole prompt (three minutes of audio) into 8 bits.
        dict(name="append_prompt", kind="append", dtype="bf16", q8=True, batch=1, hkv=8, group=4, dim=128, page=64,
             rot=128, axes=1, interleaved=False, tokens=4564, cached=0, ragged=False, layout=3),
        # Ragged chunks onto pages that are partly filled, half precision, half of each head rotated in adjacent pairs.
        dict(name="append_chunks_f16", kind="append", dtype="fp16", q8=True, batch=6, hkv=4, group=8, dim=64, page=32,
             rot=32, axes=1, interleaved=True, tokens=701, cached=1203, ragged=True, layout=4),
        # One user, one minute of audio: the shortest decode attention.
        dict(name="decode_b1_short", kind="decode", dtype="bf16", q8=True, batch=1, hkv=8, group=4, dim=128, page=64,
             heads_a=2, full=813, short=160, ragged=False, layout=5),
        # The benchmark's decode step in 8 bits: batch 8, ten minutes of audio each.
        dict(name="decode_b8_long", kind="decode", dtype="bf16", q8=True, batch=8, hkv=8, group=4, dim=128, page=64,
             heads_a=2, full=7564, short=512, ragged=False, layout=6),
        # A serving batch of very different lengths, groups of seven, 16-bit pages of 16 rows.
        dict(name="decode_b64_ragged", kind="decode", dtype="bf16", q8=False, batch=64, hkv=4, group=7, dim=128, page=16,
             heads_a=2, full=5003, short=516, ragged=True, layout=7),
        # Heads of 256 elements in groups of sixteen, half precision over 8 bits.
        dict(name="decode_f16_d256", kind="decode", dtype="fp16", q8=True, batch=8, hkv=2, group=16, dim=256, page=128,
             heads_a=1, full=8099, short=1777, ragged=True, layout=8),
        # A whole prompt over the 8-bit cache that its append has filled.
        dict(name="prompt_b1", kind="prompt", dtype="bf16", q8=True, batch=1, hkv=8, group=4, dim=128, page=64,
             tokens=4564, cached=0, ragged=False, layout=9),
        # A chunk of a long prompt: 512 tokens behind 22,116 cached ones.
        dict(name="prompt_chunk", kind="prompt", dtype="bf16", q8=True, batch=1, hkv=8, group=4, dim=128, page=64,
             tokens=512, cached=22116, ragged=False, layout=10),
        # Prompts of several users, half precision, 16-bit pages of 16 rows, some with a cached beginning.
        dict(name="prompt_ragged_f16", kind="prompt", dtype="fp16", q8=False, batch=5, hkv=4, group=7, dim=128, page=16,
             tokens=1501, cached=333, ragged=True, layout=11),
        # Four proposed tokens a user, checked against long caches.
        dict(name="prompt_four_tokens", kind="prompt", dtype="bf16", q8=True, batch=8, hkv=8, group=4, dim=128, page=64,
             tokens=4, cached=7560, ragged=False, layout=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt"])
    dim = rng.choice([128, 128, 128, 64, 256])
    c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16"]), q8=rng.random() < 0.7, batch=_log(rng, 1, 48),
             hkv=rng.choice([1, 2, 4, 8, 8]), group=rng.choice([1, 2, 4, 4, 7, 8, 16]), dim=dim,
             page=rng.choice([16, 32, 64, 64, 128, 256]), ragged=rng.random() < 0.6, layout=rng.randrange(1, 1 << 20))
    if kind == "append":
        c |= dict(rot=rng.choice([dim, dim, dim // 2]), axes=rng.choice([1, 1, 3]), interleaved=rng.random() < 0.3,
                  tokens=rng.choice([1, _log(rng, 1, 4000)]), cached=_log(rng, 1, 9000))
        while c["batch"] * c["tokens"] * c["hkv"] * (c["group"] + 2) * dim > 20e6:
            c["batch"], c["tokens"] = max(1, c["batch"] // 2), max(1, int(c["tokens"] * 0.8))
        while c["batch"] * c["hkv"] * (c["cached"] + c["tokens"]) * dim > 60e6:
            c["batch"], c["cached"] = max(1, c["batch"] // 2), max(1, int(c["cached"] * 0.7))
    elif kind == "decode":
        c |= dict(heads_a=max(1, round(c["hkv"] * rng.uniform(0.15, 0.5))), full=_log(rng, 1, 24000),
                  short=_log(rng, 1, 1500))
        while c["batch"] * c["hkv"] * max(c["full"], c["short"]) * dim > 200e6:
            c["batch"], c["full"] = max(1, c["batch"] // 2), max(1, int(c["full"] * 0.7))
    else:
        c |= dict(batch=_log(rng, 1, 8), tokens=_log(rng, 2, 4000), cached=rng.choice([0, _log(rng, 1, 20000)]))
        while c["batch"] * c["hkv"] * c["group"] * c["tokens"] * (c["tokens"] + c["cached"]) * dim > 60e9:
            c["batch"], c["tokens"] = max(1, c["batch"] // 2), max(2, int(c["tokens"] * 0.8))
            c["cached"] = int(c["cached"] * 0.8)
    return c


# --------------------------------------------------------------------------
# geometry: fixed by the case alone
# --------------------------------------------------------------------------
def _mixed(layout, n, size, least, ragged):
    """n lengths up to ``size``, the first of them ``size`` itself."""
    g = torch.Generator().manual_seed(layout)
    x = torch.rand(n, generator=g)
    return [size if i == 0 or not ragged else max(least, int(size * (0.1 + 0.9 * float(x[i])))) for i in range(n)]


def _geometry(c):
    """Host lengths: tokens of each sample in this call, rows of each segment before and after it."""
    B, H = c["batch"], c["hkv"]
    if c["kind"] == "decode":
        full = _mixed(c["layout"], B, c["full"], 1, c["ragged"])
        lens = [full[b] if h < c["heads_a"] else min(full[b], c["short"]) for b in range(B) for h in range(H)]
        return [1] * B, lens, lens
    new = _mixed(c["layout"], B, c["tokens"], 1, c["ragged"])
    old = _mixed(c["layout"] + 1, B, c["cached"], 0, c["ragged"])
    before = [old[b] for b in range(B) for _ in range(H)]
    return new, before, [before[b * H + h] + new[b] for b in range(B) for h in range(H)]


def _sections(c):
    pairs = c["rot"] // 2
    return [pairs] if c["axes"] == 1 else [pairs // 4, pairs // 8 * 3, pairs - pairs // 4 - pairs // 8 * 3]


def _elem(c):
    return 1 if c["q8"] else 2


def work(c):
    new, before, after = _geometry(c)
    T, hq = sum(new), c["hkv"] * c["group"]
    D, H = c["dim"], c["hkv"]
    if c["kind"] == "append":
        rows = T * (2 * hq + 2 * H) * D * 2 + 2 * T * H * D * _elem(c)
        return {"bytes": rows + T * c["axes"] * 8, "flops": 6 * T * (hq + H) * c["rot"] // 2}
    cache = 2 * sum(after) * D * _elem(c)
    if c["kind"] == "decode":
        return {"bytes": cache + 2 * T * hq * D * 2, "flops": 4 * D * c["group"] * sum(after)}
    pairs = sum(n * (after[b * H] - n) + n * (n + 1) // 2 for b, n in enumerate(new)) * hq
    return {"bytes": cache + 2 * T * hq * D * 2, "flops": 4 * D * pairs}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _scale_of(amax):
    """The power of two by which a page with this largest magnitude is held: the least 2^e, e >= -64, with amax <= 448 * 2^e."""
    m, e = torch.frexp(amax.clamp_min(1e-30))  # amax = m * 2^e, m in [0.5, 1)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.ldexp(torch.ones_like(amax), e.clamp_min(-64))


def prepare(c, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    B, H, G, D, R = c["batch"], c["hkv"], c["group"], c["dim"], c["page"]
    new, before, after = _geometry(c)
    N, T = B * H, sum(new)
    used = [-(-n // R) for n in after]
    M = max(used) + 1
    P = sum(used) + 3  # a pool has pages that no table names; the last one is among them
    order = torch.randperm(P - 1, generator=g, device=dev, dtype=torch.int32)
    table = torch.full((N, M), -1, dtype=torch.int32, device=dev)
    have = torch.arange(M, device=dev).unsqueeze(0) < torch.tensor(used, device=dev).unsqueeze(1)
    table[have] = order[:sum(used)]

    def pages():
        x = torch.randn(P, R, D, device=dev, generator=g) * torch.empty(P, 1, 1, device=dev).uniform_(0.5, 2.0, generator=g)
        if not c["q8"]:
            return x.to(dt), None
        s = _scale_of(x.abs().amax(dim=(1, 2)))
        return (x / s[:, None, None]).to(E4M3), s

    kp, ks = pages()
    vp, vs = pages()
    s = dict(case=c, k_pages=kp, v_pages=vp, k_scale=ks, v_scale=vs, page_table=table, scale=D ** -0.5, longest=max(after),
             max_tokens=max(new), seg_len=torch.tensor(after, dtype=torch.int32, device=dev),
             cu_tokens=torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=dev))
    if c["kind"] == "decode":
        s["q"] = torch.randn(N, G, D, device=dev, generator=g).to(dt)
        return s
    if c["kind"] == "prompt":
        s["q"] = torch.randn(T, H * G, D, device=dev, generator=g).to(dt)
        return s
    # q, k and v as one projection leaves them: views of [T, (Hq + 2 Hkv) D]
    qkv = torch.randn(T, (G + 2) * H * D, device=dev, generator=g).to(dt)
    s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, D)) for x in qkv.split([H * G * D, H * D, H * D], dim=1))
    s["seg_len"] = torch.tensor(before, dtype=torch.int32, device=dev)
    first = torch.tensor([before[b * H] for b in range(B)], device=dev).repeat_interleave(torch.tensor(new, device=dev))
    at = torch.arange(T, device=dev) - s["cu_tokens"][:-1].long().repeat_interleave(torch.tensor(new, device=dev))
    pos = first + at
    if c["axes"] == 3:  # frames in time, each a small image
        pos = torch.stack([pos, pos // 7 % 40, pos % 7 + 3])
    s["positions"], s["sections"] = pos, _sections(c)
    pairs = c["rot"] // 2
    s["inv_freq"] = 1e6 ** (-torch.arange(pairs, device=dev, dtype=torch.float64) / pairs)
    return s


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------
def _rotated(x, positions, inv_freq, sections, interleaved):
    """Rows [T, heads, D] rotated by their positions, in 32 bits; the angles in 64."""
    axis = torch.repeat_interleave(torch.arange(len(sections), device=x.device), torch.tensor(sections, device=x.device),
                                   output_size=sum(sections))
    at = positions.reshape(len(sections), -1).double()
    angle = at[axis].t() * inv_freq
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    x = x.float()
    r = 2 * inv_freq.numel()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, w], dim=-1).flatten(-2) if interleaved else torch.cat([u, w], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _put(s, rows, pages, scales):
    """Rows [T, Hkv, D] (32 bits) into their places in the pages."""
    c = s["case"]
    B, H, R, D = c["batch"], c["hkv"], c["page"], c["dim"]
    P = pages.shape[0]
    units = (s["max_tokens"] + R - 2) // R + 1  # pages that one segment's new rows can touch
    before = s["seg_len"].long()
    b = torch.arange(B * H, device=rows.device) // H
    n = (s["cu_tokens"][1:] - s["cu_tokens"][:-1]).long()[b]
    block = (before // R).unsqueeze(1) + torch.arange(units, device=rows.device)
    named = block * R < (before + n).unsqueeze(1)
    page = torch.where(named, s["page_table"].long().gather(1, block.clamp_max(s["page_table"].shape[1] - 1)), P - 1)
    at = block.unsqueeze(2) * R + torch.arange(R, device=rows.device)  # [N, units, R] rows of the segment
    token = at - before[:, None, None]
    fresh = named.unsqueeze(2) & (token >= 0) & (token < n[:, None, None])
    there = named.unsqueeze(2) & (token < 0)
    token = (s["cu_tokens"].long()[b][:, None, None] + token).clamp(0, rows.shape[0] - 1)
    head = (torch.arange(B * H, device=rows.device) % H)[:, None, None]
    x = rows[token, head]  # [N, units, R, D]
    if scales is None:
        held = torch.where(fresh.unsqueeze(3), x.to(pages.dtype), pages[page])
    else:
        need = _scale_of(torch.where(fresh.unsqueeze(3), x.abs(), 0.0).amax(dim=(2, 3)))
        was = scales[page]
        now = torch.where(there.any(2), torch.maximum(was, need), need)
        now = torch.where(named, now, was)
        codes = pages.view(torch.uint8)[page]
        moved = codes.view(E4M3).float() * (was / now)[:, :, None, None]
        mine = torch.where(fresh.unsqueeze(3), x / now[:, :, None, None], moved).to(E4M3).view(torch.uint8)
        held = torch.where((fresh | there).unsqueeze(3), mine, codes)
        scales[page] = now
        pages = pages.view(torch.uint8)
    pages[page] = held


def _dense(s, pages, scales):
    """The segments' rows [N, longest, D] in 32 bits; zeros past each length."""
    table = s["page_table"].long()[:, :-(-s["longest"] // pages.shape[1])].clamp_min(0)
    x = (pages if scales is None else pages.view(torch.uint8))[table]
    x = x.float() if scales is None else x.view(E4M3).float() * scales[table][:, :, None, None]
    x = x.flatten(1, 2)[:, :s["longest"]]
    inside = torch.arange(s["longest"], device=x.device) < s["seg_len"].unsqueeze(1)
    return torch.where(inside.unsqueeze(2), x, 0.0)


def _weights(scores, limit):
    """Softmax over the first ``limit`` keys of each row; a row of none: zeros."""
    keys = torch.arange(scores.shape[-1], device=scores.device)
    scores = torch.where(keys < limit.unsqueeze(-1), scores, -torch.inf)
    e = torch.exp(scores - scores.amax(dim=-1, keepdim=True).clamp_min(-1e30))
    return e / e.sum(dim=-1, keepdim=True).clamp_min(1e-37)


def run(s):
    c = s["case"]
    cache = (s["k_pages"], s["v_pages"], s["page_table"], s["seg_len"])
    if own:
        from wnw_amd.kv.paged import paged_append, paged_decode_attn, paged_prompt_attn

        if c["kind"] == "append":
            q, new_len = paged_append(s["k"], s["v"], *cache, q=s["q"], positions=s["positions"], inv_freq=s["inv_freq"],
                                      sections=s["sections"], interleaved=c["interleaved"], cu_tokens=s["cu_tokens"],
                                      max_tokens=s["max_tokens"], k_scale=s["k_scale"], v_scale=s["v_scale"])
            return _appended(s, q, new_len)
        if c["kind"] == "decode":
            return paged_decode_attn(s["q"], *cache, s["scale"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return paged_prompt_attn(s["q"], *cache, s["cu_tokens"], s["scale"], max_tokens=s["max_tokens"],
                                 k_scale=s["k_scale"], v_scale=s["v_scale"])
    B, H, G, D = c["batch"], c["hkv"], c["group"], c["dim"]
    if c["kind"] == "append":
        turn = (s["positions"], s["inv_freq"], s["sections"], c["interleaved"])
        _put(s, _rotated(s["k"], *turn), s["k_pages"], s["k_scale"])
        _put(s, s["v"].float(), s["v_pages"], s["v_scale"])
        n = s["cu_tokens"][1:] - s["cu_tokens"][:-1]
        new_len = s["seg_len"] + torch.repeat_interleave(n, H, output_size=B * H)
        return _appended(s, _rotated(s["q"], *turn).to(s["q"].dtype), new_len)
    k, v = _dense(s, s["k_pages"], s["k_scale"]), _dense(s, s["v_pages"], s["v_scale"])
    if c["kind"] == "decode":
        scores = torch.matmul(s["q"].float(), k.transpose(1, 2)) * s["scale"]
        return torch.matmul(_weights(scores, s["seg_len"].unsqueeze(1)), v).to(s["q"].dtype)
    # the samples' tokens beside each other, padded to the longest
    cu, width = s["cu_tokens"].long(), s["max_tokens"]
    n = cu[1:] - cu[:-1]
    token = (cu[:-1].unsqueeze(1) + torch.arange(width, device=cu.device)).clamp_max(s["q"].shape[0] - 1)
    q = s["q"].float()[token].view(B, width, H, G, D).permute(0, 2, 3, 1, 4).reshape(B * H, G * width, D)
    reach = s["seg_len"].long() - n.repeat_interleave(H, output_size=B * H)
    limit = (reach.unsqueeze(1) + torch.arange(width, device=cu.device) + 1).repeat(1, G)
    o = torch.matmul(_weights(torch.matmul(q, k.transpose(1, 2)) * s["scale"], limit), v)
    o = o.view(B, H, G, width, D).permute(0, 3, 1, 2, 4).reshape(B, width, H * G, D).to(s["q"].dtype)
    sample = torch.repeat_interleave(torch.arange(B, device=cu.device), n, output_size=s["q"].shape[0])
    return o[sample, torch.arange(s["q"].shape[0], device=cu.device) - cu[sample]]


def _appended(s, q, new_len):
    out = {"q": q, "len": new_len, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    return out if s["k_scale"] is None else {**out, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


# --------------------------------------------------------------------------
# 64 bits
# --------------------------------------------------------------------------
def _rows_of(s, seg, pages, scales):
    n = int(s["seg_len"][seg])
    R = pages.shape[1]
    ids = s["page_table"][seg, :-(-n // R)].long()
    x = pages.view(torch.uint8)[ids].view(E4M3).double() * scales[ids].double()[:, None, None] if scales is not None \
        else pages[ids].double()
    return x.reshape(-1, pages.shape[2])[:n]


def exact(c, seed):
    s = prepare(c, seed)
    new, before, after = _geometry(c)
    B, H, G, D, R = c["batch"], c["hkv"], c["group"], c["dim"], c["page"]
    if c["kind"] != "append":
        q = s["q"].double()
        out = torch.zeros_like(q)
        start = 0
        for b in range(B):
            for h in range(H):
                seg = b * H + h
                k, v = _rows_of(s, seg, s["k_pages"], s["k_scale"]), _rows_of(s, seg, s["v_pages"], s["v_scale"])
                if c["kind"] == "decode":
                    out[seg] = torch.softmax(q[seg] @ k.t().contiguous() * s["scale"], dim=-1) @ v
                    continue
                last = after[seg] - new[b] + torch.arange(new[b], device=q.device)
                later = torch.arange(after[seg], device=q.device) > last.unsqueeze(1)
                for head in range(h * G, (h + 1) * G):
                    p = q[start:start + new[b], head] @ k.t().contiguous() * s["scale"]
                    out[start:start + new[b], head] = torch.softmax(p.masked_fill_(later, -torch.inf), dim=-1) @ v
            start += new[b]
        return out

    pairs = c["rot"] // 2
    pos = s["positions"].double().reshape(len(s["sections"]), -1)

    def turned(x):
        x = x.double().clone()
        j = 0
        for a, size in enumerate(s["sections"]):
            for _ in range(size):
                lo, hi = (2 * j, 2 * j + 1) if c["interleaved"] else (j, j + pairs)
                z = torch.complex(x[..., lo], x[..., hi]) * torch.polar(torch.ones_like(pos[a]),
                                                                       pos[a] * s["inv_freq"][j]).unsqueeze(1)
                x[..., lo], x[..., hi] = z.real, z.imag
                j += 1
        return x

    def filled(rows, pages, scales):
        """Pages (in units of their scales, not rounded) and scales after the append."""
        pages, scales = pages.double(), None if scales is None else scales.double().clone()
        table = s["page_table"].tolist()
        firsts = [sum(new[:b]) for b in range(B)]
        for seg in range(B * H):
            b, h = divmod(seg, H)
            at = before[seg]
            while at < after[seg]:
                page, row = table[seg][at // R], at % R
                stop = min(after[seg], at - row + R)
                x = rows[firsts[b] + at - before[seg]:firsts[b] + stop - before[seg], h]
                if scales is not None:
                    big = float(x.abs().max())
                    fit = 2.0 ** max(-64, math.ceil(math.log2(big / 448.0))) if big > 0 else 2.0 ** -64
                    if row:
                        was = float(scales[page])
                        fit = max(fit, was)
                        pages[page, :row] *= was / fit
                    scales[page] = fit
                    x = x / fit
                pages[page, row:row + stop - at] = x
                at = stop
        return pages, scales

    if sum(-(-n // R) + 1 for n in new) * H > 8000:  # a page at a time takes too long
        return None
    kp, ks = filled(turned(s["k"]), s["k_pages"], s["k_scale"])
    vp, vs = filled(s["v"].double(), s["v_pages"], s["v_scale"])
    out = {"q": turned(s["q"]), "len": None, "k_pages": kp, "v_pages": vp}
    return out if ks is None else {**out, "k_scale": ks, "v_scale": vs}
