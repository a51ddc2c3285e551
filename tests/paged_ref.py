"""Plain 64-bit forms of the paged cache's operators, and caches to try them on.

``make_cache`` lays segments out over shuffled pages; rows past a segment's
length hold NaN, table entries past its pages hold numbers that are no page.
"""
from __future__ import annotations

import torch

E4M3 = torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def scale_of(amax):
    """Least 2^e, e >= -64, with amax <= 448 * 2^e (amax a float64 tensor)."""
    m, e = torch.frexp(amax.double())
    e = torch.where(m <= 0.875, e - 9, e - 8)
    power = ((e.clamp_min(-64).long() + 1023) << 52).view(torch.float64)  # torch.ldexp is off by a rounding
    return torch.where(amax > 0, power, 2.0 ** -64)


class Cache:
    def __init__(self, dev, lens, page, D, dtype, q8, seed=0, spare=3, joined=False, room=1, scales="pow2", values=None):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.dev, self.page, self.D, self.q8, self.dtype = dev, page, D, q8, dtype
        self.lens = list(lens)
        N = len(self.lens)
        used = [-(-n // page) + (room if room > 1 else 0) for n in self.lens]
        P = max(sum(used) + spare, 1)
        M = max([-(-n // page) for n in self.lens] + [0]) + max(room, 1)
        order = torch.randperm(P, generator=g, device=dev).int()
        table = torch.full((N, M + 1), 0x7fffffff, dtype=torch.int32, device=dev)[:, :M]  # rows M + 1 apart
        table[:, 1::2] = -7
        at = 0
        for s, n in enumerate(used):
            table[s, :n] = order[at:at + n]
            at += n
        self.table, self.P, self.M = table, P, M
        self.seg_len = torch.tensor(self.lens, dtype=torch.int32, device=dev)
        both = torch.randn(P, 2, page, D, device=dev, generator=g, dtype=torch.float32)
        both *= torch.empty(P, 2, 1, 1, device=dev).uniform_(0.5, 2.0, generator=g)
        if values is not None:
            both = values(both)
        self.k_scale = self.v_scale = None
        if q8:
            s = scale_of(both.abs().amax(dim=(2, 3))).float()
            if scales == "any":
                s = s * torch.empty(P, 2, device=dev).uniform_(0.3, 3.0, generator=g) ** 3
                codes = (both / both.abs().amax(dim=(2, 3), keepdim=True) * 448).to(E4M3)
            else:
                codes = (both / s[:, :, None, None]).to(E4M3)
            self.k_scale, self.v_scale = s[:, 0].contiguous(), s[:, 1].contiguous()
            both = codes.view(torch.uint8)
        else:
            both = both.to(dtype)
        keep = torch.zeros(P, page, dtype=torch.bool, device=dev)
        for s, n in enumerate(self.lens):
            for i in range(-(-n // page)):
                keep[table[s, i].item(), :min(page, n - i * page)] = True
        junk = 0x7f if q8 else float("nan")
        both = torch.where(keep[:, None, :, None], both, torch.full_like(both, junk))
        if q8:
            both = both.view(E4M3)
        if joined:
            self.k, self.v = both[:, 0], both[:, 1]
        else:
            self.k, self.v = both[:, 0].contiguous(), both[:, 1].contiguous()

    def args(self):
        return self.k, self.v, self.table, self.seg_len

    def scales(self):
        return dict(k_scale=self.k_scale, v_scale=self.v_scale)

    def rows(self, s, n=None):
        """K and V rows of segment s in 64 bits."""
        n = self.lens[s] if n is None else n
        ids = self.table[s, :-(-n // self.page)].long()
        out = []
        for pages, sc in ((self.k, self.k_scale), (self.v, self.v_scale)):
            x = pages.contiguous().view(torch.uint8)[ids].view(E4M3).double() * sc[ids].double()[:, None, None] \
                if self.q8 else pages[ids].double()
            out.append(x.reshape(-1, self.D)[:n])
        return out


def attend(q, k, v, limit, scale):
    """q [R, D] (64 bits) against the first limit[r] of k's rows each: the result and sum |w v|."""
    s = (q @ k.t().contiguous()) * scale
    seen = torch.arange(k.shape[0], device=q.device) < limit.unsqueeze(1)
    s = s.masked_fill(~seen, float("-inf"))
    e = torch.where(seen, torch.exp(s - s.amax(1, keepdim=True).clamp_min(-1e300)), 0.0) if k.shape[0] else s
    w = e / e.sum(1, keepdim=True).clamp_min(1e-300)
    return w @ v, w @ v.abs()


def rotate(x, positions, inv_freq, sections, interleaved):
    """[T, H, D] in 64 bits, and |a| + |b| of each element's pair."""
    x = x.double()
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=x.device)
    ang = positions.reshape(len(sections), -1).double()[axis].t() * inv_freq.double()
    cos, sin = ang.cos().unsqueeze(1), ang.sin().unsqueeze(1)
    r = 2 * inv_freq.numel()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    u, w, size = a * cos - b * sin, b * cos + a * sin, a.abs() + b.abs()
    def join(y, z):
        return torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)
    return torch.cat([join(u, w), x[..., r:]], -1), torch.cat([join(size, size), x[..., r:].abs()], -1)
