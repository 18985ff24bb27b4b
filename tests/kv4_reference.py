"""Plain 64-bit forms of the paged 4-bit cache, from its definition (torch, any device)."""
import math

import torch


def make_cache(gen, B, lengths, hkv, hd, page, device="cuda", spread=1.0, zero_scale=False, extra_pages=3):
    """Pages in random order with random codes, finite scales and zeros where a token is, and bytes of 0xFF (NaN as scales)
    everywhere else.  -> pages uint8 [n, hkv, page * (hd + 8)], table int32 [B, width] (-1: none), k, v [B][hkv, L, hd] fp64."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + extra_pages
    order = torch.randperm(total, generator=gen).tolist()
    width = max(1, max(need, default=1))
    table = torch.full((B, width), -1, dtype=torch.int32)
    pages = torch.full((total, hkv, page * (hd + 8)), 255, dtype=torch.uint8)
    ks, vs, used = [], [], 0
    for b, n in enumerate(lengths):
        ids = order[used : used + need[b]]
        used += need[b]
        table[b, : need[b]] = torch.tensor(ids, dtype=torch.int32)
        both = []
        for kv in range(2):
            c = torch.randint(0, 16, (n, hkv, hd), generator=gen, dtype=torch.uint8)
            s = (torch.rand(n, hkv, 1, generator=gen) * 0.4 + 0.05) * spread
            if zero_scale:
                s = s * (torch.rand(n, hkv, 1, generator=gen) > 0.3)
            z = (-7.5 * s + torch.randn(n, hkv, 1, generator=gen) * 0.3 * spread).half()
            s = s.half()
            pos = torch.arange(n)
            page_of = torch.tensor(ids, dtype=torch.long)[pos // page] if n else pos
            slot = pos % page
            lo = kv * page * hd // 2
            view = pages[:, :, lo : lo + page * hd // 2].view(total, hkv, page, hd // 2)
            view[page_of, :, slot] = c[..., 0::2] | (c[..., 1::2] << 4)
            lo = page * hd + kv * 4 * page
            view = pages[:, :, lo : lo + 4 * page].view(total, hkv, page, 4)
            view[page_of, :, slot] = torch.cat([s, z], -1).contiguous().view(torch.uint8)
            both.append((c.double() * s.double() + z.double()).transpose(0, 1))
        ks.append(both[0].to(device))
        vs.append(both[1].to(device))
    return pages.to(device), table.to(device), ks, vs


def attention(q, ks, vs, new, lengths, window=0, sinks=0, scale=None, missing=None):
    """q [T, hq, hd]; ks / vs: per sequence [hkv, L, hd] fp64 of all tokens.  missing: (b, token) -> True where the page is not
    there.  -> [T, hq, hd] fp64"""
    T, hq, hd = q.shape
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(T, hq, hd, dtype=torch.float64, device=q.device)
    first = 0
    for b, (n, m) in enumerate(zip(new, lengths)):
        k, v = ks[b], vs[b]
        hkv, L = k.shape[0], min(k.shape[1], max(m, 0))
        if n and L:
            j = torch.arange(L, device=q.device)
            gone = torch.tensor([missing is not None and missing(b, t) for t in range(L)], device=q.device)
            for at in range(0, n, 256):
                p = (m - n + torch.arange(at, min(n, at + 256), device=q.device))[:, None]
                see = (j <= p) & ~gone
                if window:
                    see &= (j > p - window) | (j < sinks)
                x = q[first + at : first + at + len(p)].double().view(len(p), hkv, hq // hkv, hd)
                w = torch.einsum("ihgd,hjd->hgij", x, k[:, :L]) * scale
                w = torch.softmax(w.masked_fill(~see, -math.inf), dim=-1)
                w = torch.where(see.any(-1)[:, None], w, torch.zeros_like(w))
                out[first + at : first + at + len(p)] = torch.einsum("hgij,hjd->ihgd", w, v[:, :L]).reshape(len(p), hq, hd)
        first += n
    return out


def attention_tolerance(ref, vs, lengths):
    """bf16 result: half a step, 2^-8 of the value; the weights of the second product are fp16 (2^-11 of the weight, in the worst
    case all of one sign, against codes that span 15 steps, or 2^-25 of the largest weight for the smallest ones), scores in
    fp32 (|score| below 64 here: 64 * 2^-20 relative in a weight): on top of the largest span of a token's values."""
    span = max([float((v.amax(-1) - v.amin(-1)).max()) for v in vs if v.numel()] + [0.0])
    n = max(list(lengths) + [1])
    return 2.0 ** -8 * ref.abs() + span * (2.0 ** -11 + n * 2.0 ** -25 + 2.0 ** -14) + 1e-6


def quantise(x):
    """fp64 head values -> (codes, scale, zero) as the append stores them: the grid from fp32 arithmetic on fp32 values."""
    x = torch.where(x.isnan(), torch.zeros_like(x), x).clamp(-65504.0, 65504.0)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s, z = ((hi - lo) * (1.0 / 15.0)).half(), lo.half()
    # a grid that passes what fp16 holds (15 s + z rounds to infinity from 65520 on): one step of fp16 less
    s = torch.where(15 * s.double() + z.double() >= 65520, (s.view(torch.int16) - 1).view(torch.float16), s)
    inv = torch.where(s > 0, 1.0 / s.float(), torch.zeros_like(lo))
    return ((x - z.float()) * inv).round().clamp(0, 15), s, z


def rotate_positions(x, cos, sin):
    """fp32, each operation rounded on its own: x [T, heads, d], cos / sin [T, d / 2]"""
    d = x.shape[-1] // 2
    c, s = cos[:, None], sin[:, None]
    return torch.cat([x[..., :d] * c - x[..., d:] * s, x[..., d:] * c + x[..., :d] * s], -1)


def walsh_hadamard(x):
    """Butterflies h = 1, 2, 4 ... and the factor d ** -0.5, in x's type."""
    h, d = 1, x.shape[-1]
    while h < d:
        y = x.reshape(*x.shape[:-1], d // (2 * h), 2, h)
        x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], -2).reshape(x.shape)
        h *= 2
    return x * (1.0 / math.sqrt(d))


def unpack(pages, table, lengths, hkv, hd, page):
    """Codes and (scale, zero) of every token: per sequence (kc [n, hkv, hd], kp [n, hkv, 2], vc, vp)"""
    got = []
    for b, n in enumerate(lengths):
        pos = torch.arange(n, device=pages.device)
        pg, slot = table[b].long()[pos // page], pos % page
        item = []
        for kv in range(2):
            lo = kv * page * hd // 2
            raw = pages[:, :, lo : lo + page * hd // 2].reshape(-1, hkv, page, hd // 2)[pg, :, slot]
            item.append(torch.stack([raw & 15, raw >> 4], -1).reshape(n, hkv, hd))
            lo = page * hd + kv * 4 * page
            item.append(pages[:, :, lo : lo + 4 * page].reshape(-1, hkv, page, 4)[pg, :, slot].contiguous().view(torch.float16))
        got.append(item)
    return got
