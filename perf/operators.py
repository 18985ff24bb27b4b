"""Cases of the paged 4-bit key/value cache: appending to it, attention over it, reading it back.

The operators (`own`):
  ops.kv4_append     position rotation and optional Walsh-Hadamard rotation of queries and keys, 4-bit quantisation of keys and
                     values per (token, head), write into the pages; returns the rotated queries
  ops.kv4_attention  causal grouped-query attention of each sequence's new tokens over its pages, with an optional sliding
                     window and first tokens that stay visible
  ops.kv4_read       the values that the cache stands for, as bf16 rows

A page holds P tokens.  Its block for one key/value head is P * (d + 8) bytes: key codes [P][d / 2] (element 2i in the low half
of byte i), value codes [P][d / 2], key (scale, zero) pairs [P][2] in fp16, value pairs [P][2].  A code c stands for
scale * c + zero.

The plain forms compute in 32 bits with elementary tensor operations; `exact` goes by the definitions, in 64.
"""
import functools
import math
import random

import torch

own = False

# (query heads, key/value heads, head size): the decoder configuration, its shards under tensor parallelism, the tests'
# small decoder, and generic layouts around them
_HEADS = ((32, 8, 128), (16, 4, 128), (8, 2, 64), (28, 4, 128), (32, 32, 64), (16, 2, 64), (8, 8, 128))
_MOST_TOKENS = 1 << 20   # tokens in the cache of the largest case
_MOST_PAIRS = 1.1e9      # query x key x head products of the largest case, masked ones among them


def _case(name, op, batch, ctx, new, heads=(32, 8, 128), page=64, ragged=True, window=0, sinks=0, rotate=True):
    hq, hkv, hd = heads
    return {"name": name, "op": op, "batch": batch, "ctx": ctx, "new": new, "hq": hq, "hkv": hkv, "hd": hd, "page": page,
            "ragged": ragged, "window": window, "sinks": sinks, "rotate": rotate}


def listed():
    return [
        # one new token for each of eight sequences: the cache write of a decode step
        _case("append 8 tokens", "append", 8, 2048, 1),
        # the prompts of eight sequences at once, odd lengths
        _case("append prompts 8 x 2048", "append", 8, 2048, 2048),
        # small heads without the rotation of keys, pages of 16, a mixture of short prompts behind a shared prefix
        _case("append 24 x 300 d64", "append", 24, 1500, 300, heads=(8, 2, 64), page=16, rotate=False),
        # the smallest attention: one token of one sequence over a short cache
        _case("attend 1 x 300", "attend", 1, 300, 1, ragged=False),
        # one long conversation
        _case("attend 1 x 100000", "attend", 1, 100003, 1, ragged=False, page=32),
        # an ordinary decode batch with ragged lengths and small pages
        _case("attend 16 ragged 8000", "attend", 16, 8000, 1, page=16),
        # the largest decode batch: one million tokens in the cache
        _case("attend 64 x 16384", "attend", 64, 16384, 1, ragged=False),
        # streaming: a window of 4096 tokens and four first tokens over long sequences, a shard of heads
        _case("attend 32 window 4096", "attend", 32, 30000, 1, heads=(16, 4, 128), window=4096, sinks=4),
        # four tokens of a sequence at once (verification of drafted tokens), small heads in large groups
        _case("attend 24 x 4 drafts d64", "attend", 24, 6000, 4, heads=(16, 2, 64)),
        # the prompts of eight sequences
        _case("attend prompts 8 x 2048", "attend", 8, 2048, 2048, ragged=False),
        # the next piece of long prompts, over what the cache holds already, with a window
        _case("attend pieces 4 x 512", "attend", 4, 16000, 512, window=6000, sinks=64),
        # the cache of a batch handed to something that wants 16-bit rows
        _case("read 16 x 4096", "read", 16, 4096, 4096, page=128),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    heads = rng.choice(_HEADS)
    op = rng.choice(("append", "attend", "attend", "attend pieces", "read"))
    batch = spread(1, 64)
    page = rng.choice((16, 32, 64, 128, 256))
    ctx = spread(1, min(131072, _MOST_TOKENS * 8 // heads[1] // batch))
    if op == "attend":
        new = min(ctx, rng.choice((1, 1, 1, 2, 3, 4, 8)))
    else:
        new = min(ctx, spread(1, 4096))
    if op.startswith("attend"):
        while batch * new * ctx * heads[0] > _MOST_PAIRS or batch * ctx * heads[1] * heads[2] > 1.1e9:
            batch, ctx, new = max(1, batch // 2), max(1, ctx * 3 // 4), max(1, min(new * 3 // 4, ctx * 3 // 4))
    else:
        new = max(1, min(new, 32768 // batch))
        ctx = min(ctx, max(new, 65536 // batch))
    window, sinks = (spread(1, 8192), rng.choice((0, 1, 4, 64, 200))) if rng.random() < 0.4 else (0, 0)
    if not op.startswith("attend"):
        window, sinks = 0, 0
    c = _case("", op.split()[0], batch, ctx, new, heads, page, rng.random() < 0.8, window, sinks, rng.random() < 0.7)
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, length with them) of every sequence: part of the case, alike for every seed.  Ragged batches of eight or
    more hold one sequence without tokens; new tokens are uneven where a sequence brings more than eight."""
    r = random.Random(case["batch"] * 7919 + case["ctx"] * 31 + case["new"])
    new, length = [], []
    for b in range(case["batch"]):
        n, m = case["new"], case["ctx"]
        if case["ragged"]:
            n = max(1, int(n * r.uniform(0.3, 1.0))) if n > 8 else n
            m = max(n, int(m * r.uniform(0.2, 1.0)))
            if case["batch"] >= 8 and b == 5:
                n = m = 0
        new.append(n)
        length.append(m)
    if case["ragged"]:
        length[0] = max(new[0], case["ctx"])
    return new, length


# ------------------------------------------------------------------------------------------- what a program holds
def _pack_pages(pages, hd, P, page, slot, kc, kp, vc, vp):
    """Codes [T, hkv, d] (uint8) and (scale, zero) fp16 [T, hkv, 2] of T tokens into their page slots."""
    n, h = pages.shape[:2]
    pages[:, :, : P * hd // 2].view(n, h, P, hd // 2)[page, :, slot] = kc[..., 0::2] | kc[..., 1::2] << 4
    pages[:, :, P * hd // 2 : P * hd].view(n, h, P, hd // 2)[page, :, slot] = vc[..., 0::2] | vc[..., 1::2] << 4
    pages[:, :, P * hd : P * hd + 4 * P].view(n, h, P, 4)[page, :, slot] = kp.view(torch.uint8)
    pages[:, :, P * hd + 4 * P :].view(n, h, P, 4)[page, :, slot] = vp.view(torch.uint8)


def _random_codes(shape, gen, outliers):
    """Quantised heads of normal values, some channels of them four times larger where `outliers`."""
    x = torch.randn(shape, generator=gen, device="cuda")
    if outliers:
        x[..., ::17] *= 4.0
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s, z = ((hi - lo) / 15).half(), lo.half()
    c = ((x - z.float()) / s.float()).round_().clamp_(0, 15).to(torch.uint8)
    return c, torch.cat([s, z], dim=-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hq, hkv, hd, P, B = case["hq"], case["hkv"], case["hd"], case["page"], case["batch"]
    new, length = _lengths(case)
    T = sum(new)
    # pages in random order, as an allocator leaves them after a while
    need = [-(-n // P) for n in length]
    width = max(1, max(need))
    ids = torch.randperm(sum(need) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    first = 0
    for b in range(B):
        table[b, : need[b]] = ids[first : first + need[b]]
        first += need[b]
    # slots that hold no token hold anything
    pages = torch.randint(0, 256, (sum(need) + 3, hkv, P * (hd + 8)), dtype=torch.uint8, generator=g, device="cuda")
    held = [m if case["op"] != "append" else m - n for n, m in zip(new, length)]
    step = max(1, (1 << 28) // (hkv * hd))
    for b in range(B):
        for lo in range(0, held[b], step):
            pos = torch.arange(lo, min(lo + step, held[b]), device="cuda")
            kc, kp = _random_codes((len(pos), hkv, hd), g, not case["rotate"])
            vc, vp = _random_codes((len(pos), hkv, hd), g, False)
            _pack_pages(pages, hd, P, table[b, pos // P].long(), pos % P, kc, kp, vc, vp)
    cu = torch.tensor([0] + [sum(new[: b + 1]) for b in range(B)], dtype=torch.int32, device="cuda")
    st = {"case": case, "pages": pages, "table": table, "cu": cu, "new": max(new), "tokens": T, "longest": max(length),
          "kv_len": torch.tensor(length, dtype=torch.int32, device="cuda")}
    n_new = torch.tensor(new, device="cuda")
    st["row_b"] = torch.repeat_interleave(torch.arange(B, device="cuda"), n_new)
    st["row_i"] = torch.arange(T, device="cuda") - cu[:-1].long()[st["row_b"]]
    st["n_new"] = n_new
    if case["op"] == "append":
        st["qkv"] = torch.randn(T, (hq + 2 * hkv) * hd, generator=g, device="cuda")
        st["qkv"][:, ::37] *= 4.0
        st["qkv"] = st["qkv"].to(torch.bfloat16)
        n = max(length)
        ang = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * (
            1.0 / 500000.0 ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd))[None, :]
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
    elif case["op"] == "attend":
        st["q"] = (1.5 * torch.randn(T, hq, hd, generator=g, device="cuda")).to(torch.bfloat16)
    return st


# ------------------------------------------------------------------------------------------- plain forms
def _unpack(block, P, hd):
    """Page blocks [..., P * (d + 8)] -> keys and values [..., P, d] in fp32."""
    lead = block.shape[:-1]

    def part(lo, hi, p):
        c = block[..., lo:hi].reshape(*lead, P, hd // 2)
        c = torch.stack([c & 15, c >> 4], dim=-1).reshape(*lead, P, hd).float()
        sz = block[..., p : p + 4 * P].contiguous().view(torch.float16).reshape(*lead, P, 2).float()
        return c * sz[..., :1] + sz[..., 1:]

    return part(0, P * hd // 2, P * hd), part(P * hd // 2, P * hd, P * hd + 4 * P)


def _rows(st, page, slot):
    """Keys and values of single tokens, bf16 [T, hkv, d]."""
    c = st["case"]
    P, hd = c["page"], c["hd"]

    def part(lo, hi, p):
        pg = st["pages"]
        n, h = pg.shape[:2]
        code = pg[:, :, lo:hi].view(n, h, P, hd // 2)[page, :, slot]
        code = torch.stack([code & 15, code >> 4], dim=-1).reshape(-1, h, hd).float()
        sz = pg[:, :, p : p + 4 * P].view(n, h, P, 4)[page, :, slot].view(torch.float16).float()
        return (code * sz[..., :1] + sz[..., 1:]).to(torch.bfloat16)

    return part(0, P * hd // 2, P * hd), part(P * hd // 2, P * hd, P * hd + 4 * P)


def _butterfly(x, h):
    y = x.reshape(*x.shape[:-1], -1, 2, h)
    return torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], dim=-2).reshape(x.shape)


def _quantise(x):
    x = torch.where(x.isnan(), torch.zeros_like(x), x).clamp(-65504.0, 65504.0)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s, z = ((hi - lo) * (1.0 / 15.0)).half(), lo.half()
    inv = torch.where(s > 0, 1.0 / s.float(), torch.zeros_like(lo))
    return ((x - z.float()) * inv).round().clamp(0, 15).to(torch.uint8), torch.cat([s, z], dim=-1)


def _place(st):
    """Position, page and slot of every new token."""
    pos = st["kv_len"].long()[st["row_b"]] - st["n_new"][st["row_b"]] + st["row_i"]
    P = st["case"]["page"]
    return pos, st["table"][st["row_b"], pos // P].long(), pos % P


def _plain_append(st):
    c = st["case"]
    hq, hkv, hd = c["hq"], c["hkv"], c["hd"]
    pos, page, slot = _place(st)
    x = st["qkv"].float().view(-1, hq + 2 * hkv, hd)
    x1, x2 = x[:, : hq + hkv, : hd // 2], x[:, : hq + hkv, hd // 2 :]
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    r = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1)
    if c["rotate"]:
        r = functools.reduce(_butterfly, [1 << i for i in range(hd.bit_length() - 1)], r) * hd ** -0.5
    kc, kp = _quantise(r[:, hq:])
    vc, vp = _quantise(x[:, hq + hkv :])
    _pack_pages(st["pages"], hd, c["page"], page, slot, kc, kp, vc, vp)
    return [r[:, :hq].to(torch.bfloat16), *_rows(st, page, slot)]


def _plain_attend(st):
    c = st["case"]
    hq, hkv, hd, P, B = c["hq"], c["hkv"], c["hd"], c["page"], c["batch"]
    G, Q, L = hq // hkv, st["new"], st["longest"]
    k, v = _unpack(st["pages"][st["table"].clamp(min=0).long()], P, hd)            # [B, pages, hkv, P, d]
    k = k.transpose(2, 3).reshape(B, -1, hkv, hd)[:, :L].permute(0, 2, 1, 3)         # [B, hkv, L, d]
    v = v.transpose(2, 3).reshape(B, -1, hkv, hd)[:, :L].permute(0, 2, 1, 3)
    j = torch.arange(L, device="cuda")
    there = (j[None, :] < st["kv_len"][:, None])[:, None, :, None]
    k = torch.where(there, k, torch.zeros_like(k))
    v = torch.where(there, v, torch.zeros_like(v))
    q = torch.zeros(B, Q, hq, hd, device="cuda")
    q[st["row_b"], st["row_i"]] = st["q"].float()
    q = q.view(B, Q, hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * Q, hd)
    s = torch.matmul(q, k.transpose(2, 3)) * hd ** -0.5                              # [B, hkv, G * Q, L]
    p = (st["kv_len"].long() - st["n_new"])[:, None] + torch.arange(Q, device="cuda")
    see = j <= p[..., None]
    if c["window"]:
        see = see & ((j > p[..., None] - c["window"]) | (j < c["sinks"]))
    s = s.view(B, hkv, G, Q, L).masked_fill_(~see[:, None, None], -math.inf).view(B, hkv, G * Q, L)
    m = s.amax(-1, keepdim=True).clamp(min=-3e38)
    e = s.sub_(m).exp_()
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True).clamp(min=1e-37)
    o = o.view(B, hkv, G, Q, hd).permute(0, 3, 1, 2, 4).reshape(B, Q, hq, hd)
    return o[st["row_b"], st["row_i"]].to(torch.bfloat16)


def _plain_read(st):
    _, page, slot = _place(st)
    return list(_rows(st, page, slot))


# ------------------------------------------------------------------------------------------- the framework's calls
def _own(st):
    from dualquant_b200 import ops

    c = st["case"]
    cache = ops.KV4Cache(st["pages"], c["hd"], c["page"])
    if c["op"] == "append":
        q = ops.kv4_append(st["qkv"], st["cos"], st["sin"], cache, st["table"], st["kv_len"], c["hq"], cu_new=st["cu"],
                           rotate=c["rotate"])
        return [q, *ops.kv4_read(cache, st["table"], st["kv_len"], st["tokens"], cu_new=st["cu"])]
    if c["op"] == "read":
        return list(ops.kv4_read(cache, st["table"], st["kv_len"], st["tokens"], cu_new=st["cu"]))
    return ops.kv4_attention(st["q"], cache, st["table"], st["kv_len"], cu_new=st["cu"], max_new=st["new"],
                             window=c["window"], sinks=c["sinks"])


def run(st):
    if own:
        return _own(st)
    return {"append": _plain_append, "attend": _plain_attend, "read": _plain_read}[st["case"]["op"]](st)


def work(case):
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    new, length = _lengths(case)
    T, row = sum(new), hkv * (hd + 8)
    tables = 4 * sum(-(-m // case["page"]) for m in length)
    if case["op"] == "append":
        # queries, keys, values and angles in; queries out, the cache written and its values out
        return {"bytes": 2 * T * (hq + 2 * hkv) * hd + 4 * T * hd + 2 * T * hq * hd + T * row + 4 * T * hkv * hd,
                "flops": T * (hq + hkv) * hd * (3 + (hd.bit_length() if case["rotate"] else 0)) + 6 * T * hkv * hd}
    if case["op"] == "read":
        return {"bytes": T * row + 4 * T * hkv * hd + tables, "flops": 4 * T * hkv * hd}
    seen = pairs = 0
    W, S = case["window"], case["sinks"]
    for n, m in zip(new, length):
        if not n:
            continue
        if not W:
            seen += m
            pairs += n * m - n * (n - 1) // 2
            continue
        lo = max(0, m - n - W + 1)                       # first token that the first row's window holds
        seen += m - lo + min(S, lo)
        for p in range(m - n, m):
            start = max(0, p - W + 1)
            pairs += p + 1 - start + min(S, start)
    return {"bytes": seen * row + 4 * T * hq * hd + tables, "flops": 4 * pairs * hq * hd}


# ------------------------------------------------------------------------------------------- 64 bits
def _exact_token(st, b, lo, hi):
    """Keys and values of positions lo .. hi - 1 of sequence b, by the definition of a page, in 64 bits [hkv, n, d]."""
    c = st["case"]
    P, hd = c["page"], c["hd"]
    pos = torch.arange(lo, hi, device="cuda")
    block = st["pages"].view(st["pages"].shape[0], c["hkv"], -1)
    page, slot = st["table"][b].long()[torch.div(pos, P, rounding_mode="floor")], pos.remainder(P)
    byte = torch.arange(hd // 2, device="cuda")

    def heads(codes, params):
        at = codes + slot[:, None] * (hd // 2) + byte                                 # [n, d / 2]
        raw = block.transpose(0, 1)[:, page[:, None], at]                             # [hkv, n, d / 2]
        val = torch.empty(*raw.shape[:2], hd, dtype=torch.float64, device="cuda")
        val[..., 0::2], val[..., 1::2] = raw.remainder(16).double(), torch.div(raw, 16, rounding_mode="floor").double()
        word = block.transpose(0, 1)[:, page[:, None], params + slot[:, None] * 4 + torch.arange(4, device="cuda")]
        pair = word.contiguous().view(torch.float16).double()
        return val * pair[..., 0:1] + pair[..., 1:2]

    return heads(0, P * hd), heads(P * hd // 2, P * hd + 4 * P)


def _exact_heads(x):
    """What a 4-bit head stands for: scale and zero as fp16 numbers, codes nearest to the value."""
    x = x.nan_to_num(nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504.0, 65504.0)
    low = x.min(dim=-1).values
    step = ((x.max(dim=-1).values - low) / 15).to(torch.float16).double()
    zero = low.to(torch.float16).double()
    code = torch.where(step[..., None] > 0, (x - zero[..., None]) / step[..., None].clamp(min=2.0 ** -30), 0.0)
    return torch.round(code).clamp(0, 15) * step[..., None] + zero[..., None]


def exact(case, seed):
    st = prepare(case, seed)
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    new, length = _lengths(case)
    first = 0
    out = []
    if case["op"] == "append":
        if case["rotate"]:
            mat = torch.ones(1, 1, dtype=torch.float64, device="cuda")
            while mat.shape[0] < hd:
                mat = torch.cat([torch.cat([mat, mat], 1), torch.cat([mat, -mat], 1)], 0)
            mat = mat / math.sqrt(hd)
        parts = [[], [], []]
        for n, m in zip(new, length):
            x = st["qkv"][first : first + n].double().view(n, hq + 2 * hkv, hd)
            turn = torch.complex(st["cos"][m - n : m].double(), st["sin"][m - n : m].double())[:, None]
            z = torch.complex(x[:, : hq + hkv, : hd // 2], x[:, : hq + hkv, hd // 2 :]) * turn
            y = torch.cat([z.real, z.imag], dim=-1)
            if case["rotate"]:
                y = y @ mat
            parts[0].append(y[:, :hq])
            parts[1].append(_exact_heads(y[:, hq:]))
            parts[2].append(_exact_heads(x[:, hq + hkv :]))
            first += n
        return [torch.cat(p) for p in parts]
    for b, (n, m) in enumerate(zip(new, length)):
        if case["op"] == "read":
            out.append([t.transpose(0, 1) for t in _exact_token(st, b, m - n, m)])
            continue
        for at in range(0, n, 256):
            rows = min(256, n - at)
            last = m - n + at + rows                                                  # tokens that the last of these rows sees
            q = st["q"][first + at : first + at + rows].double().view(rows, hkv, hq // hkv, hd)
            pos = torch.arange(last - rows, last, device="cuda")
            lo = max(0, last - rows - case["window"] + 1) if case["window"] else 0
            spans = [(lo, last)] + ([(0, min(case["sinks"], lo))] if lo and case["sinks"] else [])
            kv = [_exact_token(st, b, *s) for s in spans]
            k, v = (torch.cat([t[i] for t in kv], dim=1) for i in (0, 1))
            j = torch.cat([torch.arange(*s, device="cuda") for s in spans])
            see = j[None, :] <= pos[:, None]
            if case["window"]:
                see &= (pos[:, None] - j[None, :] < case["window"]) | (j[None, :] < case["sinks"])
            w = torch.einsum("rhgd,hjd->hgrj", q, k) / math.sqrt(hd)
            w = torch.softmax(w.masked_fill(~see, -math.inf), dim=-1)
            out.append(torch.einsum("hgrj,hjd->rhgd", w, v).reshape(rows, hq, hd))
        first += n
    if case["op"] == "read":
        return [torch.cat([o[i] for o in out]) for i in (0, 1)]
    return torch.cat(out)
