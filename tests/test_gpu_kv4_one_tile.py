"""Attention of 33 to 128 rows to a key/value head over the paged 4-bit cache (one tile of 128 query rows): maxima that rise in the
middle of token tiles, in some warps only, and windows with first tokens, against 64-bit attention over keys as the kernel takes
them (rounded to fp16)."""
import pytest
import torch

import kv4_reference as ref
from dualquant_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def cu_of(new):
    return torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device="cuda")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def put_keys(pages, table, b, s, z, sign, hd, page):
    """Keys of sequence b: s * 15 + z where sign > 0, z elsewhere (s, z [n] fp16).  -> their values [n, hd] fp64"""
    n, hkv = len(s), pages.shape[1]
    pos = torch.arange(n, device="cuda")
    at, slot = table[b].long()[pos // page], pos % page
    code = torch.where(sign > 0, 15, 0).to(torch.uint8)
    packed = (code[0::2] | code[1::2] << 4).expand(n, hkv, hd // 2)
    pages[:, :, : page * hd // 2].view(-1, hkv, page, hd // 2)[at, :, slot] = packed
    pair = torch.stack([s, z], -1).view(torch.uint8)[:, None].expand(n, hkv, 4)
    pages[:, :, page * hd : page * (hd + 4)].view(-1, hkv, page, 4)[at, :, slot] = pair
    return s.double()[:, None] * code.double() + z.double()[:, None]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("each", [64, 128])  # tokens from rise to rise: every half of a token tile, or its second half
@pytest.mark.parametrize("rows", [(0, 32), (32, 64), (96, 128), (0, 128), (17, 18)])
@pytest.mark.parametrize("new", [16, 32])
def test_maxima_that_rise_in_some_warps_only(hd, each, rows, new):
    gen = torch.Generator().manual_seed(hd + each + rows[0] + new)
    hkv, page, B, length = 8, 32, 10, 2603
    lengths = [length] * B
    pages, table, ks, vs = ref.make_cache(gen, B, lengths, hkv, hd, page)
    sign = torch.where(torch.rand(hd, generator=gen) < 0.5, -1.0, 1.0).cuda()
    # Scores of q = sign rise by 9.5 in base 2 with every level: sqrt(hd) log2(e) g each
    level = (torch.arange(length, device="cuda") + (64 if each == 128 else 0)) // each
    g = level * 9.5 / (hd ** 0.5 * 1.4427)
    for b in range(B):
        k = put_keys(pages, table, b, (2 * g / 15).half(), (-g).half(), sign, hd, page)
        ks[b] = k.expand(hkv, length, hd).half().double()
    q = torch.randn(B * new, hkv, 4, hd, generator=gen).cuda()
    q -= (q * sign).mean(-1, keepdim=True) * sign  # rows without a rise
    row = (torch.arange(new)[:, None] * 4 + torch.arange(4)).cuda().repeat(B, 1)[:, None, :, None]
    q = torch.where((row >= rows[0]) & (row < rows[1]), sign, q)
    q = q.to(torch.bfloat16).view(B * new, 4 * hkv, hd)
    cache, n = ops.KV4Cache(pages, hd, page), i32(lengths)
    got = ops.kv4_attention(q, cache, table, n, max_new=new)
    want = ref.attention(q, ks, vs, [new] * B, lengths)
    # scores of up to 9.5 ln 2 a level, to 2^-20 (the helper counts 64 of them), against the largest span of a token's values
    span = max(float((v.amax(-1) - v.amin(-1)).max()) for v in vs)
    tol = ref.attention_tolerance(want, vs, lengths) + span * 9.5 * 0.694 * float(level.max()) * 2.0 ** -20
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), (err > tol).any(-1).nonzero()[:5].tolist())
    again = [ops.kv4_attention(q, cache, table, n, max_new=new) for _ in range(20)]
    assert all(torch.equal(a, got) for a in again)
    _lib.device_status(0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("most,new", [(20, [20, 1, 11]), (32, [32]), (9, [9, 0, 4]), (32, [100, 32, 70]), (10, [200])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 5), (63, 1), (64, 64), (65, 130), (150, 3), (700, 40), (5000, 9)])
def test_a_single_row_tile_with_windows_and_sinks(hd, most, new, window, sinks):
    gen = torch.Generator().manual_seed(hd + most + window)
    lengths = [n + 100 * i + 613 for i, n in enumerate(new)]
    pages, table, ks, vs = ref.make_cache(gen, len(new), lengths, 2, hd, 16)
    q = (torch.randn(sum(new), 8, hd, generator=gen) * 1.5).to(torch.bfloat16).cuda()
    got = ops.kv4_attention(q, ops.KV4Cache(pages, hd, 16), table, i32(lengths), cu_of(new), most, window=window, sinks=sinks)
    want = ref.attention(q, [k.half().double() for k in ks], vs, new, lengths, window, sinks)
    assert bool(((got.double() - want).abs() <= ref.attention_tolerance(want, vs, lengths)).all())


@pytest.mark.parametrize("q_scale", [3.0, 20.0])
def test_sharp_scores_of_a_single_row_tile(q_scale):
    # one token or a few carry a row: a token that is masked wrongly, left out or weighted late shows
    gen = torch.Generator().manual_seed(21)
    new, lengths = [30, 17, 5], [3000, 900, 130]
    pages, table, ks, vs = ref.make_cache(gen, 3, lengths, 2, 128, 32)
    q = (torch.randn(sum(new), 8, 128, generator=gen) * q_scale).to(torch.bfloat16).cuda()
    for window, sinks in ((0, 0), (100, 4)):
        got = ops.kv4_attention(q, ops.KV4Cache(pages, 128, 32), table, i32(lengths), cu_of(new), 30, window=window, sinks=sinks)
        want = ref.attention(q, [k.half().double() for k in ks], vs, new, lengths, window, sinks)
        # scores of up to 5.5 * q_scale * 1.5 to 2^-20, as above
        span = max(float((v.amax(-1) - v.amin(-1)).max()) for v in vs)
        tol = ref.attention_tolerance(want, vs, lengths) + span * 8.3 * q_scale * 2.0 ** -20
        assert bool(((got.double() - want).abs() <= tol).all())
