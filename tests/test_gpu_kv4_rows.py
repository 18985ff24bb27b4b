"""Attention over the paged 4-bit cache: rows of any size beside one another."""
import pytest
import torch

import kv4_reference as ref
from dualquant_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def cu_of(new):
    return torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device="cuda")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# (new tokens, most rows that a sequence is said to bring): four heads a group, so tiles of 8 and 16 rows
TILES = [pytest.param([1, 2], 2, id="8"), pytest.param([4, 3], 4, id="16")]
# ... and of 128 and 256, whose keys are rounded to fp16 (no more rows count than the call has tokens)
MANY = [pytest.param([9, 3], 12, id="128"), pytest.param([30, 13], 43, id="256")]


def taken(ks, most):
    """Keys as the kernel of so many rows takes them."""
    return [k.half().double() for k in ks] if most * 4 > 32 else ks


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,most", TILES + MANY)
@pytest.mark.parametrize("size", [1e7, 1e9, 1e12, 1e20, 1e30, 1e36, 3.3e38])
def test_a_row_of_large_finite_queries_leaves_its_neighbours_as_they_are(hd, new, most, size):
    gen = torch.Generator().manual_seed(hd + most)
    lengths = [400, 77]
    pages, table, ks, vs = ref.make_cache(gen, 2, lengths, 1, hd, 16)
    q = torch.randn(sum(new), 4, hd, generator=gen).to(torch.bfloat16).cuda()
    # head 1 of the first token has the signs of the key with the largest sum of sizes, which no other key's score reaches: its own
    # row is that token's values (a gap of 2^-10 of the score is 2^10 times what fp32 resolves, and above 1000 at 1e7)
    seen = ks[0][0, : lengths[0] - new[0] + 1]
    one = int(seen.abs().sum(-1).argmax())
    q[0, 1] = (seen[one].sign() * size).to(torch.bfloat16)
    score = seen @ q[0, 1].double()
    assert int(score.argmax()) == one and float(score.topk(2).values.diff()) < -(2.0 ** -10) * float(score.abs().max())
    got = ops.kv4_attention(q, ops.KV4Cache(pages, hd, 16), table, i32(lengths), cu_of(new), most)
    want = ref.attention(q, taken(ks, most), vs, new, lengths)
    tol = ref.attention_tolerance(want, vs, lengths)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), (err > tol).any(-1).nonzero().tolist())
    _lib.device_status(0)


@pytest.mark.parametrize("new,most", TILES + MANY)
@pytest.mark.parametrize("size", [1e-38, 1e-36, 1e-33, 1e-20, 1e20, 1e30, 1e34, 2.0 ** 118, 2.0 ** 124])
def test_queries_of_any_size_with_a_scale_that_makes_their_scores_ordinary(new, most, size):
    gen = torch.Generator().manual_seed(most)
    hd, lengths = 128, [400, 77]
    pages, table, ks, vs = ref.make_cache(gen, 2, lengths, 1, hd, 16)
    q = (torch.randn(sum(new), 4, hd, generator=gen).double() * size).to(torch.bfloat16).cuda()
    scale = hd ** -0.5 / size
    got = ops.kv4_attention(q, ops.KV4Cache(pages, hd, 16), table, i32(lengths), cu_of(new), most, scale=scale)
    want = ref.attention(q, taken(ks, most), vs, new, lengths, scale=scale)
    assert bool(((got.double() - want).abs() <= ref.attention_tolerance(want, vs, lengths)).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,most", TILES + MANY)
@pytest.mark.parametrize("size", [1.0, 30.0, 1e3, 1e5, 1e9, 1e20, -1e3, -1e9])
def test_scores_that_grow_to_any_size(hd, new, most, size):
    """Keys of every 64 tokens are eight times as large as those before: a row is the mean of the last of them that it sees (with
    a negative factor of the first)."""
    gen = torch.Generator().manual_seed(hd + most)
    page, lengths = 16, [448 - 5, 448 - 64 * (most % 5) - 5]
    pages, table, ks, vs = ref.make_cache(gen, 2, lengths, 1, hd, page)
    sign = torch.where(torch.rand(hd, generator=gen) < 0.5, 1, 0).cuda()
    for b, n in enumerate(lengths):
        g = 0.1 * 8.0 ** (torch.arange(n, device="cuda") // 64)  # up to 26214
        s, z = (2 * g / 15).half(), (-g).half()
        pos = torch.arange(n, device="cuda")
        at, slot = table[b].long()[pos // page], pos % page
        code = (15 * sign).to(torch.uint8)
        pages[:, :, : page * hd // 2].view(-1, 1, page, hd // 2)[at, :, slot] = (code[0::2] | code[1::2] << 4).expand(n, 1, -1)
        pages[:, :, page * hd : page * (hd + 4)].view(-1, 1, page, 4)[at, :, slot] = torch.stack([s, z], -1).view(torch.uint8)[:, None]
        ks[b] = (s.double()[:, None] * code.double() + z.double()[:, None])[None]
    # all of a row's products have one sign, so that scores are known to 2^-18 of their size in any order of sums; the gap between
    # levels is seven eighths of the larger one
    q = (1 + torch.rand(sum(new), 4, 1, generator=gen)).cuda() * size * (2.0 * sign - 1)
    q = q.to(torch.bfloat16)
    got = ops.kv4_attention(q, ops.KV4Cache(pages, hd, page), table, i32(lengths), cu_of(new), most)
    want = ref.attention(q, taken(ks, most), vs, new, lengths)
    # neighbouring levels may both count where scores are small (0.1 * 128 / sqrt(128) and 8 times that)
    assert bool(((got.double() - want).abs() <= ref.attention_tolerance(want, vs, lengths)).all())
    _lib.device_status(0)


@pytest.mark.parametrize("most", [1, 12, 43])
def test_scales_up_to_the_largest_and_refusal_of_larger_ones(most):
    gen = torch.Generator().manual_seed(3)
    pages, table, ks, vs = ref.make_cache(gen, 1, [90], 1, 64, 16)
    q = (torch.randn(most, 4, 64, generator=gen).double() * 1e-38).to(torch.bfloat16).cuda()
    cache, n = ops.KV4Cache(pages, 64, 16), i32([90])
    for scale in (3.4e38, -3.4e38, 2.4e38):  # times log2(e): past the largest number of fp32
        with pytest.raises(ValueError):
            ops.kv4_attention(q, cache, table, n, max_new=most, scale=scale)
    for scale in (2.3e38, -2.3e38):
        got = ops.kv4_attention(q, cache, table, n, max_new=most, scale=scale)
        want = ref.attention(q, taken(ks, most), vs, [most], [90], scale=scale)
        # scores of up to 60 or so: within the 64 that the tolerance counts on
        assert bool(((got.double() - want).abs() <= ref.attention_tolerance(want, vs, [90])).all())


@pytest.mark.parametrize("q_scale", [1.5, 5.0, 20.0])
@pytest.mark.parametrize("new,most", MANY)
def test_rounded_keys_move_a_row_by_no_more_than_their_rounding(new, most, q_scale):
    """Against the definition, with keys as the cache holds them: fp16 is off by 2^-11 of an element, a score by up to d of
    them, and weights of scores that are off by d each lie within exp(+-2 d) of theirs."""
    gen = torch.Generator().manual_seed(most)
    hd, lengths = 128, [700, 90]
    pages, table, ks, vs = ref.make_cache(gen, 2, lengths, 1, hd, 32)
    q = (torch.randn(sum(new), 4, hd, generator=gen) * q_scale).to(torch.bfloat16).cuda()
    got = ops.kv4_attention(q, ops.KV4Cache(pages, hd, 32), table, i32(lengths), cu_of(new), most)
    want = ref.attention(q, ks, vs, new, lengths)
    d = torch.cat([torch.einsum("ihd,jd->ihj", q[a : a + n].double().abs(), k[0].abs()).amax(-1)
                   for a, n, k in zip((0, new[0]), new, ks)]) * hd ** -0.5 * 2.0 ** -11
    span = max(float((v.amax(-1) - v.amin(-1)).max()) for v in vs)
    tol = ref.attention_tolerance(want, vs, lengths) + span * (torch.expm1(2 * d)[..., None] + 8.3 * q_scale * 2.0 ** -20)
    assert bool(((got.double() - want).abs() <= tol).all())
