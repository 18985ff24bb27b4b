"""Paged 4-bit key/value cache on the GPU: append, read and attention against plain 64-bit forms."""
import pytest
import torch

import kv4_reference as ref
from dualquant_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def cu_of(new):
    return torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device="cuda")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def tables(n, hd):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * (1.0 / 10000.0 ** (torch.arange(0, hd, 2).double() / hd))[None]
    return ang.cos().float().cuda(), ang.sin().float().cuda()


# ------------------------------------------------------------------------------------------------ append and read
def plain_append(qkv, cos, sin, new, lengths, hq, hkv, hd, rotate):
    """-> q fp32 [T, hq, hd], k and v as (codes, scale, zero), all for tokens in order"""
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(new, lengths)]).to(qkv.device)
    x = qkv[: len(pos)].float().view(len(pos), hq + 2 * hkv, hd)
    qk = ref.rotate_positions(x[:, : hq + hkv], cos[pos], sin[pos])
    if rotate:
        qk = ref.walsh_hadamard(qk)
    return qk[:, :hq], ref.quantise(qk[:, hq:]), ref.quantise(x[:, hq + hkv :])


APPENDS = [
    # hq, hkv, hd, page, new tokens, lengths with them
    (4, 2, 128, 16, [1], [1]),
    (32, 8, 128, 64, [1] * 5, [1, 64, 65, 128, 777]),
    (28, 4, 128, 32, [3, 0, 17, 40], [3, 9, 50, 72]),
    (8, 2, 64, 16, [33, 1, 0, 2], [33, 100, 0, 17]),
    (3, 1, 64, 256, [300], [555]),
    (5, 5, 128, 128, [2] * 40, [2 + 7 * i for i in range(40)]),
]


@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("hq,hkv,hd,page,new,lengths", APPENDS)
def test_append_writes_the_quantised_heads(hq, hkv, hd, page, new, lengths, rotate):
    gen = torch.Generator().manual_seed(1)
    T = sum(new)
    qkv = torch.randn(T, (hq + 2 * hkv) * hd, generator=gen)
    qkv[:, ::29] *= 6.0
    qkv = qkv.to(torch.bfloat16).cuda()
    cos, sin = tables(max(lengths) + 1, hd)
    pages, table, ks, vs = ref.make_cache(gen, len(new), lengths, hkv, hd, page)
    before = pages.clone()
    cache = ops.KV4Cache(pages, hd, page)
    q = ops.kv4_append(qkv, cos, sin, cache, table, i32(lengths), hq, cu_new=cu_of(new), rotate=rotate)
    want_q, (kc, ksc, kz), (vc, vsc, vz) = plain_append(qkv, cos, sin, new, lengths, hq, hkv, hd, rotate)
    # the same fp32 operations in the same order: the same bits (torch's d^-0.5 factor is the same fp32 number)
    assert torch.equal(q, want_q.to(torch.bfloat16))
    # every byte of the cache: the new tokens' codes and grids, all other bytes as they were
    got = ref.unpack(pages, table, lengths, hkv, hd, page)
    old = ref.unpack(before, table, lengths, hkv, hd, page)
    first = 0
    for b, (n, m) in enumerate(zip(new, lengths)):
        for i, w in ((0, kc), (2, vc)):
            assert torch.equal(got[b][i][m - n :], w[first : first + n].to(torch.uint8))
            assert torch.equal(got[b][i][: m - n], old[b][i][: m - n])
        for i, (s, z) in ((1, (ksc, kz)), (3, (vsc, vz))):
            assert torch.equal(got[b][i][m - n :], torch.cat([s, z], -1)[first : first + n])
            assert torch.equal(got[b][i][: m - n].view(torch.int16), old[b][i][: m - n].view(torch.int16))
        first += n
    per_token = hkv * (hd + 8)
    assert int((pages != before).sum()) <= T * per_token
    # what a token's grid can represent is within half a step of the value, plus the roundings of the grid's two numbers
    # (scale: 15 * 2^-11 of a step at the far end; zero: 2^-11 of its size)
    k, v = ops.kv4_read(cache, table, i32(lengths), T, cu_new=cu_of(new))
    x = qkv.float().view(T, hq + 2 * hkv, hd)[:, hq + hkv :]
    bound = vsc.float() * (0.5 + 15 * 2.0 ** -11) + vz.float().abs() * 2.0 ** -11 + 2.0 ** -8 * x.abs() + 1e-6
    assert bool(((v.float() - x).abs() <= bound).all())


@pytest.mark.parametrize("hkv,hd,page", [(1, 64, 16), (8, 128, 64), (3, 128, 32), (2, 64, 256)])
def test_read_returns_the_values_and_zeros_for_tokens_that_are_not_there(hkv, hd, page):
    gen = torch.Generator().manual_seed(2)
    lengths, new = [70, 0, 300, 5], [70, 0, 33, 9]  # the last one asks for four tokens before the first
    pages, table, ks, vs = ref.make_cache(gen, 4, lengths, hkv, hd, page)
    table[2, (290 // page)] = 10 ** 6  # a page that is not there
    cache = ops.KV4Cache(pages, hd, page)
    k, v = ops.kv4_read(cache, table, i32(lengths), sum(new), cu_new=cu_of(new))
    first = 0
    for b, (n, m) in enumerate(zip(new, lengths)):
        for i in range(n):
            j = m - n + i
            gone = j < 0 or (b == 2 and j // page == 290 // page)
            for got, want in ((k, ks), (v, vs)):
                w = torch.zeros(hkv, hd, dtype=torch.float64, device="cuda") if gone else want[b][:, j]
                # fp32 product and sum (2^-24 of the larger of the two terms), then half a bf16 step
                assert bool(((got[first + i].double() - w).abs() <= 2.0 ** -8 * w.abs() + 1e-5).all())
        first += n


def test_append_of_infinities_nan_and_huge_numbers_stores_finite_ones():
    hq, hkv, hd, page = 2, 1, 64, 16
    x = torch.randn(4, (hq + 2 * hkv) * hd, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    x[0, 2 * hd + 3], x[0, 3 * hd + 5] = float("nan"), float("inf")
    x[1, 3 * hd + 1], x[1, 3 * hd + 2] = float("-inf"), 3e38
    x[2, 3 * hd :] = 0.0
    x[3, 3 * hd :] = 1e-7
    x = x.cuda()
    cos, sin = torch.ones(16, hd // 2).cuda(), torch.zeros(16, hd // 2).cuda()
    cache = ops.kv4_cache(2, hkv, hd, page)
    cache.pages.fill_(255)
    table, n = i32([[1]]), i32([4])
    ops.kv4_append(x, cos, sin, cache, table, n, hq, rotate=False)
    k, v = ops.kv4_read(cache, table, n, 4)
    assert bool(k.isfinite().all()) and bool(v.isfinite().all())
    kc, kp, vc, vp = ref.unpack(cache.pages, table, [4], hkv, hd, page)[0]
    heads = x.float().view(4, 4, hd)
    # (the rotation by no angle multiplies the other half by 0: a NaN is in both halves behind it)
    for got_c, got_p, h in ((kc, kp, ref.rotate_positions(heads[:, 2:3], cos[:4], sin[:4])), (vc, vp, heads[:, 3:])):
        c, s, z = ref.quantise(h)
        assert torch.equal(got_c, c.to(torch.uint8)) and torch.equal(got_p, torch.cat([s, z], -1))


def test_append_skips_tokens_without_a_place_and_leaves_rows_behind_the_last_sequence():
    hq, hkv, hd, page = 4, 2, 128, 16
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(40, (hq + 2 * hkv) * hd, generator=gen).to(torch.bfloat16).cuda()
    cos, sin = tables(30, hd)
    cache = ops.kv4_cache(8, hkv, hd, page)
    cache.pages.fill_(77)
    table = i32([[0, 1], [2, 99], [-1, 3], [4, 5]])
    # beyond the rotation tables (30 positions), on a page that is not there, beyond the table row, before position 0
    new, lengths = [10, 8, 4, 3], [34, 20, 20, 2]
    q = ops.kv4_append(x, cos, sin, cache, table, i32(lengths), hq, cu_new=cu_of(new), rotate=True)
    assert bool((q[6:10] == 0).all()) and bool((q[:6] != 0).any(-1).all())  # positions 24 ... 33
    assert bool((q[10:18] != 0).any(-1).all())
    assert bool((q[22] == 0).all()) and bool((q[23:25] != 0).any(-1).all())
    changed = (cache.pages != 77).flatten(1).any(1).tolist()
    assert changed == [False, True, True, True, True, False, False, False]
    slots = (cache.pages[1, 0, : page * hd // 2].view(page, -1) != 77).any(-1).tolist()
    assert slots == [False] * 8 + [True] * 6 + [False] * 2  # tokens 24 ... 29
    long = ops.kv4_append(x[:5], cos, sin, cache, table[:1], i32([40]), hq, rotate=False)
    assert bool((long == 0).all())


# ------------------------------------------------------------------------------------------------ attention
def run_attention(hq, hkv, hd, page, new, lengths, window=0, sinks=0, seed=5, q_scale=1.5, scale=None, spread=1.0,
                  zero_scale=False, max_new=None, uniform=False, keys_fp16=False):
    gen = torch.Generator().manual_seed(seed)
    pages, table, ks, vs = ref.make_cache(gen, len(new), lengths, hkv, hd, page, spread=spread, zero_scale=zero_scale)
    q = (torch.randn(sum(new), hq, hd, generator=gen) * q_scale).to(torch.bfloat16).cuda()
    cache = ops.KV4Cache(pages, hd, page)
    got = ops.kv4_attention(q, cache, table, i32(lengths), cu_new=None if uniform else cu_of(new),
                            max_new=max_new if max_new is not None else max(new), window=window, sinks=sinks, scale=scale)
    if keys_fp16:
        ks = [k.half().double() for k in ks]
    want = ref.attention(q, ks, vs, new, lengths, window, sinks, scale)
    tol = ref.attention_tolerance(want, vs, lengths)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), int((err / tol).argmax()))
    _lib.device_status(0)


DECODES = [
    # hq, hkv, hd, page, new, lengths
    (4, 4, 128, 16, [1], [1]),
    (4, 1, 64, 16, [1], [2]),
    (32, 8, 128, 64, [1], [300]),
    (32, 8, 128, 64, [1] * 4, [1, 64, 65, 1000]),
    (28, 4, 128, 32, [1] * 3, [31, 32, 33]),
    (16, 2, 64, 16, [1] * 6, [16, 17, 0 + 1, 250, 15, 128]),
    (16, 1, 128, 128, [1, 1], [700, 129]),           # sixteen heads in a group
    (8, 2, 64, 256, [2, 3, 0, 1], [900, 3, 0, 256]),  # drafts, a sequence without tokens
    (32, 8, 128, 16, [4, 4], [500, 4]),
    (6, 2, 128, 64, [5, 1, 7], [90, 1, 700]),          # more rows than one row tile holds
    (20, 1, 64, 32, [1], [90]),                        # twenty heads in a group
    (8, 8, 128, 16, [1] * 150, [1 + (37 * i) % 300 for i in range(150)]),
]


@pytest.mark.parametrize("hq,hkv,hd,page,new,lengths", DECODES)
def test_attention_of_a_few_rows(hq, hkv, hd, page, new, lengths):
    run_attention(hq, hkv, hd, page, new, lengths)


PROMPTS = [
    # hq, hkv, hd, page, new, lengths
    (4, 1, 128, 16, [5], [5]),
    (4, 1, 64, 16, [32], [32]),                        # one full row tile
    (4, 1, 128, 64, [33], [33]),                       # one row more
    (8, 2, 128, 32, [64, 64], [64, 127]),              # both row tiles of a segment full
    (8, 2, 64, 16, [65, 1, 0, 130], [128, 1, 0, 131]),
    (28, 4, 128, 64, [100, 37, 256], [100, 700, 300]),  # seven heads in a group
    (3, 3, 128, 256, [129, 257, 300], [129, 1000, 301]),
    (16, 1, 64, 128, [200], [1333]),
    (8, 2, 128, 16, [1] * 9 + [90], [1 + 50 * i for i in range(9)] + [450]),  # a prompt among single tokens
    (32, 8, 128, 64, [700, 900], [700, 1500]),
    (2, 2, 64, 32, [50] * 140, [50 + i for i in range(140)]),
]


@pytest.mark.parametrize("hq,hkv,hd,page,new,lengths", PROMPTS)
def test_attention_of_many_rows(hq, hkv, hd, page, new, lengths):
    run_attention(hq, hkv, hd, page, new, lengths)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (40, 1), (128, 0), (129, 130), (300, 64), (5000, 4), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 128)])
def test_attention_of_many_rows_with_a_window_and_sinks(hd, page, window, sinks):
    run_attention(8, 2, hd, page, [90, 1, 300, 33], [90, 70, 713, 900], window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (7, 1), (64, 0), (64, 33), (200, 64), (5000, 4), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 128)])
def test_attention_with_a_window_and_sinks(hd, page, window, sinks):
    run_attention(8, 2, hd, page, [1, 2, 1, 3], [1, 70, 513, 300], window=window, sinks=sinks)


@pytest.mark.parametrize("spread", [1e-5, 1e-3, 30.0, 1000.0])
@pytest.mark.parametrize("new", [[1, 1], [50, 9]])
def test_attention_over_values_of_other_sizes(spread, new):
    run_attention(8, 2, 128, 32, new, [400, 77], spread=spread, q_scale=0.5 / spread if spread > 1 else 1.0)


@pytest.mark.parametrize("new", [[1, 1], [50, 9]])
def test_attention_over_constant_heads(new):
    run_attention(8, 2, 128, 32, new, [400, 77], zero_scale=True)


@pytest.mark.parametrize("q_scale", [1e-20, 1e-4, 20.0])
@pytest.mark.parametrize("new", [[1, 2], [70, 9]])
def test_attention_of_small_and_large_queries(q_scale, new):
    # Many rows take keys as fp16(c * scale + zero), 2^-11 of an element.  With q of size 20 and k of size 2 a score of 128 terms
    # moves by 20 * 2 * 2^-12 * sqrt(128) / sqrt(128) = 0.01, a weight by 1 %, above the tolerance: the reference takes them so too.
    run_attention(8, 2, 128, 32, new, [200, 77], q_scale=q_scale, keys_fp16=max(new) * 4 > 16)


@pytest.mark.parametrize("new", [[1, 2], [70, 9]])
def test_attention_takes_a_scale(new):
    run_attention(8, 2, 128, 32, new, [200, 77], scale=0.31, keys_fp16=max(new) * 4 > 16)  # (as above: scores of size 10)
    run_attention(8, 2, 64, 32, new, [200, 77], scale=-0.1)
    run_attention(8, 2, 64, 32, new, [200, 77], scale=0.0)


@pytest.mark.parametrize("new", [[1], [3], [20], [80]])
def test_attention_one_long_sequence_over_every_cta(new):
    run_attention(8, 2, 128, 32, new, [40001])


def test_attention_without_row_offsets():
    run_attention(8, 2, 128, 32, [2] * 7, [200, 77, 2, 1000, 64, 65, 66], uniform=True)
    run_attention(8, 2, 128, 32, [40] * 7, [200, 77, 40, 1000, 64, 65, 66], uniform=True)


@pytest.mark.parametrize("most", [1, 3, 1000])
def test_more_or_fewer_rows_than_the_hint(most):
    run_attention(8, 2, 128, 32, [9, 1, 30], [200, 77, 64], max_new=most)


@pytest.mark.parametrize("each", [1, 60])
def test_attention_gives_the_same_bits_again(each):
    gen = torch.Generator().manual_seed(6)
    pages, table, ks, vs = ref.make_cache(gen, 3, [5000, 100, 9000], 2, 128, 32)
    q = torch.randn(3 * each, 8, 128, generator=gen).to(torch.bfloat16).cuda()
    cache, n = ops.KV4Cache(pages, 128, 32), i32([5000, 100, 9000])
    first = ops.kv4_attention(q, cache, table, n)
    for _ in range(5):
        assert torch.equal(first, ops.kv4_attention(q, cache, table, n))


@pytest.mark.parametrize("most", [4, 100])
def test_attention_rows_that_see_nothing_are_zero_and_pages_that_are_not_there_are_not_seen(most):
    gen = torch.Generator().manual_seed(7)
    hq, hkv, hd, page = 8, 2, 128, 16
    lengths, new = [0, 2, 200, 40], [1, 4, 2, 1]  # no token; two rows before the first token
    pages, table, ks, vs = ref.make_cache(gen, 4, lengths, hkv, hd, page)
    table[2, 3], table[2, 4] = -7, pages.shape[0]  # tokens 48 ... 79 of sequence 2
    table[3] = -1
    q = torch.randn(sum(new), hq, hd, generator=gen).to(torch.bfloat16).cuda()
    got = ops.kv4_attention(q, ops.KV4Cache(pages, hd, page), table, i32(lengths), cu_new=cu_of(new), max_new=most)
    want = ref.attention(q, ks, vs, new, lengths, missing=lambda b, j: b == 3 or (b == 2 and 48 <= j < 80))
    assert bool((want[[0, 1, 2, 7]] == 0).all()) and bool((got[[0, 1, 2, 7]] == 0).all())
    assert bool(((got.double() - want).abs() <= ref.attention_tolerance(want, vs, lengths)).all())


@pytest.mark.parametrize("most", [None, 100])
def test_attention_reads_nothing_behind_the_table_row(most):
    gen = torch.Generator().manual_seed(8)
    pages, table, ks, vs = ref.make_cache(gen, 2, [64, 64], 2, 128, 16)
    q = torch.randn(2, 4, 128, generator=gen).to(torch.bfloat16).cuda()
    cache = ops.KV4Cache(pages, 128, 16)
    # two pages of each sequence's row, and a length that passes them: tokens 32 ... are not there
    got = ops.kv4_attention(q, cache, table[:, :2], i32([64, 2 ** 31 - 1]), max_new=most)
    want = ref.attention(q, [k[:, :32] for k in ks], [v[:, :32] for v in vs], [1, 1], [64, 10 ** 9])
    want[1] = ref.attention(q[1:], [ks[1][:, :32]], [vs[1][:, :32]], [1], [64])[0]
    assert bool(((got.double() - want).abs() <= ref.attention_tolerance(want, vs, [64])).all())


@pytest.mark.parametrize("most", [None, 100])
def test_attention_keeps_a_row_that_is_not_finite_to_itself(most):
    gen = torch.Generator().manual_seed(9)
    pages, table, ks, vs = ref.make_cache(gen, 2, [100, 100], 1, 64, 16)
    q = torch.randn(2, 4, 64, generator=gen).to(torch.bfloat16).cuda()
    q[0, 1, 3], q[0, 2, 5] = float("nan"), float("inf")
    got = ops.kv4_attention(q, ops.KV4Cache(pages, 64, 16), table, i32([100, 100]), max_new=most)
    assert bool(got[0, 1:3].isnan().all())
    q[0, 1:3] = 0
    want = ref.attention(q, ks, vs, [1, 1], [100, 100])
    keep = [(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (1, 3)]
    tol = ref.attention_tolerance(want, vs, [100])
    assert all(bool(((got[i].double() - want[i]).abs() <= tol[i]).all()) for i in keep)


@pytest.mark.parametrize("most", [3, 100])
def test_attention_leaves_rows_behind_the_last_sequence(most):
    gen = torch.Generator().manual_seed(10)
    pages, table, ks, vs = ref.make_cache(gen, 2, [100, 50], 2, 64, 16)
    q = torch.randn(9, 4, 64, generator=gen).to(torch.bfloat16).cuda()
    out = torch.full((9, 4, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    back = ops.kv4_attention(q, ops.KV4Cache(pages, 64, 16), table, i32([100, 50]), cu_new=i32([0, 2, 5]), max_new=most, out=out)
    assert back.data_ptr() == out.data_ptr() and bool((out[5:] == 3.0).all())
    want = ref.attention(q[:5], ks, vs, [2, 3], [100, 50])
    assert bool(((out[:5].double() - want).abs() <= ref.attention_tolerance(want, vs, [100])).all())


def test_attention_takes_strided_queries_layers_of_a_larger_cache_and_sliced_tables():
    gen = torch.Generator().manual_seed(11)
    hq, hkv, hd, page, lengths = 4, 2, 64, 16, [33, 70]
    pages, table, ks, vs = ref.make_cache(gen, 2, lengths, hkv, hd, page)
    layers = torch.full((pages.shape[0], 3, *pages.shape[1:]), 255, dtype=torch.uint8, device="cuda")
    layers[:, 1] = pages
    wide = torch.full((2, table.shape[1] + 5), 10 ** 7, dtype=torch.int32, device="cuda")
    wide[:, 2 : 2 + table.shape[1]] = table
    want_q = torch.randn(2, hq, hd, generator=gen).to(torch.bfloat16).cuda()
    want = ref.attention(want_q, ks, vs, [1, 1], lengths)
    tol = ref.attention_tolerance(want, vs, lengths)
    cache = ops.KV4Cache(layers[:, 1], hd, page)
    for q in (want_q.transpose(0, 1).contiguous().transpose(0, 1),             # [hq, T, hd] storage
              torch.empty(2, hq, hd + 8, dtype=torch.bfloat16, device="cuda")[..., :hd].copy_(want_q),
              torch.empty(2, hq, hd + 3, dtype=torch.bfloat16, device="cuda")[..., 1 : hd + 1].copy_(want_q),  # not 16-byte
              torch.empty(2, hq, 2 * hd, dtype=torch.bfloat16, device="cuda")[..., ::2].copy_(want_q)):
        for most in (1, 100):
            got = ops.kv4_attention(q, cache, wide[:, 2 : 2 + table.shape[1]], i32(lengths), max_new=most)
            assert bool(((got.double() - want).abs() <= tol).all())


def test_append_takes_strided_rows():
    gen = torch.Generator().manual_seed(12)
    hq, hkv, hd, page = 2, 1, 64, 16
    cols = (hq + 2 * hkv) * hd
    x = torch.randn(6, cols, generator=gen).to(torch.bfloat16).cuda()
    cos, sin = tables(6, hd)
    want = None
    for y in (x, torch.empty(6, cols + 8, dtype=torch.bfloat16, device="cuda")[:, :cols].copy_(x),
              torch.empty(6, cols + 5, dtype=torch.bfloat16, device="cuda")[:, 3 : cols + 3].copy_(x),
              x.t().contiguous().t(), x.repeat(1, 2).view(12, cols)[::2]):
        cache = ops.kv4_cache(1, hkv, hd, page)
        q = ops.kv4_append(y, cos, sin, cache, i32([[0]]), i32([6]), hq)
        if want is None:
            want = (q, cache.pages)
        assert torch.equal(q, want[0]) and torch.equal(cache.pages, want[1])


def test_empty_batches():
    cache = ops.kv4_cache(0, 2, 64, 16)
    none, table = i32([]), torch.empty(0, 3, dtype=torch.int32, device="cuda")
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert ops.kv4_attention(q, cache, table, none).shape == (0, 4, 64)
    cos, sin = tables(1, 64)
    assert ops.kv4_append(torch.empty(0, 512, dtype=torch.bfloat16, device="cuda"), cos, sin, cache, table, none, 4).shape == (0, 4, 64)
    assert ops.kv4_read(cache, table, none, 0)[0].shape == (0, 2, 64)
    # sequences without a page in the cache, tables without a column
    q = torch.ones(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    got = ops.kv4_attention(q, cache, torch.empty(2, 0, dtype=torch.int32, device="cuda"), i32([5, 0]))
    assert bool((got == 0).all())
    k, v = ops.kv4_read(cache, torch.zeros(2, 1, dtype=torch.int32, device="cuda"), i32([5, 9]), 4)
    assert bool((k == 0).all()) and bool((v == 0).all())


def test_refusals():
    cache = ops.kv4_cache(4, 2, 64, 16)
    table, n, q = i32([[0, 1], [2, 3]]), i32([20, 30]), torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    cos, sin = tables(32, 64)
    x = torch.zeros(2, 8 * 64, dtype=torch.bfloat16, device="cuda")
    good = ops.kv4_attention(q, cache, table, n)
    assert good.shape == q.shape
    bad_attention = [
        dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q.view(2, 256)), dict(block_table=table.long()),
        dict(block_table=table[:1]), dict(kv_len=n.long()), dict(kv_len=n[None]), dict(block_table=table.t()),
        dict(cu_new=i32([0, 1])), dict(cu_new=n.long()), dict(q=q[:1]), dict(max_new=0), dict(window=-1), dict(sinks=-1),
        dict(window=2 ** 31), dict(scale=float("nan")), dict(scale=float("inf")), dict(out=q.float()), dict(out=q),
        dict(out=torch.zeros(2, 4, 128, dtype=torch.bfloat16, device="cuda")[..., ::2]), dict(kv_len=n.cpu()),
        dict(block_table=table.cpu()), dict(q=q.cpu()),
        dict(cache=ops.KV4Cache(cache.pages, 128, 16)), dict(cache=ops.KV4Cache(cache.pages.view(torch.int8), 64, 16)),
        dict(cache=ops.KV4Cache(cache.pages[..., :-1], 64, 16)), dict(cache=ops.KV4Cache(cache.pages.transpose(0, 1), 64, 16)),
    ]
    for change in bad_attention:
        args = dict(q=q, cache=cache, block_table=table, kv_len=n)
        args.update(change)
        with pytest.raises(ValueError):
            ops.kv4_attention(**args)
    for hd, page in ((96, 16), (64, 24), (64, 8), (64, 512), (256, 16)):
        odd = ops.KV4Cache(torch.zeros(2, 2, page * (hd + 8), dtype=torch.uint8, device="cuda"), hd, page)
        with pytest.raises(ValueError):
            ops.kv4_attention(torch.zeros(2, 4, hd, dtype=torch.bfloat16, device="cuda"), odd, table, n)
        with pytest.raises(ValueError):
            ops.kv4_cache(2, 2, hd, page)
    with pytest.raises(ValueError):  # pages that do not lie on 16 bytes
        raw = torch.zeros(cache.pages.numel() + 8, dtype=torch.uint8, device="cuda")[8:].view(cache.pages.shape)
        ops.kv4_attention(q, ops.KV4Cache(raw, 64, 16), table, n)
    for change in (dict(qkv=x.float()), dict(hq=3), dict(hq=0), dict(cos_tab=cos.double()), dict(sin_tab=sin[:5]),
                   dict(cos_tab=cos[:, :16]), dict(cos_tab=cos.cpu()), dict(qkv=x[0]), dict(kv_len=n.long())):
        args = dict(qkv=x, cos_tab=cos, sin_tab=sin, cache=cache, block_table=table, kv_len=n, hq=4)
        args.update(change)
        with pytest.raises(ValueError):
            ops.kv4_append(**args)
    with pytest.raises(ValueError):
        ops.kv4_read(cache, table, n, -1)
    with pytest.raises(ValueError):
        ops.kv4_read(cache, table, n, 3)
    with pytest.raises(TypeError):
        ops.kv4_attention(None, cache, table, n)


# ------------------------------------------------------------------------------------------------ streams, graphs, together
def test_a_generation_through_the_cache_matches_attention_over_unquantised_heads():
    """Prompt, then single tokens: appended and attended to, against 64-bit attention over what the pages hold; kv4_read says
    the same."""
    gen = torch.Generator().manual_seed(13)
    hq, hkv, hd, page, B = 8, 2, 128, 16, 3
    prompt, steps = [40, 3, 17], 4
    cache = ops.kv4_cache(24, hkv, hd, page)
    table = torch.randperm(24, generator=gen).to(torch.int32).view(3, 8).cuda()
    cos, sin = tables(128, hd)
    seen = [0] * B
    for step in range(steps + 1):
        new = prompt if step == 0 else [1] * B
        seen = [a + n for a, n in zip(seen, new)]
        x = torch.randn(sum(new), (hq + 2 * hkv) * hd, generator=gen).to(torch.bfloat16).cuda()
        n = i32(seen)
        q = ops.kv4_append(x, cos, sin, cache, table, n, hq, cu_new=cu_of(new))
        got = ops.kv4_attention(q, cache, table, n, cu_new=cu_of(new), max_new=max(new))
        held = ref.unpack(cache.pages, table, seen, hkv, hd, page)
        values = [[(c.double() * p[..., :1].double() + p[..., 1:].double()).transpose(0, 1) for c, p in (h[:2], h[2:])] for h in held]
        ks, vs = [h[0] for h in values], [h[1] for h in values]
        want = ref.attention(q, ks, vs, new, seen)
        assert bool(((got.double() - want).abs() <= ref.attention_tolerance(want, vs, seen)).all())
        k, v = ops.kv4_read(cache, table, n, sum(seen), cu_new=cu_of(seen))
        for rows, heads in ((k, ks), (v, vs)):
            all_rows = torch.cat([h.transpose(0, 1) for h in heads])
            assert bool(((rows.double() - all_rows).abs() <= 2.0 ** -8 * all_rows.abs() + 1e-5).all())


@pytest.mark.parametrize("most", [1, 100])
def test_captured_calls_follow_the_lengths_on_the_device_and_graphs_do_not_share(most):
    gen = torch.Generator().manual_seed(14)
    hq, hkv, hd, page = 8, 2, 128, 16
    lengths = [700, 90]
    pages, table, ks, vs = ref.make_cache(gen, 2, lengths, hkv, hd, page)
    cache, n = ops.KV4Cache(pages, hd, page), i32(lengths)
    q = torch.randn(2, hq, hd, generator=gen).to(torch.bfloat16).cuda()
    qs = [q.clone(), q.clone()]
    ops.kv4_attention(q, cache, table, n, max_new=most)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.kv4_attention(x, cache, table, n, max_new=most))
        graphs.append(g)
    for now in ([700, 90], [33, 1], [512, 64]):
        n.copy_(i32(now))
        fresh = torch.randn(2, 2, hq, hd, generator=gen).to(torch.bfloat16).cuda()
        for x, f in zip(qs, fresh):
            x.copy_(f)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for g, s in zip(graphs, streams):  # both at once
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for f, o in zip(fresh, outs):
            want = ref.attention(f, [k[:, :m] for k, m in zip(ks, now)], [v[:, :m] for v, m in zip(vs, now)], [1, 1], now)
            assert bool(((o.double() - want).abs() <= ref.attention_tolerance(want, vs, now)).all())


def test_calls_run_on_the_current_stream():
    gen = torch.Generator().manual_seed(15)
    pages, table, ks, vs = ref.make_cache(gen, 1, [5000], 2, 64, 16)
    q = torch.randn(1, 4, 64, generator=gen).to(torch.bfloat16)
    want = ref.attention(q.cuda(), ks, vs, [1], [5000])
    side = torch.cuda.Stream()
    staged = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda")
    n = i32([5000])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(5):
            big = big @ big * 1e-3
        staged.copy_(q.cuda(non_blocking=True))  # only this stream knows that q is there
        got = ops.kv4_attention(staged, ops.KV4Cache(pages, 64, 16), table, n)
    side.synchronize()
    assert bool(((got.double() - want).abs() <= ref.attention_tolerance(want, vs, [5000])).all())


def test_offsets_that_pass_32_bits():
    """A cache of more than 4 GiB, tokens in its first and last pages."""
    hkv, hd, page = 8, 128, 256
    per = hkv * page * (hd + 8)
    count = (1 << 32) // per + 40
    gen = torch.Generator().manual_seed(16)
    pages, table, ks, vs = ref.make_cache(gen, 1, [page * 3 - 5], hkv, hd, page, extra_pages=0)
    big = torch.zeros(count, hkv, page * (hd + 8), dtype=torch.uint8, device="cuda")
    far = i32([[count - 1, 0, count - 2]])
    for i in range(3):
        big[far[0, i]] = pages[table[0, i]]
    q = torch.randn(1, 8, hd, generator=gen).to(torch.bfloat16).cuda()
    n = i32([page * 3 - 5])
    cache = ops.KV4Cache(big, hd, page)
    got = ops.kv4_attention(q, cache, far, n)
    want = ref.attention(q, ks, vs, [1], [page * 3 - 5])
    assert bool(((got.double() - want).abs() <= ref.attention_tolerance(want, vs, [page * 3])).all())
    k, v = ops.kv4_read(cache, far, n, 1)
    assert bool(((k[0].double() - ks[0][:, -1]).abs() <= 2.0 ** -8 * ks[0][:, -1].abs() + 1e-5).all())


def test_heads_up_to_the_largest_number_of_fp16_stay_finite_where_they_are_seen_and_where_not():
    # 65504 / 15 rounds up to 4368, and 15 * 4368 = 65520 would be infinite in fp16: zero weights times it would not be zero
    hq, hkv, hd, page, n = 2, 1, 64, 16, 80
    x = torch.zeros(n, 4 * hd)
    x[:, :hd] = torch.randn(n, hd, generator=torch.Generator().manual_seed(5))
    x[n - 1, 2 * hd + 3] = 65280.0  # key and value of the last token: only it sees them
    x[n - 1, 3 * hd + 1] = float("inf")
    x = x.to(torch.bfloat16).cuda()
    cos, sin = torch.ones(n, hd // 2).cuda(), torch.zeros(n, hd // 2).cuda()
    cache = ops.kv4_cache(5, hkv, hd, page)
    table, length = i32([[3, 1, 4, 0, 2]]), i32([n])
    q = ops.kv4_append(x, cos, sin, cache, table, length, hq, rotate=False)
    _, kp, vc, vp = ref.unpack(cache.pages, table, [n], hkv, hd, page)[0]
    got = 15 * vp[n - 1, 0, 0].double() + vp[n - 1, 0, 1].double()
    assert 65400 < float(got) <= 65504 and int(vc[n - 1, 0, 1]) == 15
    assert bool((15 * kp[..., 0].double() + kp[..., 1].double() < 65520).all())
    for most in (1, n):
        out = ops.kv4_attention(q, cache, table, length, max_new=most)
        assert bool(out.isfinite().all()) and bool((out[: n - 1] == 0).all())


def test_calls_back_to_back_on_one_and_on_two_streams_give_the_same_bits():
    # nothing waits for a call before the next: barriers, workspaces and joins of neighbouring calls must not meet
    gen = torch.Generator().manual_seed(11)
    batches = []
    for new, lengths, heads in (([300, 0, 17, 128], [1700, 0, 900, 128], (8, 2, 128)), ([1] * 40, list(range(1, 4001, 100)), (8, 1, 64)),
                                ([4, 2, 9], [3000, 77, 2000], (4, 4, 128)), ([700], [700], (4, 1, 64)),
                                ([20, 9, 31], [3000, 500, 2000], (8, 2, 128)), ([100] * 5, [100, 2000, 900, 5000, 300], (2, 2, 64))):
        hq, hkv, hd = heads
        pages, table, _, _ = ref.make_cache(gen, len(new), lengths, hkv, hd, 32)
        q = torch.randn(sum(new), hq, hd, generator=gen).to(torch.bfloat16).cuda()
        args = (q, ops.KV4Cache(pages, hd, 32), table, i32(lengths), cu_of(new), max(new))
        batches.append((args, ops.kv4_attention(*args).clone()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(200):
        args, want = batches[i % len(batches)]
        with torch.cuda.stream(streams[(i // 3) % 2 if i >= 100 else 0]):
            got.append((ops.kv4_attention(*args), want))
    torch.cuda.synchronize()
    _lib.device_status(0)  # (no wait of a kernel has run out)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in got)


@pytest.mark.parametrize("most", [1, 200])
def test_row_offsets_that_decrease_touch_nothing_else(most):
    gen = torch.Generator().manual_seed(12)
    pages, table, ks, vs = ref.make_cache(gen, 3, [300, 200, 300], 2, 128, 16)
    q = torch.randn(260, 4, 128, generator=gen).to(torch.bfloat16).cuda()
    cache, length = ops.KV4Cache(pages, 128, 16), i32([300, 200, 300])
    out = torch.full((260, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.kv4_attention(q, cache, table, length, i32([0, 200, 100, 250]), most, out=out)
    assert bool((out[250:] == 7).all())
    out = ops.kv4_attention(q, cache, table, length, cu_of([100, 100, 60]), most)
    want = ref.attention(q, ks, vs, [100, 100, 60], [300, 200, 300])
    assert bool(((out.double() - want).abs() <= ref.attention_tolerance(want, vs, [300])).all())


@pytest.mark.parametrize("B,new", [(33, 1), (128, 2), (129, 1), (300, 3), (40, 40)])
def test_batches_of_more_sequences_than_lanes(B, new):
    gen = torch.Generator().manual_seed(B)
    lengths = [0 if b % 7 == 3 else new + (b * 37) % 150 for b in range(B)]
    rows = [0 if m == 0 else new for m in lengths]
    pages, table, ks, vs = ref.make_cache(gen, B, lengths, 1, 64, 16)
    q = torch.randn(sum(rows), 2, 64, generator=gen).to(torch.bfloat16).cuda()
    out = ops.kv4_attention(q, ops.KV4Cache(pages, 64, 16), table, i32(lengths), cu_of(rows), new)
    want = ref.attention(q, ks, vs, rows, lengths)
    assert bool(((out.double() - want).abs() <= ref.attention_tolerance(want, vs, lengths)).all())


@pytest.mark.parametrize("hd,hkv", [(64, 3), (128, 1), (128, 5)])
def test_read_of_warps_whose_rows_belong_to_several_sequences(hd, hkv):
    gen = torch.Generator().manual_seed(hd + hkv)
    rows = [1, 2, 0, 1, 5, 1, 0, 0, 3] * 8 + [37]
    lengths = [n + (7 * i) % 30 if n else 0 for i, n in enumerate(rows)]
    pages, table, ks, vs = ref.make_cache(gen, len(rows), lengths, hkv, hd, 16)
    total = sum(rows)
    for cu in (cu_of(rows), None):
        if cu is None:
            rows, lengths, ks, vs, table = [5] * 7, [37] * 7, ks[-1:] * 7, vs[-1:] * 7, table[-1:].repeat(7, 1)
            total = 35
        k, v = ops.kv4_read(ops.KV4Cache(pages, hd, 16), table, i32(lengths), total, cu)
        for got, want in ((k, ks), (v, vs)):
            want = torch.cat([w[:, m - n : m].transpose(0, 1) for w, n, m in zip(want, rows, lengths)])
            # fp32 fma of an exact product (2^-24), then bf16
            assert bool(((got.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -23) + 1e-7).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [[3], [4], [2, 5, 0, 3], [9, 1]])
def test_attention_of_more_than_one_tile_of_eight_rows(hd, new):
    gen = torch.Generator().manual_seed(hd + len(new))
    lengths = [n + 333 * (i + 1) for i, n in enumerate(new)]
    pages, table, ks, vs = ref.make_cache(gen, len(new), lengths, 2, hd, 16)
    q = torch.randn(sum(new), 16, hd, generator=gen).to(torch.bfloat16).cuda()
    for most, window, sinks in ((max(new), 0, 0), (4, 0, 0), (4, 70, 5)):
        out = ops.kv4_attention(q, ops.KV4Cache(pages, hd, 16), table, i32(lengths), cu_of(new), most, window=window, sinks=sinks)
        want = ref.attention(q, ks, vs, new, lengths, window, sinks)
        assert bool(((out.double() - want).abs() <= ref.attention_tolerance(want, vs, lengths)).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("most,new", [(20, [20, 1, 11]), (32, [32]), (9, [9, 0, 4]), (32, [100, 32, 70]), (10, [200])])
def test_attention_of_a_single_tile_of_128_rows(hd, most, new):
    # 33 to 128 rows by the hint; tokens behind the last group of 64, rescaled rows and missing hints among them
    gen = torch.Generator().manual_seed(hd + most)
    lengths = [n + 100 * i + 613 for i, n in enumerate(new)]
    pages, table, ks, vs = ref.make_cache(gen, len(new), lengths, 2, hd, 32)
    q = (torch.randn(sum(new), 8, hd, generator=gen) * 3).to(torch.bfloat16).cuda()
    for window, sinks in ((0, 0), (150, 3)):
        out = ops.kv4_attention(q, ops.KV4Cache(pages, hd, 32), table, i32(lengths), cu_of(new), most, window=window, sinks=sinks)
        want = ref.attention(q, ks, vs, new, lengths, window, sinks)
        # keys are rounded to fp16: 2^-11 of each product's size in a score (|q| |k| / sqrt(d), four standard deviations: 4 * 3 * 3
        # * 2^-11), which moves a weight by that much relative to the values' span
        span = max(float((v.amax(-1) - v.amin(-1)).max()) for v in vs)
        assert bool(((out.double() - want).abs() <= ref.attention_tolerance(want, vs, lengths) + span * 36 * 2.0 ** -11).all())
