"""Paged 4-bit cache, attention by tiles of 128 and 256 query rows: what there may be in a call besides ordinary rows.  (The hint
counts up to the tokens of the call, so that batches here have as many, padding among them.)"""
import pytest
import torch

import kv4_reference as ref
from dualquant_b200 import _lib, ops

pytestmark = pytest.mark.gpu

# rows of the call and hint, four query heads to a key/value head: one and two tiles of 128 rows
TILES = [pytest.param(45, 30, id="128"), pytest.param(45, 45, id="256")]


def cu_of(new):
    return torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device="cuda")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def queries(gen, T, hq, hd):
    return torch.randn(T, hq, hd, generator=gen).to(torch.bfloat16).cuda()


def rounded(ks):
    return [k.half().double() for k in ks]


def close(got, want, vs, lengths):
    err, tol = (got.double() - want).abs(), ref.attention_tolerance(want, vs, lengths)
    return bool((err <= tol).all()), (err / tol).nan_to_num(1e9).flatten().topk(min(4, err.numel())), (err > tol).any(-1).nonzero()[:4].tolist()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T,most", TILES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3), (150, 70), (1, 0)])
def test_rows_that_see_nothing_and_pages_that_are_not_there(hd, T, most, window, sinks):
    gen = torch.Generator().manual_seed(hd + most + window)
    hq, hkv, page = 8, 2, 16
    # no token; two rows before the first token; holes; no page at all; longer holes; rows before the first token, then many
    lengths, new = [0, 2, 200, 40, 700, 20], [1, 4, 2, 1, 8, 26]
    pages, table, ks, vs = ref.make_cache(gen, 6, lengths, hkv, hd, page)
    table[2, 3], table[2, 4] = -7, pages.shape[0]
    table[3] = -1
    gone = {0, 5, 12, *range(16, 24), *range(28, 33), 40, 41, 43}  # a half tile, a whole one across, pieces of 16
    for p in gone:
        table[4, p] = 2 ** 31 - 1 if p % 2 else -(2 ** 31)
    q = queries(gen, T, hq, hd)
    out = torch.full((T, hq, hd), 5.0, dtype=torch.bfloat16, device="cuda")
    ops.kv4_attention(q, ops.KV4Cache(pages, hd, page), table, i32(lengths), cu_of(new), most, window=window, sinks=sinks, out=out)
    want = ref.attention(q[: sum(new)], rounded(ks), vs, new, lengths, window, sinks,
                         missing=lambda b, j: b == 3 or (b == 2 and 48 <= j < 80) or (b == 4 and j // 16 in gone))
    blind = (want == 0).all(-1).all(-1)
    assert bool(blind[[0, 1, 2, 7]].all()) and bool((out[: sum(new)][blind] == 0).all())
    ok, *what = close(out[: sum(new)], want, vs, lengths)
    assert ok, what
    assert bool((out[sum(new) :] == 5.0).all())
    _lib.device_status(0)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T,most", TILES)
@pytest.mark.parametrize("length", [100, 5000])  # one share a segment, and segments of several shares
def test_a_row_that_is_not_finite_keeps_to_itself(hd, T, most, length):
    gen = torch.Generator().manual_seed(hd + most)
    lengths, new = [length, 3 * length], [30, 15]
    pages, table, ks, vs = ref.make_cache(gen, 2, lengths, 1, hd, 16)
    q = queries(gen, T, 4, hd)
    bad = [(0, 1, 3, "nan"), (0, 2, 5, "inf"), (9, 0, hd - 1, "-inf"), (40, 3, 0, "nan")]
    for i, h, d, v in bad:
        q[i, h, d] = float(v)
    got = ops.kv4_attention(q, ops.KV4Cache(pages, hd, 16), table, i32(lengths), cu_of(new), most)
    for i, h, d, v in bad:
        assert bool(got[i, h].isnan().all())
        q[i, h] = 0
        got[i, h] = 0
    want = ref.attention(q, rounded(ks), vs, new, lengths)
    for i, h, d, v in bad:
        want[i, h] = 0
    ok, *what = close(got, want, vs, lengths)
    assert ok, what


@pytest.mark.parametrize("T,most", TILES)
def test_nothing_is_read_behind_the_table_row(T, most):
    gen = torch.Generator().manual_seed(8)
    pages, table, ks, vs = ref.make_cache(gen, 2, [640, 640], 2, 128, 16)
    q = queries(gen, T, 8, 128)
    for columns in (0, 1, 2, 7, 8, 9, 30):
        cut = 16 * columns
        # a length that ends with the row, and one far behind it: positions of its rows lie behind the tokens that there are
        got = ops.kv4_attention(q, ops.KV4Cache(pages, 128, 16), table[:, :columns], i32([cut + 10, 2 ** 31 - 1]), cu_of([25, 20]), most)
        want = torch.zeros(T, 8, 128, dtype=torch.float64, device="cuda")
        if columns:
            k, v = rounded([x[:, :cut] for x in ks]), [x[:, :cut] for x in vs]
            # (ref.attention takes positions from the length, and no more keys than there are)
            want = ref.attention(q, k, v, [25, 20], [cut + 10, 10 ** 6])
        ok, *what = close(got, want, vs, [640])
        assert ok, (columns, what)


@pytest.mark.parametrize("T,most", TILES)
def test_strided_queries_layers_of_a_larger_cache_and_sliced_tables(T, most):
    gen = torch.Generator().manual_seed(11)
    hq, hkv, hd, page, lengths, new = 8, 2, 64, 16, [333, 70], [30, 15]
    pages, table, ks, vs = ref.make_cache(gen, 2, lengths, hkv, hd, page)
    layers = torch.full((pages.shape[0], 3, *pages.shape[1:]), 255, dtype=torch.uint8, device="cuda")
    layers[:, 1] = pages
    wide = torch.full((2, table.shape[1] + 5), 10 ** 7, dtype=torch.int32, device="cuda")
    wide[:, 2 : 2 + table.shape[1]] = table
    want_q = queries(gen, T, hq, hd)
    want = ref.attention(want_q, rounded(ks), vs, new, lengths)
    cache = ops.KV4Cache(layers[:, 1], hd, page)
    qkv = torch.full((T, (hq + 2 * hkv) * hd), float("nan"), dtype=torch.bfloat16, device="cuda")
    qkv[:, : hq * hd] = want_q.flatten(1)
    for q in (want_q.transpose(0, 1).contiguous().transpose(0, 1), qkv[:, : hq * hd].view(T, hq, hd),
              torch.empty(T, hq, hd + 8, dtype=torch.bfloat16, device="cuda")[..., :hd].copy_(want_q),
              torch.empty(T, hq, hd + 3, dtype=torch.bfloat16, device="cuda")[..., 1 : hd + 1].copy_(want_q),
              torch.empty(T, hq, 2 * hd, dtype=torch.bfloat16, device="cuda")[..., ::2].copy_(want_q)):
        got = ops.kv4_attention(q, cache, wide[:, 2 : 2 + table.shape[1]], i32(lengths), cu_of(new), most)
        ok, *what = close(got, want, vs, lengths)
        assert ok, what


@pytest.mark.parametrize("T,most", TILES)
def test_captured_calls_follow_rows_and_lengths_on_the_device(T, most):
    gen = torch.Generator().manual_seed(14)
    hq, hkv, hd, page = 8, 2, 128, 16
    lengths = [700, 900, 90]
    pages, table, ks, vs = ref.make_cache(gen, 3, lengths, hkv, hd, page)
    cache, n, cu = ops.KV4Cache(pages, hd, page), i32(lengths), cu_of([30, 10, 5])
    qs = [queries(gen, T, hq, hd), queries(gen, T, hq, hd)]
    ops.kv4_attention(qs[0], cache, table, n, cu, most)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.kv4_attention(x, cache, table, n, cu, most))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for new, now in (([30, 10, 5], [700, 900, 90]), ([1, 0, 44], [33, 0, 44]), ([0, 45, 0], [0, 899, 12]), ([0, 0, 0], [1, 1, 1]),
                     ([45, 0, 0], [45, 3, 3]), ([15, 15, 15], [15, 16, 90])):
        n.copy_(i32(now))
        cu.copy_(cu_of(new))
        for o in outs:
            o.fill_(3.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):  # both at once
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        rows = sum(new)
        for x, o in zip(qs, outs):
            want = ref.attention(x[:rows], rounded([k[:, :m] for k, m in zip(ks, now)]), [v[:, :m] for v, m in zip(vs, now)], new, now)
            ok, *what = close(o[:rows], want, vs, lengths)
            assert ok, (new, what)
            assert bool((o[rows:] == 3.0).all())
    _lib.device_status(0)


@pytest.mark.parametrize("T,most", [(45, 30), (45, 45), (5, 5)])
def test_shared_pages_and_rows_of_one_sequence_twice(T, most):
    """Two sequences over the same pages (a shared prefix), one of them longer: as each by itself."""
    gen = torch.Generator().manual_seed(15)
    pages, table, ks, vs = ref.make_cache(gen, 1, [500], 2, 64, 32)
    both = table.repeat(2, 1)
    new = [T // 3, T - T // 3]
    q = queries(gen, T, 8, 64)
    got = ops.kv4_attention(q, ops.KV4Cache(pages, 64, 32), both, i32([500, 333]), cu_of(new), most)
    want = ref.attention(q, (rounded(ks) if most > 8 else ks) * 2, vs * 2, new, [500, 333])
    ok, *what = close(got, want, vs, [500])
    assert ok, what
