"""Decoder with the paged 4-bit key/value cache: what the pages hold, attention over them, prompts whole and in pieces, single
tokens, captured steps."""
import pytest
import torch

import kv4_reference as ref
from dualquant_b200 import decoder, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def make(layers=2, head_dim=64, heads=8, kv_heads=2, seed=3):
    cfg = decoder.DecoderConfig(hidden_size=512, num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=head_dim,
                                intermediate_size=28 * 64, num_hidden_layers=layers, vocab_size=1000)
    return decoder.Decoder(cfg, DEV, seed=seed)


def held(layer, st, lengths):
    """Values of a layer's pages: per sequence (k, v) [hkv, n, d] fp64, and the raw codes and grids."""
    got = ref.unpack(layer.kv4.pages, st.table, lengths, layer.hkv, layer.cfg.head_dim, layer.kv4.page_size)
    val = lambda c, p: (c.double() * p[..., :1].double() + p[..., 1:].double()).transpose(0, 1)  # noqa: E731
    return [(val(a, b), val(c, d)) for a, b, c, d in got], got


@pytest.mark.parametrize("head_dim,page,window,sinks", [(64, 16, 0, 0), (128, 64, 0, 0), (128, 32, 20, 3)])
def test_a_layer_appends_and_attends(head_dim, page, window, sinks):
    m = make(1, head_dim)
    B, S = 3, 45
    m.alloc_cache(B, 80, kv="int4", page_size=page, window=window, sinks=sinks)
    layer = m.layers[0]
    gen = torch.Generator().manual_seed(1)
    rows = (layer.hq + 2 * layer.hkv) * head_dim
    have = 0
    for new in (S, 1, 1, 20):  # a prompt, single tokens, the next piece
        have += new
        qkv = torch.randn(B * new, rows, generator=gen).to(torch.bfloat16).to(DEV)
        n = torch.full((B,), have, dtype=torch.int32, device=DEV)
        got = layer.attend_paged(qkv, n).view(B * new, layer.hq, head_dim)
        pos = torch.arange(have - new, have, device=DEV).repeat(B)
        x = qkv.float().view(B * new, -1, head_dim)
        turned = ref.walsh_hadamard(ref.rotate_positions(x[:, : layer.hq + layer.hkv], m.paged.cos[pos], m.paged.sin[pos]))
        values, raw = held(layer, m.paged, [have] * B)
        kc, ks, kz = ref.quantise(turned[:, layer.hq :])
        for b in range(B):
            assert torch.equal(raw[b][0][have - new :], kc[b * new : (b + 1) * new].to(torch.uint8))
            assert torch.equal(raw[b][1][have - new :], torch.cat([ks, kz], -1)[b * new : (b + 1) * new])
        q = turned[:, : layer.hq].to(torch.bfloat16)
        want = ref.attention(q, [v[0] for v in values], [v[1] for v in values], [new] * B, [have] * B, window, sinks)
        tol = ref.attention_tolerance(want, [v[1] for v in values], [have])
        assert bool(((got.double() - want).abs() <= tol).all())


def test_rotation_tables_are_those_of_the_positions():
    m = make(1, 128)
    m.alloc_cache(1, 5000, kv="int4")
    p = torch.tensor([0, 1, 777, 4999])
    for i in (0, 5, 63):
        ang = p.double() * 500000.0 ** (-2.0 * i / 128)
        # fp32 results of fp64 angles: half a step
        assert torch.allclose(m.paged.cos[p.to(DEV), i].cpu().double(), ang.cos(), rtol=0, atol=2.0 ** -24 * 1.01)
        assert torch.allclose(m.paged.sin[p.to(DEV), i].cpu().double(), ang.sin(), rtol=0, atol=2.0 ** -24 * 1.01)


def test_single_tokens_store_what_the_whole_prompt_stores():
    """The first layer's keys and values depend on their own token only: a prompt of S + 3 tokens, one of S with three single
    tokens behind it, and one in three pieces store the same bytes."""
    m = make(2)
    B, S = 2, 70
    ids = torch.randint(0, 1000, (B, S + 3), generator=torch.Generator().manual_seed(2)).to(DEV)
    with torch.no_grad():
        m.alloc_cache(B, 128, kv="int4", page_size=32)
        whole = m.prefill(ids)
        want = m.layers[0].kv4.pages.clone()
        m.alloc_cache(B, 128, kv="int4", page_size=32)
        m.prefill(ids[:, :S])
        for i in range(3):
            steps = m.decode_step(ids[:, S + i], torch.tensor([S + i], device=DEV))
        assert torch.equal(m.layers[0].kv4.pages, want)
        m.alloc_cache(B, 128, kv="int4", page_size=32)
        for lo, hi in ((0, 33), (33, 34), (34, S + 3)):
            pieces = m.prefill(ids[:, lo:hi], pos0=lo)
        assert torch.equal(m.layers[0].kv4.pages, want)
    # The attention kernels add in different orders, so an output may differ by a bf16 step and flip a 4-bit activation code: a step
    # is a seventh of the largest of 512 values, half a deviation, 2 % of the vector's length.  A shift of 2 % of a deviation
    # flips 4 % of the next linear's 512 codes, 20 of them, sqrt(20) * 2 % = 9 %; four linears further the shift saturates near
    # four times that, 0.36: a cosine of 1 - 0.36^2 / 2 = 0.93.
    for other in (steps, pieces):
        assert other.shape == whole.shape and bool(other.isfinite().all())
        assert float(torch.cosine_similarity(other.float(), whole.float()).min()) > 0.9


def test_a_captured_step_equals_the_eager_one_and_follows_the_position():
    m = make(2)
    B, S = 3, 40
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, 1000, (B, S), generator=g).to(DEV)
    toks = torch.randint(0, 1000, (6, B), generator=g).to(DEV)
    with torch.no_grad():
        m.alloc_cache(B, 64, kv="int4", page_size=16, window=25, sinks=2)
        m.prefill(ids)
        want = [m.decode_step(toks[i], torch.tensor([S + i], device=DEV)).clone() for i in range(6)]
        pages = m.layers[1].kv4.pages.clone()
        m.prefill(ids)
        tok, pos = toks[0].clone(), torch.tensor([S], device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.decode_step(tok, pos)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m.decode_step(tok, pos)
        for i in range(6):
            tok.copy_(toks[i])
            pos.fill_(S + i)
            graph.replay()
            assert torch.equal(out, want[i])
        assert torch.equal(m.layers[1].kv4.pages, pages)


def test_a_captured_prompt_equals_the_eager_one():
    m = make(2)
    ids = torch.randint(0, 1000, (2, 33), generator=torch.Generator().manual_seed(8)).to(DEV)
    with torch.no_grad():
        m.alloc_cache(2, 64, kv="int4")
        want = m.prefill(ids)
        run = m.capture_prefill(ids.flip(1))
        assert torch.equal(run(ids), want)


def test_the_16_bit_cache_comes_back():
    m = make(1)
    ids = torch.randint(0, 1000, (1, 20), generator=torch.Generator().manual_seed(9)).to(DEV)
    with torch.no_grad():
        m.alloc_cache(1, 32)
        want = m.prefill(ids)
        m.alloc_cache(1, 32, kv="int4")
        m.prefill(ids)
        m.alloc_cache(1, 32)
        assert torch.equal(m.prefill(ids), want)


def test_refusals():
    m = make(1)
    ids = torch.zeros(1, 8, dtype=torch.long, device=DEV)
    for bad in (dict(kv="int8"), dict(window=5), dict(sinks=1), dict(kv="int4", page_size=20)):
        with pytest.raises(ValueError):
            m.alloc_cache(1, 32, **bad)
    m.alloc_cache(1, 32)
    with pytest.raises(ValueError):
        m.prefill(ids, pos0=4)
    m.alloc_cache(1, 32, kv="int4")
    with pytest.raises(ValueError):
        m.prefill(ids, pos0=25)
    with pytest.raises(ValueError):
        m.prefill(ids, pos0=-1)
    with pytest.raises(ValueError):
        make(1, head_dim=32, heads=16, kv_heads=4).alloc_cache(1, 32, kv="int4")


def test_refused_caches_leave_the_one_that_is_there():
    m = make(1)
    ids = torch.arange(8, device=DEV)[None]
    m.alloc_cache(1, 32, kv="int4", page_size=16)
    want = m.prefill(ids)
    for bad in (dict(kv="int4", page_size=0), dict(kv="int4", page_size=-16), dict(kv="int4", window=-1),
                dict(kv="int4", window=4, sinks=-1)):
        with pytest.raises(ValueError):
            m.alloc_cache(1, 32, **bad)
    assert torch.equal(m.prefill(ids), want)
