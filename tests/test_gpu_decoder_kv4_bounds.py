"""Decoder with the paged 4-bit cache: steps and prompts that pass the cache's end."""
import pytest
import torch

from dualquant_b200 import decoder

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def make(layers=2):
    cfg = decoder.DecoderConfig(hidden_size=512, num_attention_heads=8, num_key_value_heads=2, head_dim=64,
                                intermediate_size=28 * 64, num_hidden_layers=layers, vocab_size=1000)
    return decoder.Decoder(cfg, DEV, seed=3)


# a table row of whole pages, one with room behind the last position, and pages larger than the cache
@pytest.mark.parametrize("max_len,page", [(32, 16), (37, 16), (20, 64)])
def test_a_step_outside_of_the_cache_gives_nan_logits_and_stores_nothing(max_len, page):
    m = make()
    B = 3
    ids = torch.randint(0, 1000, (B, max_len - 1), generator=torch.Generator().manual_seed(1)).to(DEV)
    tok = ids[:, 0].clone()
    with torch.no_grad():
        m.alloc_cache(B, max_len, kv="int4", page_size=page)
        m.prefill(ids)
        last = m.decode_step(tok, torch.tensor([max_len - 1], device=DEV))
        assert bool(last.isfinite().all())
        before = [layer.kv4.pages.clone() for layer in m.layers]
        pos = torch.tensor([0], device=DEV)
        for bad in (max_len, max_len + 1, max_len + page, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 3, 2 ** 62, -1, -2 ** 40):
            pos.fill_(bad)
            assert bool(m.decode_step(tok, pos).isnan().all())
        assert all(torch.equal(layer.kv4.pages, b) for layer, b in zip(m.layers, before))
        # steps within the cache are as they were
        pos.fill_(max_len - 1)
        assert torch.equal(m.decode_step(tok, pos), last)


def test_a_captured_step_that_passes_the_cache_says_so():
    m = make(1)
    with torch.no_grad():
        m.alloc_cache(2, 24, kv="int4", page_size=16)
        m.prefill(torch.arange(44, device=DEV).view(2, 22))
        tok, pos = torch.tensor([3, 4], device=DEV), torch.tensor([22], device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.decode_step(tok, pos)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m.decode_step(tok, pos)
        for at in (22, 23, 24, 25, 23):
            pos.fill_(at)
            graph.replay()
            assert bool(out.isnan().all()) == (at >= 24) and bool(out.isfinite().all()) == (at < 24)


def test_a_position_outside_of_the_cache_of_one_sequence_keeps_to_it():
    m = make(1)
    ids = torch.arange(20, device=DEV).view(2, 10)
    with torch.no_grad():
        m.alloc_cache(2, 12, kv="int4", page_size=16)
        m.prefill(ids)
        out = m.decode_step(ids[:, 0], torch.tensor([10, 12], device=DEV))
        assert bool(out[0].isfinite().all()) and bool(out[1].isnan().all())


@pytest.mark.parametrize("kv", ["int4", "bf16"])
def test_a_captured_prompt_longer_than_the_cache_is_refused(kv):
    m = make(1)
    ids = torch.zeros(1, 33, dtype=torch.long, device=DEV)
    with torch.no_grad():
        m.alloc_cache(1, 32, kv=kv)
        with pytest.raises(ValueError):
            m.capture_prefill(ids)
        m.capture_prefill(ids[:, :32])()
