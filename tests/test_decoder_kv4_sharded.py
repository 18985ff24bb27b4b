"""Prompt passes under tensor parallelism with the paged 4-bit cache, on the CPU with stand-ins for kernels and collectives: the
attention sees every token of this rank's heads, and the lengths are those of all tokens."""
from types import SimpleNamespace

import pytest
import torch

from dualquant_b200 import decoder

HQ, HKV, HD, HIDDEN, INTER = 4, 2, 64, 32, 16


class Linear:
    def __init__(self, n):
        self.n, self.a, self.had, self.pw, self.r = n, None, None, SimpleNamespace(bytes_e4m3=lambda: None), None

    def byte_form_pays(self, M):
        return False

    def _gemm(self, codes, sx):
        # a row's first code in every column: rows stay recognisable
        return codes[:, :1].float().repeat(1, self.n)

    def __call__(self, x):
        return x[:, :1].float().repeat(1, self.n)

    def gated(self, gate, up):
        return gate[:, :1].repeat(1, HIDDEN) * 0


def make_layer(calls):
    layer = object.__new__(decoder.DecoderLayer)
    layer.cfg = SimpleNamespace(head_dim=HD, rms_norm_eps=1e-5, online_hadamard=True, hidden_size=HIDDEN)
    layer.tp, layer.hq, layer.hkv, layer.inter = 2, HQ, HKV, INTER
    layer.qkv, layer.o = Linear((HQ + 2 * HKV) * HD), Linear(HIDDEN)
    layer.gate_up, layer.down = Linear(2 * INTER), Linear(HIDDEN)
    layer.ln1 = layer.ln2 = None
    layer.kv4, layer.paged = object(), SimpleNamespace()

    def attend(qkv, kv_len):
        calls.append((qkv, kv_len))
        return qkv[:, : HQ * HD]

    layer.attend_paged = attend
    return layer


@pytest.fixture
def stand_ins(monkeypatch):
    """A rank of two that hears the other one say the same rows plus 100."""
    def quant(x, *_, **kw):
        return x.to(torch.int8), x[:, 0].float()

    def gather(out, part, group=None):
        out.copy_(torch.cat([part, part + 100 if part.dtype != torch.int8 else part + 50]))

    def scatter(out, whole, group=None):
        out.copy_(whole[: out.shape[0]])

    monkeypatch.setattr(decoder.ops, "quant_act_int4_rmsnorm", quant)
    monkeypatch.setattr(decoder.ops, "quant_act_int4", quant)
    monkeypatch.setattr(decoder.ops, "quant_act_int4_gated", lambda g, u, *_, **kw: (g.to(torch.int8), g[:, 0].float()))
    monkeypatch.setattr(decoder.ops, "gemm_w4a4_int4_e4m3_scatter", lambda *_: None)
    monkeypatch.setattr(decoder.dist, "all_gather_into_tensor", gather)
    monkeypatch.setattr(decoder.dist, "reduce_scatter_tensor", scatter)


def test_the_pass_over_collectives_attends_to_every_token(stand_ins):
    calls = []
    layer = make_layer(calls)
    B, S = 2, 3
    x = torch.arange(3.0)[:, None].repeat(1, HIDDEN)
    codes, sx = torch.empty(B * S, HIDDEN, dtype=torch.int8), torch.empty(B * S)
    n = torch.full((B,), 7, dtype=torch.int32)
    out = layer.forward_token_sharded(x, B, S, None, (None, None), codes, sx, None, n)
    (qkv, kv_len), = calls
    assert kv_len is n and qkv.shape == (B * S, (HQ + 2 * HKV) * HD)
    assert qkv[:, 0].tolist() == [0, 1, 2, 50, 51, 52]
    assert torch.equal(out, 2 * x)  # the residual and the stand-in's first column


def test_the_pass_over_peer_memory_attends_to_every_token(stand_ins):
    calls = []
    layer = make_layer(calls)
    B, S = 2, 3
    x = torch.arange(3.0)[:, None].repeat(1, HIDDEN)
    rows = torch.arange(6, dtype=torch.int8)[:, None].repeat(1, HIDDEN)
    steps = []
    xc = SimpleNamespace(codes=rows, sx=torch.ones(6), push=lambda *_: steps.append("push"),
                         barrier=lambda: steps.append("barrier"), add_partials=lambda *_: steps.append("add"))
    n = torch.full((B,), 9, dtype=torch.int32)
    layer.forward_token_sharded(x, B, S, None, (None, None), None, None, xc, n)
    (qkv, kv_len), = calls
    assert kv_len is n and qkv[:, 0].tolist() == [0, 1, 2, 3, 4, 5]
    assert steps == ["push", "barrier", "barrier", "add", "push", "barrier", "barrier", "add"]


@pytest.mark.parametrize("sharded", [True, False])
def test_pieces_of_prompts_carry_the_lengths_of_all_tokens(sharded):
    m = object.__new__(decoder.Decoder)
    m.cfg = SimpleNamespace(hidden_size=HIDDEN, rms_norm_eps=1e-5)
    m.tp, m.rank, m.group, m.device, m.max_len = 2, 1, None, torch.device("cpu"), 64
    m.token_sharded_prefill, m.prefill_exchange, m._exchange = sharded, "nccl", {}
    m.paged, m.embed = object(), torch.arange(100.0)[:, None].repeat(1, HIDDEN)
    m.cos = m.sin = torch.zeros(64, HD)
    seen = []

    class Layer:
        qkv = gate_up = Linear(1)

        def forward(self, x, cos, sin, pos0, pos_t, mask, group, ar=None, rope_tabs=None, kv_len=None):
            seen.append((x, kv_len))
            return x

        def forward_token_sharded(self, x, B, S, group, rope_tabs, codes, sx, xc=None, kv_len=None):
            assert codes.shape == (B * S, HIDDEN) and xc is None
            seen.append((x, kv_len))
            return x

    m.layers = [Layer(), Layer()]
    ids = torch.arange(12).view(2, 6)
    m._prefill_body(ids, 20)
    assert len(seen) == 2
    for x, kv_len in seen:
        assert kv_len.dtype == torch.int32 and kv_len.tolist() == [26, 26]
        assert x.reshape(-1, HIDDEN)[:, 0].tolist() == (list(range(6, 12)) if sharded else list(range(12)))
