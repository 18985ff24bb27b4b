"""Paged 4-bit cache without a GPU: refusals, and the plain forms that the GPU tests rely on."""
import ctypes

import pytest
import torch

import kv4_reference as ref
from dualquant_b200 import _lib, ops


def test_cpu_tensors_are_refused():
    cache = ops.kv4_cache(2, 2, 64, 16, device="cpu")
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.kv4_attention(q, cache, table, n)
    with pytest.raises(RuntimeError):
        ops.kv4_read(cache, table, n, 1)
    with pytest.raises(RuntimeError):
        ops.kv4_append(q.view(1, 256), torch.zeros(4, 32), torch.zeros(4, 32), cache, table, n, 2)
    with pytest.raises(ValueError):
        ops.kv4_attention(q.view(1, 256), cache, table, n)


@pytest.mark.parametrize("hd,page,pages,hkv", [(96, 16, 1, 1), (64, 24, 1, 1), (64, 512, 1, 1), (64, 16, -1, 1), (64, 16, 1, 0)])
def test_caches_of_other_geometry_are_refused(hd, page, pages, hkv):
    with pytest.raises(ValueError):
        ops.kv4_cache(pages, hkv, hd, page, device="cpu")


def test_page_bytes():
    lib = _lib.load()
    assert lib.dq_kv4_page_bytes(8, 128, 64) == 8 * 64 * 136
    assert lib.dq_kv4_page_bytes(2, 64, 16) == 2 * 16 * 72
    assert lib.dq_kv4_page_bytes(0, 64, 16) == 0
    assert ops.kv4_cache(3, 2, 64, 16, device="cpu").pages.shape == (3, 2, 16 * 72)


def test_calls_without_init_return_a_status():
    lib = _lib.load()
    b = ctypes.byref(_lib.Kv4Batch())
    assert lib.dq_kv4_append(b, None, 0, None, None, 0, 1, 0, None, None) != 0
    assert lib.dq_kv4_read(b, None, None, None) != 0
    assert lib.dq_kv4_attention(b, None, 0, 0, 1, 1, 0, 0, 1.0, None, None, 0, None) != 0
    assert lib.dq_kv4_attention_workspace_bytes(b, 1, 1) == 0


def test_plain_cache_unpacks_to_its_values():
    gen = torch.Generator().manual_seed(0)
    lengths = [5, 0, 40]
    pages, table, ks, vs = ref.make_cache(gen, 3, lengths, 2, 64, 16, device="cpu")
    got = ref.unpack(pages, table, lengths, 2, 64, 16)
    for b, n in enumerate(lengths):
        kc, kp, vc, vp = got[b]
        for c, p, want in ((kc, kp, ks[b]), (vc, vp, vs[b])):
            val = c.double() * p[..., :1].double() + p[..., 1:].double()
            assert torch.equal(val.transpose(0, 1), want)


def test_plain_attention_masks_rows():
    gen = torch.Generator().manual_seed(1)
    _, _, ks, vs = ref.make_cache(gen, 1, [9], 1, 64, 16, device="cpu")
    q = torch.randn(2, 1, 64, generator=gen)
    out = ref.attention(q, ks, vs, [2], [9], window=1)
    assert torch.allclose(out[1, 0], vs[0][0, 8]) and torch.allclose(out[0, 0], vs[0][0, 7])
    assert bool((ref.attention(q, ks, vs, [2], [0]) == 0).all())


def test_walsh_hadamard_is_orthogonal():
    x = torch.eye(64, dtype=torch.float64)
    h = ref.walsh_hadamard(x)
    assert torch.allclose(h @ h.T, x)
