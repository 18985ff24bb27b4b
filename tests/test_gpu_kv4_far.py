"""Paged 4-bit cache of more than 4 GiB: append and attention of many rows in its first and last pages."""
import pytest
import torch

import kv4_reference as ref
from dualquant_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("new", [20, 60])  # tiles of 128 and 256 rows
def test_prompts_in_pages_that_pass_32_bits(new):
    hq, hkv, hd, page, n = 32, 8, 128, 256, 256 * 3 - 5
    per = hkv * page * (hd + 8)
    count = (1 << 32) // per + 40
    gen = torch.Generator().manual_seed(17)
    big = torch.zeros(count, hkv, page * (hd + 8), dtype=torch.uint8, device="cuda")
    near = torch.zeros(3, hkv, page * (hd + 8), dtype=torch.uint8, device="cuda")
    far = i32([[count - 1, 0, count - 2]])
    x = torch.randn(n, (hq + 2 * hkv) * hd, generator=gen).to(torch.bfloat16).cuda()
    ang = torch.arange(n, device="cuda").double()[:, None] * (1e4 ** (-torch.arange(0, hd, 2, device="cuda").double() / hd))[None]
    cos, sin = ang.cos().float(), ang.sin().float()
    length = i32([n])
    # the same tokens into a small cache and into the far pages: the same bytes, and nowhere else
    want_q = ops.kv4_append(x, cos, sin, ops.KV4Cache(near, hd, page), i32([[0, 1, 2]]), length, hq)
    cache = ops.KV4Cache(big, hd, page)
    q = ops.kv4_append(x, cos, sin, cache, far, length, hq)
    assert torch.equal(q, want_q)
    for i in range(3):
        assert torch.equal(big[far[0, i]], near[i])
    assert bool((big[1 : count - 2].view(-1, per // 8, 8).amax((1, 2)) == 0).all())
    last = q[n - new :]
    got = ops.kv4_attention(last, cache, far, length)
    same = ops.kv4_attention(last, ops.KV4Cache(near, hd, page), i32([[0, 1, 2]]), length)
    assert torch.equal(got, same)
    kc, kp, vc, vp = ref.unpack(near, i32([[0, 1, 2]]), [n], hkv, hd, page)[0]
    k, v = ((c.double() * p[..., :1].double() + p[..., 1:].double()).transpose(0, 1) for c, p in ((kc, kp), (vc, vp)))
    want = ref.attention(last, [k.half().double()], [v], [new], [n])
    assert bool(((got.double() - want).abs() <= ref.attention_tolerance(want, [v], [n])).all())
    _lib.device_status(0)
