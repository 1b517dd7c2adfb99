"""Steps of the paged cache in which some rows have no new tokens."""
import pytest
import torch

import kvmix_b200 as kv

pytestmark = pytest.mark.gpu


def test_angles_reach_as_far_as_new_tokens_do(cuda):
    """A long sequence that has none this time does not ask for longer tables."""
    gen = torch.Generator().manual_seed(1)
    cache = kv.KVmixPagedCache([(4, 2)], 2, 128, 3, 1024, 8, 20, 64)
    cache.extend([0, 1], [700, 13])
    step = cache.extend([0, 1, 2], [0, 3, 1])
    turns = torch.arange(16)[:, None] * 10000.0 ** (-torch.arange(64) / 64)
    cos, sin = turns.cos().cuda(), turns.sin().cuda()
    k, v, q = (torch.randn(4, h, 128, generator=gen).half().cuda() for h in (2, 2, 4))
    got = cache.append(0, k, v, cos, sin, step, q=q)
    cache.check()
    pos = torch.tensor([13, 14, 15, 0]).cuda()
    c, s = cos[pos][:, None].double(), sin[pos][:, None].double()
    x, y = q[..., :64].double(), q[..., 64:].double()
    want = torch.cat([x * c - y * s, y * c + x * s], -1)
    assert ((got.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -20 * q.abs().max().double()).all()       # rounded once; two products and a sum in fp32
    for short, least in (([0, 1, 0], 16), ([0, 0, 1], 1), ([1, 0, 0], 700)):
        step = cache.extend([0, 1, 2], short)
        with pytest.raises(RuntimeError, match="angles for"):
            cache.append(0, k[:1], v[:1], cos[:least].contiguous(), sin[:least].contiguous(), step)
    step = cache.extend([0, 1, 2], [0, 0, 0])
    assert cache.append(0, k[:0], v[:0], cos[:0], sin[:0], step) is None
    cache.check()
