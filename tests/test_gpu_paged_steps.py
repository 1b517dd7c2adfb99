"""Steps of the paged cache: rows without new tokens, a search as the documentation has it."""
import math

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


def test_a_search_over_two_requests(cuda):
    """Rows branch into their groups, then select, reorder and extend: every row's tokens are those of the beam that it continues."""
    beams, requests, V = 3, 2, 50
    rows = [4, 0, 5, 1, 7, 2]
    cache = kv.KVmixPagedCache([(4, 2)], 2, 128, 8, 900, 30, 40, 64)
    cache.extend(rows[::beams], [200, 131])
    heads = [r for r in rows[::beams] for _ in range(beams)]
    cache.reorder(rows, heads)
    assert [cache.lengths[r] for r in rows] == [200] * 3 + [131] * 3
    scores = torch.tensor(([0.0] + [-math.inf] * (beams - 1)) * requests, device="cuda")
    eos = torch.tensor([7], dtype=torch.int32, device="cuda")
    gen = torch.Generator().manual_seed(2)
    said = {r: [] for r in rows}
    for _ in range(12):
        logits = (torch.randn(requests * beams, V, generator=gen) * 2).cuda()
        chosen = cache.advance(rows, logits, scores, beams, ends=eos)
        scores = chosen.next_scores.flatten()
        step = cache.extend(rows, [1] * len(rows))
        parents, tokens = chosen.next_beams.flatten().tolist(), chosen.next_tokens.flatten().tolist()
        said = {r: said[rows[i // beams * beams + p]] + [t] for i, (r, p, t) in enumerate(zip(rows, parents, tokens))}
        x = chosen.next_tokens.flatten()[:, None, None].expand(-1, 2, 128).half().contiguous()
        cache.write(0, x, x, step)
    cache.check()
    for r, n in zip(rows, [200] * 3 + [131] * 3):
        k = cache.sequence(0, r)[3]
        assert 7 not in said[r] and cache.lengths[r] == n + 12
        at = torch.arange(n, n + 12) - int(cache.book.packed[r]) * 128
        assert k[0, at.cuda(), 0].tolist() == said[r]
