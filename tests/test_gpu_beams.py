"""Beam search on the device: the selection against its definition in 64 bits, the reordering of the paged cache's rows against a simulation in
lists, steps of both, captured ones, refusals."""
import math
import random

import pytest
import torch

import kvmix_b200 as kv
from test_gpu_paged_book import Sim, ints, snapshot, unchanged

pytestmark = pytest.mark.gpu
P = 128


# ---- selection --------------------------------------------------------------------------------------------------------------------------

def definition(logits, scores, beams, n, ends):
    """[requests] of [(value, beam, token)], best first, in 64 bits; values of beams that offer nothing are -infinity."""
    x = logits.double().cpu()
    total = torch.logsumexp(x, 1)
    value = scores.double().cpu()[:, None] + (x - total[:, None])
    value[~(torch.isfinite(total) & torch.isfinite(scores.cpu()))] = -math.inf
    out = []
    for r in range(x.shape[0] // beams):
        flat = value[r * beams:(r + 1) * beams].flatten()
        at = torch.sort(flat, descending=True, stable=True).indices[:n + 40].tolist()
        out.append([(float(flat[i]), i // x.shape[1], i % x.shape[1]) for i in at])
    return out


def check(logits, scores, beams, n=None, ends=()):
    got = kv.beam_select(logits, scores, beams, n=n, ends=ints(*ends) if ends else None)
    V, n = logits.shape[1], got.scores.shape[1]
    # a thread's terms: exponentials to 2^-22 of themselves (ex2.approx) and of arguments d off by 3 * 2^-24 |d| -- e^d |d| is at most 1/e, and their share of
    # a sum that holds a term of 1 and V terms at most ln V --, summed one after the other; partial sums meet in 64 bits
    turns = V / 4096 + 2
    off = 2.0 ** -22 + 3 * 2.0 ** -24 * (math.log(V) + 1) + (turns + 20) * 2.0 ** -24
    for r, want in enumerate(definition(logits, scores, beams, n, ends)):
        mine = list(zip(got.scores[r].tolist(), got.beams[r].tolist(), got.tokens[r].tolist()))
        for i in range(n):
            v = want[i][0]
            slack = off + 2.0 ** -23 * abs(v) if math.isfinite(v) else 0.0
            assert mine[i][0] == v or abs(mine[i][0] - v) <= slack, (r, i, mine[i], want[i])
            near = [w[1:] for w in want if w[0] == v or abs(w[0] - v) <= 2 * slack]
            if v == -math.inf or len(near) == 1 or len({w[0] for w in near}) == 1:        # one beam's continuations are compared exactly
                assert mine[i][1:] == want[i][1:], (r, i, mine[i], want[i])
            else:
                assert mine[i][1:] in near
        assert len({m[1:] for m in mine}) == n
        goes = ([m for m in mine if m[2] not in ends] + [(-math.inf, 0, 0)] * beams)[:beams]
        assert list(zip(got.next_scores[r].tolist(), got.next_beams[r].tolist(), got.next_tokens[r].tolist())) == goes
    return got


def inputs(rows, V, kind, seed, size=3.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, V, generator=gen) * size).to(kind).cuda(), (-20 * torch.rand(rows, generator=gen)).cuda()


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("requests,beams,V,n", [(1, 1, 1, 1), (1, 1, 7, 2), (2, 3, 5, 6), (1, 4, 32000, None), (3, 5, 4097, None), (2, 2, 50257, None), (5, 1, 9001, 1), (1, 64, 1000, None),
                                                (2, 7, 12289, 128), (1, 1, 130, 128), (40, 4, 8191, 8), (1, 16, 128256, 33), (160, 4, 5000, 12)])
def test_selection(cuda, kind, requests, beams, V, n):
    x, scores = inputs(requests * beams, V, kind, V + beams)
    check(x, scores, beams, n)


@pytest.mark.parametrize("ends", [(3,), (3, 17, 3), tuple(range(40))])
def test_tokens_that_end(cuda, ends):
    x, scores = inputs(8, 300, torch.float16, 1)
    x[:, list(ends)] += 9.0                                      # all of them lead
    check(x, scores, 2, ends=ends)
    small, scores = inputs(4, 3, torch.float32, 2)
    got = check(small, scores, 2, n=6, ends=(0, 1, 2))           # everything ends
    assert (got.next_scores == -math.inf).all()


@pytest.mark.parametrize("kind", [torch.float16, torch.float32])
def test_ties_go_to_the_lowest(cuda, kind):
    for V, n in ((9000, 16), (50000, 128), (300, 128)):
        scores = torch.tensor([-1.0, -1.0, -1.0, -2.0]).cuda()
        for x in (torch.zeros(4, V), torch.randint(0, 3, (1, V), generator=torch.Generator().manual_seed(3)).repeat(4, 1).float(), -torch.zeros(4, V)):
            x = x.to(kind).cuda()
            got, want = check(x, scores, 4, n), definition(x, scores, 4, n, ())[0][:n]
            assert list(zip(got.beams[0].tolist(), got.tokens[0].tolist())) == [w[1:] for w in want]        # rows alike: so are their sums
    x = torch.zeros(2, 5000)
    x[:, 1::2] = -0.0                                            # equal numbers
    assert check(x.to(kind).cuda(), torch.zeros(2).cuda(), 2, 8).tokens[0].tolist()[:4] == [0, 1, 2, 3]


def test_rows_in_order(cuda):
    """The order in which least or most of a row passes the threshold."""
    for V in (40000, 128256):
        up = torch.arange(V, dtype=torch.float32) * 1e-3
        x = torch.stack([up, up.flip(0), up.roll(V // 2), up.view(-1, 2).flip(1).flatten()]).cuda()
        for n in (8, 100):
            check(x, torch.tensor([0.0, -0.5, -0.25, -0.125]).cuda(), 4, n)


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, torch.float32])
def test_masks_and_numbers_that_are_none(cuda, kind):
    x, scores = inputs(24, 20000, kind, 4)
    low = torch.finfo(kind).min
    x[1, 5], x[2, 7], x[3, :], x[4, 1:], x[5, :] = math.nan, math.inf, -math.inf, -math.inf, low
    x[6, :] = torch.where(torch.rand(20000, generator=torch.Generator().manual_seed(5)).cuda() < 0.9995, -math.inf, x[6])
    x[7, :] = torch.where(torch.rand(20000, generator=torch.Generator().manual_seed(6)).cuda() < 0.9, low, x[7])
    x[8, 1000:], x[9, :19990], x[12:16], x[16, 3], x[17, 19999] = -math.inf, -math.inf, -math.inf, math.nan, math.inf
    scores[10], scores[11], scores[18], scores[21:24] = -math.inf, math.nan, math.inf, -math.inf
    for beams in (1, 3, 4, 8):
        for n in (2 * beams, 50):
            got = check(x, scores, beams, n)
    assert (got.scores[1, :].isfinite()).any()


def test_more_that_reach_a_bound_than_there_is_room_for(cuda):
    """Beams that offer nothing, or the same: 64 of them, 128 wanted."""
    x = torch.zeros(128, 500, device="cuda")
    for scores in (torch.zeros(128), torch.full((128,), -math.inf), torch.where(torch.arange(128) % 3 == 0, -1.0, -math.inf)):
        got, want = check(x, scores.cuda(), 64, 128), definition(x, scores.cuda(), 64, 128, ())
        for r in range(2):
            assert list(zip(got.beams[r].tolist(), got.tokens[r].tolist())) == [w[1:] for w in want[r][:128]]
    x[:] = -math.inf
    x[:, 77] = 1.0
    check(x, torch.zeros(128).cuda(), 64, 128)


def test_a_row_made_to_overflow_a_part(cuda):
    """All of a part's large logits in the pieces of few threads, each thread's above the next one's: thousands reach the first threshold."""
    V = 131072
    token = torch.arange(V)
    thread = token // 4 % 256                                    # pieces of four fp32 numbers, 256 threads by turns
    for chosen in (thread % 2 == 0, thread < 128, thread % 8 == 5):
        x = torch.where(chosen, thread + (token * 2654435761 % 2 ** 20).float() / 2 ** 20, -5.0 + token * 1e-6)
        for n in (128, 100, 40, 8):
            check(torch.stack([x, x.flip(0) * 0.9]).float().cuda(), torch.tensor([-1.0, -1.5]).cuda(), 2, n)


@pytest.mark.parametrize("beams,n", [(16, 17), (16, 48), (40, 40), (64, 64), (64, 128), (3, 128)])
def test_many_lists(cuda, beams, n):
    """Beams' scores close together and far apart, many parts and few."""
    for V in (700, 9000, 60000):
        x, scores = inputs(2 * beams, V, torch.bfloat16, V + n)
        for spread in (0.0, 1.0, 100.0):
            check(x, scores * spread, beams, n)


def test_first_step_of_a_request(cuda):
    """One beam is all there is: every continuation is its own."""
    x, _ = inputs(8, 3000, torch.float32, 7)
    got = check(x, torch.tensor([0.0] + [-math.inf] * 3).repeat(2).cuda(), 4)
    assert (got.next_beams == 0).all() and got.next_scores.isfinite().all()


@pytest.mark.parametrize("shift", range(1, 8))
def test_layouts(cuda, shift):
    """Rows at any alignment and distance."""
    for kind in (torch.float16, torch.float32):
        gen = torch.Generator().manual_seed(shift)
        wide = torch.full((6, 5000 + 2 * shift + 5), 1e4).to(kind).cuda()
        x = wide[:, shift:5000 + shift]
        x.copy_(torch.randn(6, 5000, generator=gen).to(kind))
        scores = -torch.rand(6, generator=gen).cuda()
        assert torch.equal(check(x, scores, 3).scores, kv.beam_select(x.contiguous(), scores, 3).scores)
        check(x[:, :3], scores, 3, 9)
        check(x.t().contiguous().t(), scores, 3)
        check(x[:1].expand(6, -1), scores, 3)


def test_rows_beyond_32_bits(cuda):
    x = torch.empty(17, 140_000_000, dtype=torch.float16, device="cuda")       # the last row begins 2.24e9 elements from the first
    x.zero_()
    gen = torch.Generator().manual_seed(8)
    x[:, :9000] = (torch.randn(17, 9000, generator=gen) * 3).half().cuda()
    view = x[:, :9000]
    check(view, -torch.rand(17, generator=gen).cuda(), 17)


def test_sums_of_far_exponentials(cuda):
    """A maximum that comes last, sums over spans beyond fp32's exponents."""
    x = torch.full((4, 30000), -200.0)
    x[0, -1], x[1, 0], x[2, 15000] = 300.0, 300.0, 80.0
    x[3] = torch.linspace(-3e38, 3e38, 30000)
    check(x.cuda(), torch.tensor([-1.0, -1.1, -1.2, -1.3]).cuda(), 4)


def test_equal_calls_give_equal_bits_on_any_stream_and_captured(cuda):
    x, scores = inputs(32, 30000, torch.bfloat16, 9)
    want = kv.beam_select(x, scores, 4, ends=ints(5))
    same = lambda got: all(torch.equal(a.view(torch.int32), b.view(torch.int32)) for a, b in zip(got, want))      # noqa: E731
    for _ in range(20):
        assert same(kv.beam_select(x, scores, 4, ends=ints(5)))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    ends = ints(5)
    torch.cuda.synchronize()
    got = []
    for i in range(10):                                          # two at once
        for st in (a, b):
            with torch.cuda.stream(st):
                got.append(kv.beam_select(x, scores, 4, ends=ends))
    torch.cuda.synchronize()
    assert all(same(g) for g in got)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(kv.beam_select(x, scores, 4, ends=ends))
    for i in range(4):
        x.copy_(inputs(32, 30000, torch.bfloat16, 20 + i)[0])
        want = kv.beam_select(x, scores, 4, ends=ends)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert same(outs[i % 2])


def test_no_requests_and_refused_selections(cuda):
    x, scores = inputs(6, 100, torch.float16, 10)
    empty = kv.beam_select(x[:0], scores[:0], 3)
    assert empty.scores.shape == (0, 6) and empty.next_tokens.shape == (0, 3) and empty.scores.dtype is torch.float32
    for bad in (dict(logits=x.double()), dict(logits=x[0]), dict(beams=4), dict(beams=0), dict(beams=-3), dict(scores=scores[:5]), dict(scores=scores.double()), dict(scores=scores.cpu()),
                dict(n=2), dict(n=129), dict(n=0), dict(ends=ints(1, 2), n=6), dict(ends=torch.zeros(2, device="cuda")), dict(ends=ints(1).cpu()), dict(logits=x.cpu()),
                dict(logits=x[:, :0]), dict(ends=ints(*range(43))), dict(scores=scores.repeat(2)[::2])):
        args = dict(logits=x, scores=scores, beams=3)
        args.update(bad)
        with pytest.raises(RuntimeError):
            kv.beam_select(**args)
    many = torch.zeros(65, 10, device="cuda")
    with pytest.raises(RuntimeError):
        kv.beam_select(many, torch.zeros(65, device="cuda"), 65)


# ---- reordering -------------------------------------------------------------------------------------------------------------------------

class Order(Sim):
    def reorder(self, rows, parents):
        old = {r: (list(p), n, a) for r, (p, n, a) in self.seq.items()}
        keeper = {}
        for r, p in zip(rows, parents):
            if p == r or p not in rows:
                keeper[p] = p
        for r, p in zip(rows, parents):
            keeper.setdefault(p, r)
        gone, late, moves = [[], []], [], []
        for r, p in zip(rows, parents):
            if p == r:
                continue
            pages, n, a = old[p]
            own = list(pages)
            for j, i in enumerate(own):
                if (j + 1) * P > n and keeper[p] != r:
                    late.append((r, j, i))
                else:
                    self.refs[self.kind(j, a)][i] += 1
            for j, i in enumerate(old[r][0]):
                gone[self.kind(j, old[r][2])].append(i)
            self.seq[r] = (own, n, a)
        self.drop(gone)
        for r, j, i in late:
            to = self.free[1].pop()
            self.refs[1][to] = 1
            moves.append((i, to, self.seq[r][1] % P))
            self.seq[r][0][j] = to
        return moves


def lived(seed, beams, requests, spare=4, residual=128, length=None, extra=0):
    """A cache of `requests` prompts whose beams have been apart for some tokens."""
    rng = random.Random(seed)
    n = requests * beams + extra
    cache = kv.KVmixPagedCache([(4, 2), (3, 3)], 2, 128, n + 2, 900, 60 * requests, n * 5 + spare, 64, residual)
    sim = Order(n + 2, 8, 60 * requests, n * 5 + spare)
    for l in cache.layers:
        l.kfull.normal_()
        l.vfull.normal_()
    rows = list(range(n + 2))
    rng.shuffle(rows)
    rows = rows[:n]
    heads = rows[:requests * beams:beams] + rows[requests * beams:]
    counts = [rng.randint(1, 500) if length is None else length for _ in heads]
    cache.extend(heads, counts)
    sim.extend(heads, counts)
    cache.settle(heads)
    sim.settle(heads, residual)
    for b in range(1, beams):
        cache.fork(heads[:requests], rows[b:requests * beams:beams])
        sim.fork(heads[:requests], rows[b:requests * beams:beams])
    return rng, cache, sim, rows


def contents(cache, rows):
    """What every row's fp16 tokens are, in both layers."""
    return {r: [cache.sequence(l, r)[i].clone() for l in range(len(cache.layers)) for i in (3, 7)] for r in rows}


@pytest.mark.parametrize("seed", range(4))
def test_random_reorderings(cuda, seed):
    """Steps of search, by slots and by beams: page numbers, references and stacks against the simulation, tokens against the parents'."""
    beams = [2, 3, 8, 5][seed]
    rng, cache, sim, rows = lived(seed, beams, 3)
    for step in range(25):
        counts = [rng.choice([1, 1, 1, 40])] * len(rows) if sum(cache.lengths) < len(rows) * 600 else [1] * len(rows)
        cache.extend(rows, counts)
        sim.extend(rows, counts)
        for l in cache.layers:                                   # the new tokens
            last = cache.book.length[rows].long() - 1
            page = cache.book.table[torch.tensor(rows).cuda(), last // P].long()
            l.kfull[page, :, last % P] = torch.randn(len(rows), 2, 128, device="cuda").half()
            l.vfull[page, :, last % P] = torch.randn(len(rows), 2, 128, device="cuda").half()
        taken = [rng.randrange(beams) for _ in rows]
        parents = [rows[i // beams * beams + t] for i, t in enumerate(taken)]
        before = contents(cache, rows)
        if step % 3 == 0:
            cache.reorder(rows, taken, beams)
        elif step % 3 == 1:
            cache.reorder(rows, ints(*taken), beams)
        else:
            cache.reorder(rows, parents)
        sim.reorder(rows, parents)
        sim.same(cache.book)
        assert cache.lengths == cache.book.length.tolist()
        after = contents(cache, rows)
        for r, p in zip(rows, parents):
            assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(after[r], before[p]))
        cache.settle(rows)
        sim.settle(rows, 128)
        sim.same(cache.book)
    cache.free(rows)
    assert cache.free_pages() == (180, len(rows) * 5 + 4)
    cache.check()


def test_parents_of_other_lengths_and_outside(cuda):
    """Rows take sequences of other lengths, empty ones too, and parents that are not among the rows stay."""
    rng, cache, sim, rows = lived(7, 2, 3, extra=4, spare=12)
    empty = [r for r in range(12) if r not in rows]
    for step in range(30):
        some = rng.sample(rows + empty, rng.randint(1, 9))
        parents = [rng.choice(rows + empty) for _ in some]
        before = contents(cache, rows + empty)
        cache.reorder(some, parents)
        sim.reorder(some, parents)
        sim.same(cache.book)
        assert cache.lengths == cache.book.length.tolist()
        after = contents(cache, rows + empty)
        new = dict(zip(some, parents))
        for r in rows + empty:
            assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(after[r], before[new.get(r, r)]))
        short = [r for r in rows if cache.lengths[r] < 200][:2]
        if short:
            cache.extend(short, [150] * len(short))
            sim.extend(short, [150] * len(short))
        cache.check()


def test_pages_that_come_free_serve_the_copies(cuda):
    """No spare page is needed where as many rows end as are taken twice."""
    cache = kv.KVmixPagedCache([(2, 2)], 1, 128, 5, 512, 1, 5, 64, 10 ** 6)
    sim = Order(5, 4, 1, 5)
    cache.extend([3], [130])
    sim.extend([3], [130])
    cache.fork([3, 3, 3], [0, 4, 1])
    sim.fork([3, 3, 3], [0, 4, 1])
    assert cache.free_pages()[1] == 0
    for taken in ([1, 1, 1, 3], [0, 0, 0, 0], [3, 2, 1, 0], [2, 3, 3, 2], [1, 2, 3, 3]):
        before = contents(cache, [3, 0, 4, 1])
        cache.reorder([3, 0, 4, 1], taken, 4)
        sim.reorder([3, 0, 4, 1], [[3, 0, 4, 1][t] for t in taken])
        sim.same(cache.book)
        after = contents(cache, [3, 0, 4, 1])
        for r, t in zip([3, 0, 4, 1], taken):
            assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(after[r], before[[3, 0, 4, 1][t]]))
    cache.check()


def test_reorderings_that_are_refused_change_nothing(cuda):
    _, cache, sim, rows = lived(9, 3, 2, length=200)
    book, layers, row = cache.book, cache.layers, rows[0]
    for call in (lambda: kv.pages_reorder(ints(row, row), ints(rows[1], rows[1]), book, layers), lambda: kv.pages_reorder(ints(row), ints(99), book, layers),
                 lambda: kv.pages_reorder(ints(row), ints(-1), book, layers), lambda: kv.pages_reorder(ints(-1), ints(row), book, layers),
                 lambda: kv.pages_reorder(ints(2 ** 30), ints(row), book, layers), lambda: kv.pages_reorder(ints(*rows[:3]), ints(0, 1, 3), book, layers, beams=3),
                 lambda: kv.pages_reorder(ints(*rows[:3]), ints(0, -1, 1), book, layers, beams=3)):
        before = snapshot(cache)
        call()
        with pytest.raises(RuntimeError, match="bad rows"):
            cache.check()
        unchanged(cache, before)
    before = snapshot(cache)
    cache.book.count[2] = 2                                      # another call was refused
    kv.pages_reorder(ints(*rows[:3]), ints(0, 0, 0), book, layers, beams=3)
    unchanged(cache, before)
    cache.book.count[2] = 0
    other = [r for r in range(8) if r not in rows][0]
    for call in (lambda: cache.reorder(rows, [0] * 5, 3), lambda: cache.reorder(rows, [3] * 6, 3), lambda: cache.reorder(rows[:4], [0] * 4, 3), lambda: cache.reorder(rows[:2], [0, 99]),
                 lambda: cache.reorder(rows[:2], ints(0, 0)), lambda: cache.reorder([row, row], [0, 0]), lambda: cache.reorder(rows, ints(0, 0), 3),
                 lambda: kv.pages_reorder(ints(*rows), ints(0), book, layers), lambda: kv.pages_reorder(ints(*rows), ints(*rows), book, layers, beams=4),
                 lambda: kv.pages_reorder(ints(*rows), ints(*rows).long(), book, layers), lambda: cache.reorder([row, other, rows[1]], ints(0, 0, 0), 3)):
        with pytest.raises(RuntimeError):
            call()
    unchanged(cache, before)


@pytest.mark.parametrize("seed", range(3))
def test_no_page_left_gives_the_references_back(cuda, seed):
    """Empty rows that take a partial one need a page each: none is there, and everything is as it was."""
    rng = random.Random(seed)
    cache = kv.KVmixPagedCache([(2, 2)], 1, 128, 12, 900, 10, 9, 64, 0)
    cache.extend([0, 1, 2], [300, 290, 310])                     # all nine pages
    cache.settle([0])                                            # two packed
    cache.extend([4], [200])
    assert cache.free_pages()[1] == 0
    rows = [0, 5, 6, 7, 1]
    parents = [1, 0, 1, 2, rng.choice([0, 2, 4])]
    before = snapshot(cache)
    lengths = list(cache.lengths)
    kv.pages_reorder(ints(*rows), ints(*parents), cache.book, cache.layers)
    count = cache.book.count.tolist()
    assert count[2] == 1
    cache.book.count[2] = 0
    unchanged(cache, before)
    assert cache.book.length.tolist() == lengths


def test_more_rows_than_threads(cuda):
    rng = random.Random(3)
    n = 1600
    cache = kv.KVmixPagedCache([(2, 2)], 1, 128, n, 256, 1, 3 * n, 64, 10 ** 6)
    sim = Order(n, 2, 1, 3 * n)
    rows = list(range(n))
    rng.shuffle(rows)
    counts = [rng.choice([0, 1, 127, 128, 200, 256]) for _ in rows]
    cache.extend(rows, counts)
    sim.extend(rows, counts)
    for _ in range(2):
        parents = [rng.choice(rows) for _ in rows]
        cache.reorder(rows, parents)
        sim.reorder(rows, parents)
        sim.same(cache.book)
    cache.check()


def test_lists_beyond_the_registers(cuda):
    """Few rows of many pages: more of them than the CTA's threads hold."""
    cache = kv.KVmixPagedCache([(2, 2)], 1, 128, 8, 128 * 1100, 1, 4400, 64, 10 ** 7)
    sim = Order(8, 1100, 1, 4400)
    rows = [6, 1, 3, 0, 7]
    for r, n in zip(rows, (1100 * 128, 900 * 128 + 7, 128 * 500, 128 * 1000 + 1, 0)):
        cache.extend([r], [n])
        sim.extend([r], [n])
    for parents in ([6, 1, 3, 0, 7], [1, 6, 0, 3, 7], [3, 3, 3, 3, 3], [6, 7, 7, 7, 1], [0, 0, 0, 0, 0]):
        cache.reorder(rows, parents)
        sim.reorder(rows, parents)
        sim.same(cache.book)
    cache.check()


def test_nothing_to_reorder(cuda):
    _, cache, sim, rows = lived(10, 3, 1, length=200)
    before = snapshot(cache)
    cache.reorder([], [])
    cache.reorder(rows, rows)
    cache.reorder(rows, [0, 1, 2], 3)
    unchanged(cache, before)
    cache.check()
    cache.reset()
    cache.reorder(rows, [0, 0, 0], 3)                            # empty ones
    assert cache.free_pages() == (60, 19)


@pytest.mark.parametrize("what,value", [("table", 10 ** 6), ("table", -7), ("length", 2 ** 31 - 1), ("length", -5), ("packed", 2 ** 31 - 1), ("packed", -3), ("count", 2 ** 24 * 64 - 64),
                                        ("refs", 0), ("refs", -2 ** 31), ("free_ids", 2 ** 31 - 1), ("free_ids", -1)])
def test_wrong_numbers_in_the_bookkeeping_stay_inside(cuda, what, value):
    _, cache, sim, rows = lived(11, 3, 2, length=300)
    t = getattr(cache.book, what)
    if what == "count":
        t[:2] = value
    else:
        t.fill_(value)
    for _ in range(2):
        kv.pages_reorder(ints(*rows), ints(0, 0, 1, 2, 2, 2), cache.book, cache.layers, beams=3)
    torch.cuda.synchronize()


def test_a_captured_search(cuda):
    """One graph is every step: selection, reordering, the next tokens' pages; against the same calls one by one."""
    gen = torch.Generator().manual_seed(12)
    caches = []
    for _ in range(2):
        cache = kv.KVmixPagedCache([(4, 2), (2, 2)], 2, 128, 8, 900, 30, 60, 64, 128)
        cache.extend([5, 2], [100, 260])
        for l in cache.layers:
            l.kfull.copy_(torch.randn(l.kfull.shape, generator=torch.Generator().manual_seed(1)).half())
            l.vfull.copy_(torch.randn(l.vfull.shape, generator=torch.Generator().manual_seed(2)).half())
        rows = ints(5, 1, 7, 2, 0, 4)
        kv.pages_reorder(ints(1, 7, 0, 4), ints(5, 5, 2, 2), cache.book, cache.layers)       # branches, without a fork
        caches.append(cache)
    logits = torch.zeros(6, 500, device="cuda")
    ends, ones, starts = ints(3, 9), ints(*[1] * 6), ints(*range(7))
    k = torch.zeros(6, 2, 128, dtype=torch.float16, device="cuda")
    scores = [torch.tensor([0.0, -math.inf, -math.inf] * 2, device="cuda") for _ in range(2)]

    def step(cache, scores):
        chosen = kv.beam_select(logits, scores, 3, ends=ends)
        kv.pages_reorder(rows, chosen.next_beams, cache.book, cache.layers, beams=3)
        kv.pages_extend(rows, ones, cache.book)
        for l in cache.layers:
            kv.page_write(k, k, starts, rows, cache.book, l)
        kv.pages_settle(rows, 128, cache.book, cache.layers)
        scores.copy_(chosen.next_scores.view(-1))
        return chosen

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0], scores[0])
    for i in range(200):
        logits.copy_(torch.randn(6, 500, generator=gen) * 2)
        k.copy_(torch.randn(k.shape, generator=gen).half())
        graph.replay()
        want = step(caches[1], scores[1])
        assert all(torch.equal(a.view(torch.int32), b.view(torch.int32)) for a, b in zip(got, want)), i
    for a, b in zip(caches[0].book[:6], caches[1].book[:6]):
        assert torch.equal(a, b)
    for a, b in zip(caches[0].layers, caches[1].layers):
        assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip((a.kfull, a.vfull), (b.kfull, b.vfull)))
    assert int(caches[0].book.count[2]) == 0 and caches[0].book.length.tolist()[5] == 300


def test_a_step_of_the_cache(cuda):
    rng, cache, sim, rows = lived(13, 4, 2, length=150)
    x, scores = inputs(8, 900, torch.float16, 11)
    want = kv.beam_select(x, scores, 4, ends=ints(1))
    got = cache.advance(rows, x, scores, 4, ends=ints(1))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    sim.reorder(rows, [rows[i // 4 * 4 + b] for i, b in enumerate(got.next_beams.flatten().tolist())])
    sim.same(cache.book)


def test_layers_beyond_one_launch_of_copies(cuda):
    layers = [(2, 2)] * 130
    cache = kv.KVmixPagedCache(layers, 1, 128, 3, 256, 1, 6, 64, 256)
    cache.extend([0], [70])
    for l in cache.layers:
        l.kfull.normal_()
        l.vfull.normal_()
    cache.reorder([1, 2], [0, 0])
    ids = cache.book.table[:, 0].tolist()
    assert len(set(ids)) == 3
    for l in cache.layers:
        for t in (l.kfull, l.vfull):
            assert torch.equal(t[ids[0], :, :70], t[ids[1], :, :70]) and torch.equal(t[ids[0], :, :70], t[ids[2], :, :70])
