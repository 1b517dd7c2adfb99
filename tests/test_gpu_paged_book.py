"""Bookkeeping of the paged cache against a plain simulation (every page number), contents of its pages against the tokens that were written
and the stand-alone quantizer, refusals, captured and replayed steps."""
import random

import pytest
import torch

import kvmix_b200 as kv
from kvmix_b200 import paged

pytestmark = pytest.mark.gpu
P = 128


class Sim:
    """The bookkeeping in lists."""

    def __init__(self, slots, max_pages, n, n16):
        self.seq = {s: ([], 0, 0) for s in range(slots)}                # pages, length, packed
        self.n, self.n16, self.max_pages = n, n16, max_pages
        self.free = [list(range(n - 1, -1, -1)), list(range(n16 - 1, -1, -1))]
        self.refs = [dict(), dict()]

    def kind(self, j, packed):
        return 0 if j < packed else 1

    def extend(self, rows, counts):
        for r, c in zip(rows, counts):
            pages, n, a = self.seq[r]
            for _ in range(-(-(n + c) // P) - len(pages)):
                pages.append(self.free[1].pop())
                self.refs[1][pages[-1]] = 1
            self.seq[r] = (pages, n + c, a)

    def drop(self, gone):
        for kind, ids in enumerate(gone):
            for i in ids:
                self.refs[kind][i] -= 1
            zero = sorted({i for i in ids if self.refs[kind].get(i) == 0})
            for i in zero:
                del self.refs[kind][i]
            self.free[kind] += zero

    def free_rows(self, rows):
        gone = [[], []]
        for r in rows:
            pages, n, a = self.seq[r]
            for j, i in enumerate(pages):
                gone[self.kind(j, a)].append(i)
            self.seq[r] = ([], 0, 0)
        self.drop(gone)

    def settle(self, rows, window):
        gone, moves = [[], []], []
        for r in rows:
            pages, n, a = self.seq[r]
            want = max(a, max(0, n - window) // P)
            for j in range(a, want):
                to = self.free[0].pop()
                self.refs[0][to] = 1
                gone[1].append(pages[j])
                moves.append((pages[j], to))
                pages[j] = to
            self.seq[r] = (pages, n, want)
        self.drop(gone)

    def fork(self, parents, children):
        for p, c in zip(parents, children):
            pages, n, a = self.seq[p]
            own = list(pages)
            for j, i in enumerate(own):
                if (j + 1) * P > n:
                    own[j] = self.free[1].pop()
                    self.refs[1][own[j]] = 1
                else:
                    self.refs[self.kind(j, a)][i] += 1
            self.seq[c] = (own, n, a)

    def compact(self):
        to = []
        for kind, total in enumerate((self.n, self.n16)):
            live = sorted(self.refs[kind])
            holes = [i for i in range(len(live)) if i not in self.refs[kind]]
            m = {i: h for i, h in zip([i for i in live if i >= len(live)], holes)}
            self.refs[kind] = {m.get(i, i): c for i, c in self.refs[kind].items()}
            self.free[kind] = list(range(total - 1, len(live) - 1, -1))
            to.append(m)
        for r, (pages, n, a) in self.seq.items():
            self.seq[r] = ([to[self.kind(j, a)].get(i, i) for j, i in enumerate(pages)], n, a)

    def same(self, book):
        table, length, packed, refs, free, count = (t.cpu() for t in book[:6])
        assert count.tolist() == [len(self.free[0]), len(self.free[1]), 0, 0]
        assert free[:len(self.free[0])].tolist() == self.free[0]
        assert free[self.n:self.n + len(self.free[1])].tolist() == self.free[1]
        assert refs.tolist() == [self.refs[0].get(i, 0) for i in range(self.n)] + [self.refs[1].get(i, 0) for i in range(self.n16)]
        for r, (pages, n, a) in self.seq.items():
            assert (int(length[r]), int(packed[r])) == (n, a)
            assert table[r].tolist() == pages + [-1] * (self.max_pages - len(pages))


def poison(cache):
    for l in cache.layers:
        for t in (l.kscale, l.kmn, l.kfull, l.vscale, l.vmn, l.vfull):
            t.fill_(float("nan"))
        l.kcode.fill_(-1)
        l.vcode.fill_(-1)


def quantized(x, group, bits):
    """What the stand-alone quantizer gives for one page [heads, rows, 128]."""
    h, r, _ = x.shape
    g = 11 if bits == 3 else group
    n = paged.page_groups(bits, group)
    code = torch.empty(1, h, r, paged.page_words(bits), dtype=torch.int32, device=x.device)
    scale = torch.empty(1, h, r, n, dtype=torch.float16, device=x.device)
    mn = torch.empty_like(scale)
    kv.quantize_into(x[None], g, bits, code, scale, mn, ragged_tail=bits == 3)
    return code[0], scale[0], mn[0]


def holds(cache, layer, row, k, v, packed):
    """Row `row` of the layer holds tokens k, v [n, heads, 128], the first `packed` pages packed."""
    l = cache.layers[layer]
    n = k.shape[0]
    ids = cache.book.table[row].tolist()
    for j in range(-(-n // P)):
        a, b = k[j * P:(j + 1) * P].transpose(0, 1), v[j * P:(j + 1) * P].transpose(0, 1)
        if j < packed:
            for got, want in zip((l.kcode, l.kscale, l.kmn), quantized(a.transpose(1, 2), l.group, l.k_bits)):
                assert torch.equal(got[ids[j]], want)
            for got, want in zip((l.vcode, l.vscale, l.vmn), quantized(b, l.group, l.v_bits)):
                assert torch.equal(got[ids[j]], want)
        else:
            assert torch.equal(l.kfull[ids[j], :, :a.shape[1]], a) and torch.equal(l.vfull[ids[j], :, :b.shape[1]], b)


@pytest.mark.parametrize("seed", range(6))
def test_random_life(cuda, seed):
    """Sequences come, grow, branch, settle and go in random order; every page number and every token is followed."""
    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    layers = [[(4, 2), (3, 3)], [(2, 1)], [(1, 4), (2, 2)], [(3, 2)], [(4, 3), (1, 1)], [(2, 4)]][seed]
    group, heads, window, slots = rng.choice([32, 64, 128]), rng.choice([1, 2]), rng.choice([0, 100, 128, 300]), 9
    cache = kv.KVmixPagedCache(layers, heads, 128, slots, 2000, 90, 90, group, window)
    poison(cache)
    sim = Sim(slots, cache.book.table.shape[1], 90, 90)
    told = {s: [(torch.empty(0, heads, 128, dtype=torch.half, device="cuda"),) * 2 for _ in layers] for s in range(slots)}
    for step in range(40):
        rows = rng.sample(range(slots), rng.randint(1, 4))
        what = rng.choice(["extend", "extend", "extend", "settle", "settle", "fork", "free", "compact"])
        used = [r for r in range(slots) if sim.seq[r][1]]
        empty = [r for r in range(slots) if not sim.seq[r][1]]
        if what == "extend":
            counts = [rng.choice([0, 1, 1, 5, 127, 128, 129, 300]) for _ in rows]
            counts = [min(c, 2000 // P * P - sim.seq[r][1]) for r, c in zip(rows, counts)]
            if sum(c // P + 1 for c in counts) > len(sim.free[1]):
                continue
            s = cache.extend(rows, counts)
            sim.extend(rows, counts)
            for l in range(len(layers)):
                k, v = (torch.randn(s.tokens, heads, 128, generator=gen).half().cuda() for _ in range(2))
                wide = torch.stack([k, v], 1)                           # strided views of a projection's output
                cache.write(l, wide[:, 0], wide[:, 1], s)
                at = 0
                for r, c in zip(rows, counts):
                    told[r][l] = tuple(torch.cat([old, new[at:at + c]]) for old, new in zip(told[r][l], (k, v)))
                    at += c
        elif what == "settle":
            if sum(len(sim.seq[r][0]) for r in rows) > len(sim.free[0]):
                continue
            cache.settle(rows)
            sim.settle(rows, window)
        elif what == "fork" and used and empty:
            parents = [rng.choice(used) for _ in empty[:2]]
            if len(sim.free[1]) < 3:
                continue
            cache.fork(parents, empty[:2])
            sim.fork(parents, empty[:2])
            for p, c in zip(parents, empty[:2]):
                told[c] = list(told[p])
        elif what == "free":
            cache.free(rows)
            sim.free_rows(rows)
            for r in rows:
                told[r] = [(x[:0], y[:0]) for x, y in told[r]]
        elif what == "compact":
            cache.compact()
            sim.compact()
        sim.same(cache.book)
    cache.check()
    assert cache.lengths == [sim.seq[r][1] for r in range(slots)]
    assert sum(len(told[r][0][0]) for r in range(slots)) > 0
    for r in range(slots):
        for l in range(len(layers)):
            holds(cache, l, r, *told[r][l], sim.seq[r][2])


@pytest.mark.parametrize("kb", [1, 2, 3, 4])
@pytest.mark.parametrize("vb", [1, 2, 3, 4])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_packed_pages_are_the_quantizers(cuda, kb, vb, group):
    """Constant groups, ties, the largest and smallest fp16 among them."""
    gen = torch.Generator().manual_seed(kb * 4 + vb)
    cache = kv.KVmixPagedCache([(kb, vb)], 2, 128, 2, 400, 3, 4, group, 0)
    poison(cache)
    k, v = (torch.randn(384, 2, 128, generator=gen).half() for _ in range(2))
    for x in (k, v):
        x[:, 0, 5] = 1.5                                                # constant along tokens
        x[7] = -0.25                                                    # constant along channels
        x[128:256] = (torch.randint(-8, 9, (128, 2, 128), generator=gen) / 2).half()       # many ties
        x[256:300] *= 6e-8 * 20
        x[300:302, :, :3] = 60000.0
    k, v = k.cuda(), v.cuda()
    s = cache.extend([1], [384])
    cache.write(0, k, v, s)
    cache.settle([1])
    holds(cache, 0, 1, k, v, 3)
    cache.check()


def test_odd_strides_and_alignment(cuda):
    gen = torch.Generator().manual_seed(0)
    cache = kv.KVmixPagedCache([(4, 4)], 3, 128, 2, 400, 1, 4, 64, 400)
    flat = torch.randn(2 * 200 * 3 * 131 + 1, generator=gen).half().cuda()
    k = flat[1:1 + 200 * 3 * 131].view(200, 3, 131)[:, :, 2:130]                # rows that begin at any fp16
    v = flat[:200 * 3 * 256].view(200, 3, 128, 2)[..., 0]                       # channels two apart
    s = cache.extend([0], [200])
    cache.write(0, k, v, s)
    holds(cache, 0, 0, k, v, 0)


# ---- refusals ----------------------------------------------------------------------------------------------------------------------------

def snapshot(cache):
    return [t.clone() for t in (*cache.book[:5], cache.book.count[:2], *[t for l in cache.layers for t in l[:8]])]


def unchanged(cache, before):
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, snapshot(cache)))


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def small():
    cache = kv.KVmixPagedCache([(4, 2)], 1, 128, 5, 1024, 3, 6, 64, 0)      # four of six fp16 pages taken
    poison(cache)
    s = cache.extend([0, 2], [300, 10])
    x = torch.randn(310, 1, 128, device="cuda").half()
    cache.write(0, x, x, s)
    return cache


@pytest.mark.parametrize("call,text", [
    (lambda c: kv.pages_extend(ints(1), ints(300), c.book), "fp16 page"),
    (lambda c: kv.pages_extend(ints(1, 0), ints(1, 1000), c.book), "longer than the table"),
    (lambda c: kv.pages_extend(ints(1, 1), ints(1, 1), c.book), "bad rows"),
    (lambda c: kv.pages_extend(ints(5), ints(1), c.book), "bad rows"),
    (lambda c: kv.pages_extend(ints(-1), ints(1), c.book), "bad rows"),
    (lambda c: kv.pages_extend(ints(1), ints(-1), c.book), "bad rows"),
    (lambda c: kv.pages_free(ints(0, 0), c.book), "bad rows"),
    (lambda c: kv.pages_free(ints(7), c.book), "bad rows"),
    (lambda c: kv.pages_settle(ints(2), 0, c.book, c.layers), "packed page"),
    (lambda c: kv.pages_settle(ints(0, 0), 0, c.book, c.layers), "bad rows"),
    (lambda c: kv.pages_fork(ints(0), ints(2), c.book, c.layers), "bad rows"),
    (lambda c: kv.pages_fork(ints(0, 0), ints(1, 1), c.book, c.layers), "bad rows"),
    (lambda c: kv.pages_fork(ints(1), ints(1), c.book, c.layers), "bad rows"),
    (lambda c: kv.pages_fork(ints(0, 0, 0), ints(1, 3, 5), c.book, c.layers), "bad rows"),
    (lambda c: kv.pages_fork(ints(0, 0, 2), ints(1, 3, 4), c.book, c.layers), "fp16 page"),
])
def test_refused_calls_change_nothing(cuda, call, text):
    cache = small()
    if text == "packed page":                       # two of three packed pages taken, two due
        kv.pages_settle(ints(0), 0, cache.book, cache.layers)
        kv.pages_extend(ints(2), ints(300), cache.book)
    before = snapshot(cache)
    call(cache)
    assert int(cache.book.count[2])
    unchanged(cache, before)
    # until the status is cleared nothing changes the cache
    held = snapshot(cache)
    x = torch.zeros(10, 1, 128, device="cuda").half()
    kv.page_write(x, x, ints(0, 10), ints(2), cache.book, cache.layers[0])
    kv.pages_free(ints(0), cache.book)
    kv.pages_compact(cache.book, cache.layers)
    kv.pages_extend(ints(0), ints(0), cache.book)
    unchanged(cache, held)
    with pytest.raises(RuntimeError, match=text):
        cache.check()
    cache.check()
    cache.free([0])
    assert cache.lengths == cache.book.length.tolist()


def test_host_checks(cuda):
    cache = small()
    x = torch.zeros(10, 1, 128, device="cuda").half()
    b, l = cache.book, cache.layers[0]
    for bad in (lambda: cache.extend([0, 0], [1, 1]), lambda: cache.extend([9], [1]), lambda: cache.extend([0], [-1]), lambda: cache.fork([0], [2]),
                lambda: kv.pages_extend(ints(0), ints(1).long(), b), lambda: kv.pages_extend(ints(0).cpu(), ints(1), b),
                lambda: kv.pages_free(ints(0, 1)[::2], b._replace(table=b.table[:, ::2])), lambda: kv.pages_settle(ints(0), -1, b, [l]),
                lambda: kv.page_write(x.float(), x, ints(0, 10), ints(0), b, l), lambda: kv.page_write(x, x, ints(0), ints(0), b, l),
                lambda: kv.page_write(x, x, ints(0, 10), ints(0), b, l._replace(kcode=l.kcode[:2])), lambda: kv.paged_attention(x, ints(0, 10), ints(0), b, l._replace(group=16)),
                lambda: kv.paged_attention(x.float(), ints(0, 10), ints(0), b, l), lambda: kv.paged_attention(x, ints(0, 10, 10), ints(0), b, l),
                lambda: kv.paged_attention(x, ints(0, 10), ints(0), b, l, window=-1), lambda: kv.paged_attention(x, ints(0, 10), ints(0), b, l, softcap=-1.0),
                lambda: kv.paged_attention(x, ints(0, 10), ints(0), b, l, alibi_slopes=torch.ones(2, device="cuda")),
                lambda: kv.paged_attention(x, ints(0, 10), ints(0), b, l, first=ints(0)), lambda: kv.paged_attention(x, ints(0, 10), ints(0), b, l, prefix=ints(0, 0)),
                lambda: kv.paged_attention(x, ints(0, 10), ints(0), b, l, out=x.float()), lambda: kv.paged_attention(x, ints(0, 10), ints(0), b, l, max_new=0),
                lambda: kv.paged_attention(x[..., :64], ints(0, 10), ints(0), b, l), lambda: kv.KVmixPagedCache([(5, 2)], 1, 128, 1, 1, 1, 1, 32),
                lambda: kv.KVmixPagedCache([(4, 2)], 1, 64, 1, 1, 1, 1, 32), lambda: kv.KVmixPagedCache([(4, 2)], 1, 128, 1, 1, 1, 1, 16)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(RuntimeError, match="divisible"):
        big = kv.KVmixPagedCache([(4, 2)], 2, 128, 1, 256, 1, 2, 64)
        kv.paged_attention(torch.zeros(1, 3, 128, device="cuda").half(), ints(0, 1), ints(0), big.book, big.layers[0])


def test_numbers_that_lead_nowhere(cuda):
    """Rows and pages outside their ranges, more new tokens than the sequence has: nothing is read there, such rows of q see nothing."""
    cache = small()
    b, l = cache.book, cache.layers[0]
    q = torch.randn(300, 4, 128, device="cuda").half()
    for n in (1, 300):
        out = kv.paged_attention(q[:n], ints(0, n), ints(77), b, l)
        assert not out.any()
        out = kv.paged_attention(q[:n], ints(0, n), ints(1), b, l)
        assert not out.any()
    out = kv.paged_attention(q, ints(0, 300), ints(2), b, l)                 # ten tokens, 300 queries
    assert not out[:290].any() and out[290:].isfinite().all() and out[290:].any()
    ids = b.table[0].clone()
    want = kv.paged_attention(q[:100], ints(0, 100), ints(0), b, l, window=172)
    for bad in (-1, 99, -2 ** 31):
        b.table[0, 0] = bad                                                  # 100 tokens at 200.., each sees the page numbered `bad` and others
        got = kv.paged_attention(q[:100], ints(0, 100), ints(0), b, l)
        one = kv.paged_attention(q[:1], ints(0, 1), ints(0), b, l)
        assert got.isfinite().all() and one.isfinite().all() and got.any() and one.any()
    b.table[0].copy_(ids)
    assert want.isfinite().all()
    x = torch.zeros(400, 1, 128, device="cuda").half()
    before = snapshot(cache)
    kv.page_write(x, x, ints(0, 400), ints(1), b, l)                         # an empty sequence takes nothing
    kv.page_write(x, x, ints(0, 400), ints(-3), b, l)
    unchanged(cache, before)


def test_rows_behind_the_last_sequence_stay(cuda):
    cache = small()
    for counts, nh in (([1, 1], 4), ([100, 3], 4)):
        q = torch.randn(sum(counts) + 5, nh, 128, device="cuda").half()
        out = torch.full_like(q, 7.0)
        kv.paged_attention(q, ints(0, counts[0], sum(counts)), ints(0, 2), cache.book, cache.layers[0], out=out)
        assert (out[sum(counts):] == 7).all() and (out[:sum(counts)] != 7).any(-1).all()


# ---- streams, graphs ---------------------------------------------------------------------------------------------------------------------

def test_on_another_stream(cuda):
    cache = small()
    q = torch.randn(2, 4, 128, device="cuda").half()
    want = kv.paged_attention(q, ints(0, 1, 2), ints(0, 2), cache.book, cache.layers[0])
    at, rows, side = ints(0, 1, 2), ints(0, 2), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kv.paged_attention(q, at, rows, cache.book, cache.layers[0])
    side.synchronize()
    assert torch.equal(got, want)


def test_captured_steps(cuda):
    """A decode step of three sequences -- pages, keys and values, attention, packing -- captured once and replayed 300 times, beside the same
    steps launched one by one; two graphs replayed in turn keep apart what they work with."""
    gen = torch.Generator().manual_seed(5)
    caches = [kv.KVmixPagedCache([(2, 2), (3, 4)], 2, 128, 4, 1500, 40, 16, 64, 128) for _ in range(2)]
    rows, prompt = [3, 0, 2], [200, 127, 1]
    first = [torch.randn(sum(prompt), 2, 128, generator=gen).half().cuda() for _ in range(4)]
    for c in caches:
        s = c.extend(rows, prompt)
        for l in range(2):
            c.write(l, first[2 * l], first[2 * l + 1], s)
        c.settle(rows)
    graphed, plain = caches
    at, ones, starts = ints(*rows), ints(1, 1, 1), ints(0, 1, 2, 3)
    q, k, v = (torch.zeros(2, 3, h, 128, dtype=torch.half, device="cuda") for h in (8, 2, 2))
    outs = torch.zeros(2, 3, 8, 128, dtype=torch.half, device="cuda")

    def step(c, out):
        kv.pages_extend(at, ones, c.book)
        for l in range(2):
            kv.page_write(k[l], v[l], starts, at, c.book, c.layers[l])
            kv.paged_attention(q[l], starts, at, c.book, c.layers[l], max_new=1, max_tokens=1500, out=out[l])
        kv.pages_settle(at, 128, c.book, c.layers)

    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    torch.cuda.synchronize()
    for g in graphs:
        with torch.cuda.graph(g):
            step(graphed, outs)
    want = torch.zeros_like(outs)
    for i in range(300):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen).half())
        graphs[i % 2].replay()
        step(plain, want)
        assert torch.equal(outs, want), i
    for a, b in zip(graphed.book[:6], plain.book[:6]):
        assert torch.equal(a, b)
    assert plain.book.packed.tolist() == [2, 0, 1, 2][:4] or plain.book.length[3] == 500
    graphed.check()
    plain.check()


def test_a_sequence_in_chunks_is_the_sequence_at_once(cuda):
    """The cached attention of a prompt in chunks, of its fork and of single tokens behind it against attention over what the cache holds."""
    gen = torch.Generator().manual_seed(11)
    cache = kv.KVmixPagedCache([(4, 4)], 2, 128, 3, 1200, 12, 20, 32, 128)
    k, v, q = (torch.randn(900, h, 128, generator=gen).half().cuda() for h in (2, 2, 8))

    def exact(row, q, at):
        kc, ks, km, kf, vc, vs, vm, vf, n = cache.sequence(0, row)
        K, V = kf.double(), vf.double()
        if kc is not None:
            f = torch.arange(0, 32, 4, device="cuda")
            un = lambda c: ((c[..., None] >> f) & 15).flatten(-2).double().unflatten(-1, (-1, 32))      # noqa: E731
            K = torch.cat([(un(kc) * ks.double()[..., None] + km.double()[..., None]).flatten(-2).transpose(1, 2), K], 1)
            V = torch.cat([(un(vc) * vs.double()[..., None] + vm.double()[..., None]).flatten(-2), V], 1)
        assert K.shape[1] == n
        s = torch.einsum("thd,hnd->htn", q.double(), K.repeat_interleave(4, 0)) / 128 ** 0.5
        pos = torch.arange(at, at + q.shape[0], device="cuda")
        s = s.masked_fill(torch.arange(n, device="cuda")[None, None] > pos[None, :, None], float("-inf"))
        return torch.einsum("htn,hnd->thd", s.softmax(-1), V.repeat_interleave(4, 0))

    at = 0
    for n in (250, 1, 300, 128, 1, 1, 100):
        s = cache.extend([1], [n])
        cache.write(0, k[at:at + n], v[at:at + n], s)
        got, want = cache.attend(0, q[at:at + n], s), exact(1, q[at:at + n], at)
        # two roundings of 2^-11 at most of keys, values and weights, by rows
        assert ((got.double() - want).norm(dim=-1) <= 4e-3 * want.norm(dim=-1)).all()
        cache.settle()
        at += n
    cache.fork([1], [0])
    cache.free([1])
    cache.compact()
    s = cache.extend([0], [1])
    cache.write(0, k[at:at + 1], v[at:at + 1], s)
    got, want = cache.attend(0, q[at:at + 1], s), exact(0, q[at:at + 1], at)
    assert ((got.double() - want).norm(dim=-1) <= 4e-3 * want.norm(dim=-1)).all()
    cache.check()


def test_more_rows_than_a_cta_has_threads(cuda):
    """Prefix sums that go on over several turns of 1024 rows, stacks and tables against the simulation; the pools are odd sizes."""
    rng = random.Random(1)
    n = 2600
    cache = kv.KVmixPagedCache([(2, 2)], 1, 128, n, 512, 5001, 6003, 128, 0)
    sim = Sim(n, 4, 5001, 6003)
    rows = list(range(n))
    rng.shuffle(rows)
    counts = [rng.choice([0, 1, 128, 200, 256]) for _ in rows]
    cache.extend(rows, counts)
    sim.extend(rows, counts)
    for l in cache.layers:
        l.kfull.zero_()
        l.vfull.zero_()
    cache.settle(rows[:2000])
    sim.settle(rows[:2000], 0)
    sim.same(cache.book)
    gone = rows[::2]
    cache.free(gone)
    sim.free_rows(gone)
    sim.same(cache.book)
    parents = [r for r in rows[1::2] if sim.seq[r][1]]
    cache.fork(parents, gone[:len(parents)])
    sim.fork(parents, gone[:len(parents)])
    sim.same(cache.book)
    cache.free(parents[:700])
    sim.free_rows(parents[:700])
    cache.compact()
    sim.compact()
    sim.same(cache.book)
    cache.check()


def test_calls_without_rows(cuda):
    cache = small()
    before = snapshot(cache)
    none = ints()
    kv.pages_extend(none, none, cache.book)
    kv.pages_free(none, cache.book)
    kv.pages_settle(none, 0, cache.book, cache.layers)
    kv.pages_fork(none, none, cache.book, cache.layers)
    x = torch.zeros(0, 1, 128, device="cuda").half()
    kv.page_write(x, x, ints(0), none, cache.book, cache.layers[0])
    unchanged(cache, before)
    cache.check()
    bare = kv.KVmixPagedCache([(2, 2)], 1, 128, 2, 300, 0, 3, 64, 1000)          # no packed page at all
    s = bare.extend([0], [200])
    x = torch.randn(200, 1, 128, device="cuda").half()
    bare.write(0, x, x, s)
    assert bare.attend(0, x, s).isfinite().all()
    bare.settle()
    bare.fork([0], [1])
    bare.compact()
    bare.check()


def test_layers_beyond_one_launch_of_copies(cuda):
    """More tensors than one launch copies: every layer's page follows."""
    cache = kv.KVmixPagedCache([(2, 2)] * 140, 1, 128, 2, 256, 1, 3, 128, 256)
    s = cache.extend([0], [5])
    for l in range(140):
        x = torch.full((5, 1, 128), float(l), device="cuda").half()
        cache.write(l, x, -x, s)
    cache.fork([0], [1])
    page = int(cache.book.table[1, 0])
    assert page != int(cache.book.table[0, 0])
    for l in range(140):
        assert (cache.layers[l].kfull[page, 0, :5] == l).all() and (cache.layers[l].vfull[page, 0, :5] == -l).all()
    cache.check()


def test_two_streams_read_one_cache(cuda):
    """Attention changes nothing and shares nothing: calls over one cache may run at once."""
    cache = small()
    q = torch.randn(64, 1, 4, 128, device="cuda").half()
    at, row = ints(0, 1), ints(0)
    want = [kv.paged_attention(q[i], at, row, cache.book, cache.layers[0], max_tokens=1024) for i in range(64)]
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None] * 64
    torch.cuda.synchronize()
    for i in range(64):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = kv.paged_attention(q[i], at, row, cache.book, cache.layers[0], max_tokens=1024)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_steps_of_a_cache_lay_out_their_work(cuda):
    """A step's counts tell how many sequences have several tokens: more query heads a kv head than the kernel of few rows takes, chunks beside
    single tokens, and a chunk alone give what the calls without such hints give."""
    gen = torch.Generator().manual_seed(7)
    cache = kv.KVmixPagedCache([(4, 2)], 1, 128, 6, 600, 12, 24, 64, 128)
    for counts in ([200, 1, 300], [1, 1, 40], [1, 1, 1], [3, 0, 1], [50, 50, 50]):
        s = cache.extend([4, 0, 2], counts)
        k, v = (torch.randn(s.tokens, 1, 128, generator=gen).half().cuda() for _ in range(2))
        cache.write(0, k, v, s)
        for heads in (1, 4, 12):
            q = torch.randn(s.tokens, heads, 128, generator=gen).half().cuda()
            got, want = cache.attend(0, q, s), kv.paged_attention(q, s.q_start, s.rows, cache.book, cache.layers[0])
            # other splits sum in another order and may round a weight (2^-11) the other way
            assert ((got.float() - want.float()).norm(dim=-1) <= 2e-3 * want.float().norm(dim=-1)).all()
        cache.settle([4, 0, 2])
    cache.check()
