"""Appending to the paged cache with the rotation on the way: pages and queries against the rotation in 64 bits, tokens that have no place or no
angles, layouts, other streams, captured calls, refusals."""
import pytest
import torch

import kvmix_b200 as kv

pytestmark = pytest.mark.gpu
P = 128


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def tables(rows, angles, gen, wide=0):
    t = torch.rand(rows, angles, generator=gen, dtype=torch.float64) * 6.283
    c, s = t.cos().float().cuda(), t.sin().float().cuda()
    if wide:                                                     # rows further apart than they are long
        c, s = (torch.cat([x, torch.full((rows, wide), float("nan"), device="cuda")], 1)[:, :angles] for x in (c, s))
    return c, s


def turned(x, cos, sin, parts, interleaved):
    """The rotation in 64 bits, and what fp32 products and sums and one rounding to fp16 may be off by."""
    x = x.double()
    y, bound = x.clone(), torch.zeros_like(x)
    size, angles = 128 // parts, cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    for p in range(parts):
        i = torch.arange(angles, device=x.device)
        a, b = (p * size + 2 * i, p * size + 2 * i + 1) if interleaved else (p * size + i, p * size + angles + i)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        # two products and a sum, each rounded at most once, by 2^-24 of sizes that |x c| + |y s| bounds
        bound[..., a] = 2 * 2.0 ** -24 * ((x[..., a] * c).abs() + (x[..., b] * s).abs())
        bound[..., b] = 2 * 2.0 ** -24 * ((x[..., b] * c).abs() + (x[..., a] * s).abs())
    # half a step of fp16, 2^-25 below its normal numbers
    return y, bound * 1.01 + torch.maximum((y.abs() + bound) * 2.0 ** -11, torch.full_like(y, 2.0 ** -25))


class Case:
    def __init__(self, past, new, heads=4, kv_heads=2, kind=torch.float16, angles=64, parts=1, seed=0, behind=0, wide=0, max_tokens=1024, size=1.0):
        self.gen = torch.Generator().manual_seed(seed)
        n = len(new)
        self.cache = kv.KVmixPagedCache([(4, 2)], kv_heads, 128, n + 1, max_tokens, 8, 16 + (max_tokens // 100) * n, 64)
        self.rows = torch.randperm(n + 1, generator=self.gen).tolist()[:n]
        self.cache.extend(self.rows, past)
        for t in (self.cache.layers[0].kfull, self.cache.layers[0].vfull):
            t.fill_(float("nan"))
        self.step = self.cache.extend(self.rows, new)
        tokens = self.step.tokens + behind
        self.k, self.v, self.q = ((torch.randn(tokens, h, 128, generator=self.gen) * size).to(kind).cuda() for h in (kv_heads, kv_heads, heads))
        self.cos, self.sin = tables(max_tokens, angles, self.gen, wide)
        self.pos = torch.cat([torch.arange(p, p + c) for p, c in zip(past, new)]).cuda() if sum(new) else torch.zeros(0, dtype=torch.long, device="cuda")
        self.seq = sum([[r] * c for r, c in zip(self.rows, new)], [])

    def call(self, **options):
        return kv.page_append(self.k, self.v, self.cos, self.sin, self.step.q_start, self.step.rows, self.cache.book, self.cache.layers[0], **options)

    def holds(self, angle_at=None, parts=1, interleaved=False, skip=()):
        """Every page's tokens are these, and nothing else has been written."""
        at = self.pos if angle_at is None else angle_at
        n = self.pos.numel()
        k, bound = turned(self.k[:n], self.cos[at], self.sin[at], parts, interleaved)
        layer, table = self.cache.layers[0], self.cache.book.table.long()
        rows = torch.tensor(self.seq, device="cuda", dtype=torch.long)
        page, slot = table[rows, self.pos // P], self.pos % P
        keep = torch.tensor([i not in skip for i in range(n)], device="cuda", dtype=torch.bool)
        got = layer.kfull[page, :, slot].double()
        assert ((got - k).abs() <= bound)[keep].all()
        assert torch.equal(layer.vfull[page, :, slot][keep], self.v[:n].half()[keep])
        there = torch.zeros(layer.kfull.shape[0], P, dtype=torch.bool, device="cuda")
        there[page[keep], slot[keep]] = True
        assert layer.kfull.transpose(1, 2)[~there].isnan().all() and layer.vfull.transpose(1, 2)[~there].isnan().all()


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("angles,parts,interleaved", [(64, 1, False), (64, 1, True), (8, 1, False), (40, 1, True), (24, 1, False), (32, 2, False), (16, 2, True), (8, 2, False)])
def test_rotation(cuda, kind, angles, parts, interleaved):
    past, new = [0, 127, 300, 5, 256], [130, 1, 64, 0, 128]
    c = Case(past, new, kind=kind, angles=angles, parts=parts, seed=angles + parts)
    got = c.call(q=c.q, interleaved=interleaved, parts=parts)
    want, bound = turned(c.q, c.cos[c.pos], c.sin[c.pos], parts, interleaved)
    assert got.dtype is torch.float16 and ((got.double() - want).abs() <= bound).all()
    c.holds(parts=parts, interleaved=interleaved)
    c.cache.check()


@pytest.mark.parametrize("heads,kv_heads,new", [(1, 1, [1]), (32, 8, [1] * 40), (40, 8, [700, 1, 3]), (8, 1, [129]), (5, 5, [0, 1, 0])])
def test_head_layouts(cuda, heads, kv_heads, new):
    c = Case([(37 * i) % 260 for i in range(len(new))], new, heads, kv_heads, seed=heads)
    got = c.call(q=c.q)
    want, bound = turned(c.q, c.cos[c.pos], c.sin[c.pos], 1, False)
    assert ((got.double() - want).abs() <= bound).all()
    c.holds()


@pytest.mark.parametrize("heads,kv_heads", [(0, 1), (1, 1), (2, 1), (7, 3), (33, 1), (31, 2), (100, 20), (6, 5), (64, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rows_of_a_token(cuda, heads, kv_heads, interleaved):
    """Any number of rows a token: places that are left empty, several tokens at once, several turns."""
    for new in ([3], [37, 1, 90], [400]):
        c = Case([11 * i for i in range(len(new))], new, max(heads, 1), kv_heads, seed=heads + kv_heads, behind=2)
        if heads == 0:
            assert c.call(interleaved=interleaved) is None
            assert c.call(interleaved=interleaved, q=c.q[:, :0]).shape == (sum(new) + 2, 0, 128)
        else:
            out = torch.full(c.q.shape, 7.0, dtype=torch.float16, device="cuda")
            c.call(q=c.q, q_out=out, interleaved=interleaved)
            n = sum(new)
            want, bound = turned(c.q[:n], c.cos[c.pos], c.sin[c.pos], 1, interleaved)
            assert ((out[:n].double() - want).abs() <= bound).all() and (out[n:] == 7).all()
        c.holds(interleaved=interleaved)


def test_many_tokens(cuda):
    """Several tokens a place of a CTA: more than 148 * 8 * 4 tokens."""
    c = Case([0, 200], [9001, 3000], 2, 1, seed=14, max_tokens=9100)
    got = c.call(q=c.q)
    want, bound = turned(c.q, c.cos[c.pos], c.sin[c.pos], 1, False)
    assert ((got.double() - want).abs() <= bound).all()
    c.holds()


@pytest.mark.parametrize("kind", [torch.float16, torch.float32])
def test_layouts(cuda, kind):
    """Rows that are not 16-byte aligned, heads before tokens, channels apart, tables with rows apart, queries in place."""
    for how in range(5):
        c = Case([100, 3], [60, 300], kind=kind, seed=how, wide=3 if how == 3 else 4)
        if how == 0:
            c.k, c.v, c.q = (torch.cat([torch.zeros_like(t[..., :3]), t], -1)[..., 3:] for t in (c.k, c.v, c.q))
        elif how == 1:
            c.k, c.v, c.q = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (c.k, c.v, c.q))
        elif how == 2:
            c.k, c.v, c.q = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.k, c.v, c.q))
        want, bound = turned(c.q, c.cos[c.pos], c.sin[c.pos], 1, False)
        out = None
        if how == 4 and kind is torch.float16:
            out = c.q
        elif how == 1:
            out = torch.empty(c.q.shape[1], c.q.shape[0], 131, dtype=torch.float16, device="cuda").transpose(0, 1)[..., 1:129]
        got = c.call(q=c.q, q_out=out)
        assert out is None or got is out
        assert ((got.double() - want).abs() <= bound).all()
        c.holds()


def test_no_angle_turns_nothing(cuda):
    """With angles of zero the pages are those of page_write, bit for bit."""
    c = Case([100, 0], [50, 129], seed=3)
    other = Case([100, 0], [50, 129], seed=3)
    c.cos.fill_(1.0)
    c.sin.fill_(0.0)
    assert c.call() is None
    kv.page_write(other.k, other.v, other.step.q_start, other.step.rows, other.cache.book, other.cache.layers[0])
    for a, b in zip((c.cache.layers[0].kfull, c.cache.layers[0].vfull), (other.cache.layers[0].kfull, other.cache.layers[0].vfull)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_values_that_are_no_numbers(cuda):
    c = Case([5], [4], kind=torch.float32, seed=4)
    c.v[0, 0, 3], c.v[1, 1, 5], c.v[2, 0, 0], c.k[1, 0, 0] = float("nan"), float("inf"), 1e6, 1e6
    c.cos.fill_(1.0)
    c.sin.fill_(0.0)
    c.call()
    page = int(c.cache.book.table[c.rows[0], 0])
    k, v = c.cache.layers[0].kfull[page], c.cache.layers[0].vfull[page]
    assert v[0, 5, 3].isnan() and v[1, 6, 5] == float("inf") and v[0, 7, 0] == float("inf") and k[0, 6, 0] == float("inf")       # beyond fp16: infinity


def test_positions_of_the_callers(cuda):
    c = Case([100, 20], [30, 140], seed=5)
    at = torch.randint(0, 1024, (170,), generator=c.gen)
    got = c.call(q=c.q, positions=at.int().cuda())
    want, bound = turned(c.q, c.cos[at.cuda()], c.sin[at.cuda()], 1, False)
    assert ((got.double() - want).abs() <= bound).all()
    c.holds(angle_at=at.cuda())


def test_positions_outside_the_tables(cuda):
    for given in (False, True):
        c = Case([100, 0], [30, 20], seed=6)
        if given:
            at = torch.arange(50)
            at[3], at[40], at[41] = -1, 1024, 2 ** 31 - 1
            skip, options = {3, 40, 41}, dict(positions=at.int().cuda())
            at = at.clamp(0, 1023).cuda()
        else:
            c.cos, c.sin = c.cos[:110].contiguous(), c.sin[:110].contiguous()
            skip, options, at = set(range(10, 30)), {}, c.pos.clamp(max=109)
        out = torch.full(c.q.shape, float("nan"), dtype=torch.float16, device="cuda")
        c.call(q=c.q, q_out=out, **options)
        gone = torch.tensor(sorted(skip), device="cuda")
        assert out[gone].isnan().all() and int(out.isnan().sum()) == gone.numel() * 4 * 128
        c.holds(angle_at=at, skip=skip)
        with pytest.raises(RuntimeError, match="outside the tables"):
            c.cache.check()
        c.call(q=c.q)                                            # the bit held nothing up
        assert int(c.cache.book.count[2]) in (0, 64)


def test_tokens_without_a_place(cuda):
    """Pages that are packed or shared are not written; queries are rotated all the same."""
    c = Case([0, 256], [256, 128], seed=7)
    c.call()
    before = [t.clone() for t in c.cache.layers[0][:8]]
    c.cache.settle([c.rows[0]])
    free = [r for r in range(3) if r not in c.rows][0]
    c.cache.fork([c.rows[1]], [free])
    packed = [t.clone() for t in c.cache.layers[0][:3]]
    out = c.call(q=c.q)
    want, bound = turned(c.q, c.cos[c.pos], c.sin[c.pos], 1, False)
    assert ((out.double() - want).abs() <= bound).all()
    last = int(c.cache.book.table[c.rows[0], 1])
    for i in (3, 7):                                             # the second page of the first sequence is its own, the rest is as it was
        a, b = before[i].clone(), c.cache.layers[0][i].clone()
        a[last], b[last] = 0, 0
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    assert all(torch.equal(a.view(torch.int16 if a.dtype is torch.float16 else torch.int32), b.view(torch.int16 if b.dtype is torch.float16 else torch.int32))
               for a, b in zip(packed, c.cache.layers[0][:3]))
    with pytest.raises(RuntimeError, match="not written"):
        c.cache.check()


def test_rows_behind_the_last_sequence_stay(cuda):
    c = Case([10], [5], seed=8, behind=3)
    out = torch.full(c.q.shape, 7.0, dtype=torch.float16, device="cuda")
    c.call(q=c.q, q_out=out)
    assert (out[5:] == 7).all() and not (out[:5] == 7).all(-1).any()
    c.holds()


@pytest.mark.parametrize("start", [[0, 2 ** 31 - 1], [-5, 3], [4, 2], [-2 ** 31, 2 ** 31 - 1], [0, 9]])
def test_wrong_numbers_of_new_tokens_stay_inside(cuda, start):
    c = Case([10], [5], seed=9)
    untouched = c.cache.layers[0].kfull.clone()
    kv.page_append(c.k, c.v, c.cos, c.sin, ints(*start), c.step.rows, c.cache.book, c.cache.layers[0], q=c.q)
    page = int(c.cache.book.table[c.rows[0], 0])
    others = [i for i in range(untouched.shape[0]) if i != page]
    assert c.cache.layers[0].kfull[others].isnan().all()


@pytest.mark.parametrize("what,value", [("table", 10 ** 6), ("table", -7), ("length", 2 ** 31 - 1), ("length", -5), ("packed", 2 ** 31 - 1), ("packed", -3), ("rows", 99), ("rows", -1)])
def test_wrong_bookkeeping_stays_inside(cuda, what, value):
    c = Case([100], [50], seed=10)
    if what == "rows":
        c.step = c.step._replace(rows=ints(value))
    else:
        getattr(c.cache.book, what).fill_(value)
    c.call(q=c.q)
    torch.cuda.synchronize()


def test_more_sequences_than_are_staged(cuda):
    n = 1500
    gen = torch.Generator().manual_seed(11)
    cache = kv.KVmixPagedCache([(2, 2)], 1, 128, n, 128, 1, n, 64)
    new = [i % 3 for i in range(n)]
    step = cache.extend(list(range(n)), new)
    k, v, q = (torch.randn(step.tokens, h, 128, generator=gen).half().cuda() for h in (1, 1, 2))
    cos, sin = tables(128, 64, gen)
    got = cache.append(0, k, v, cos, sin, step, q=q)
    pos = torch.cat([torch.arange(c) for c in new]).cuda()
    want, bound = turned(q, cos[pos], sin[pos], 1, False)
    assert ((got.double() - want).abs() <= bound).all()
    want, bound = turned(k, cos[pos], sin[pos], 1, False)
    page = cache.book.table[torch.tensor(sum([[i] * c for i, c in enumerate(new)], [])).cuda(), 0].long()
    assert ((cache.layers[0].kfull[page, :, pos].double() - want).abs() <= bound).all()
    cache.check()


def test_on_another_stream_and_captured(cuda):
    a, b = Case([100, 3], [1, 1], seed=12), Case([100, 3], [1, 1], seed=12)
    want = a.call(q=a.q)
    stream, out = torch.cuda.Stream(), torch.empty_like(b.q)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        b.call(q=b.q, q_out=out)
    stream.synchronize()
    assert torch.equal(out, want)
    b.cache.layers[0].kfull.fill_(float("nan"))
    out.zero_()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        b.call(q=b.q, q_out=out)
    for scale in (1, 2):
        a.q.mul_(scale)
        b.q.mul_(scale)
        want = a.call(q=a.q)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(a.cache.layers[0].kfull.view(torch.int16), b.cache.layers[0].kfull.view(torch.int16))


def test_nothing_to_do_and_refused_calls(cuda):
    c = Case([10], [5], seed=13)
    for t in ("k", "v", "q"):
        setattr(c, "full_" + t, getattr(c, t))
    empty = kv.page_append(c.k[:0], c.v[:0], c.cos, c.sin, ints(0), c.step.rows[:0], c.cache.book, c.cache.layers[0], q=c.q[:0])
    assert empty.shape == (0, 4, 128)
    c.cache.book.count[2] = 1                                    # another call was refused: nothing is written
    c.call(q=c.q)
    assert c.cache.layers[0].kfull.isnan().all()
    c.cache.book.count[2] = 0
    bad = [dict(k=c.k.double()), dict(v=c.v.float()), dict(k=c.k[:, :1]), dict(k=c.k[..., :64]), dict(q=c.q.float()), dict(q=c.q[:3]), dict(q=c.q[..., :64]), dict(cos=c.cos.half()),
           dict(cos=c.cos[:, :12], sin=c.sin[:, :12]), dict(cos=c.cos[:, :0], sin=c.sin[:, :0]), dict(sin=c.sin[:100]), dict(parts=2), dict(parts=3), dict(positions=c.pos),
           dict(positions=c.pos.int()[:3]), dict(q_out=c.q), dict(q=c.q, q_out=c.q.float()), dict(q=c.q, q_out=c.q[:, :1].expand(-1, 4, -1)), dict(k=c.k.cpu()), dict(cos=c.cos.cpu()),
           dict(cos=torch.cat([c.cos, c.cos], 1), sin=torch.cat([c.sin, c.sin], 1)), dict(cos=c.cos.t().contiguous().t())]
    for change in bad:
        args = dict(k=c.k, v=c.v, cos=c.cos, sin=c.sin, q_start=c.step.q_start, rows=c.step.rows, pages=c.cache.book, layer=c.cache.layers[0])
        args.update(change)
        with pytest.raises(RuntimeError):
            kv.page_append(**args)
    with pytest.raises(RuntimeError, match="angles for"):
        c.cache.append(0, c.k, c.v, c.cos[:14], c.sin[:14], c.step)
    with pytest.raises(RuntimeError, match="every new token"):
        c.cache.append(0, c.k[:4], c.v[:4], c.cos, c.sin, c.step)
    assert c.cache.layers[0].kfull.isnan().all()
