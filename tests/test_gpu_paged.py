"""The paged cache against a plain implementation in 64 bits: bookkeeping, packing, attention of single tokens and of chunks."""
import math

import numpy as np
import pytest
import torch

import kvmix_b200 as kv
from kvmix_b200 import paged

pytestmark = pytest.mark.gpu
P = 128


class Cache:
    """A cache filled directly (no calls of the framework): random packed pages and fp16 pages under shuffled numbers, pages that nobody
    holds full of NaN."""

    def __init__(self, lengths, packed, Hkv, kb, vb, group, seed=0, max_pages=None, slots=None, outliers=True):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.n_packed_of, self.Hkv = lengths, packed, Hkv
        pages = [-(-n // P) for n in lengths]
        n, n16 = sum(packed) + 2, sum(p - a for p, a in zip(pages, packed)) + 2
        slots = slots or len(lengths) + 1
        max_pages = max_pages or max(pages + [1])

        def packed_pool(bits):
            w, ng = paged.page_words(bits), paged.page_groups(bits, group)
            code = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, Hkv, P, w), generator=g, dtype=torch.int64).int()
            scale = (torch.rand(n, Hkv, P, ng, generator=g) * 2 + 0.5) / (2 ** bits - 1) * 2
            mn = -scale * (2 ** bits - 1) / 2 + 0.3 * torch.randn(n, Hkv, P, ng, generator=g)
            return code, scale.half(), mn.half()

        k, v = packed_pool(kb), packed_pool(vb)
        if outliers:
            for t in k[1:]:
                t[:, :, ::32] *= 4
        kf, vf = (torch.randn(n16, Hkv, P, 128, generator=g).half() for _ in range(2))
        perm, perm16 = torch.randperm(n, generator=g).tolist(), torch.randperm(n16, generator=g).tolist()
        rows = torch.randperm(slots, generator=g).tolist()[:len(lengths)]
        table = torch.full((slots, max_pages), -1, dtype=torch.int32)
        length, npk = torch.zeros(slots, dtype=torch.int32), torch.zeros(slots, dtype=torch.int32)
        for i, r in enumerate(rows):
            ids = [perm.pop() for _ in range(packed[i])] + [perm16.pop() for _ in range(pages[i] - packed[i])]
            table[r, :pages[i]] = torch.tensor(ids, dtype=torch.int32)
            length[r], npk[r] = lengths[i], packed[i]
            if lengths[i] % P and pages[i] > packed[i]:                     # behind the last token: whatever was there
                for t in (kf, vf):
                    t[ids[-1], :, lengths[i] % P:] = float("nan")
        for i in perm:
            for t in (*k[1:], *v[1:]):
                t[i] = float("nan")
        for i in perm16:
            kf[i], vf[i] = float("nan"), float("nan")
        free = torch.tensor(sorted(perm, reverse=True) + [0] * (n - len(perm)) + sorted(perm16, reverse=True) + [0] * (n16 - len(perm16)), dtype=torch.int32)
        refs = torch.ones(n + n16, dtype=torch.int32)
        refs[torch.tensor(perm + [n + i for i in perm16])] = 0
        self.kb, self.vb, self.group = kb, vb, group
        self.rows = torch.tensor(rows, dtype=torch.int32).cuda()
        self.host = dict(table=table, k=k, v=v, kf=kf, vf=vf, rows=rows)
        self.layer = kv.PageLayer(*(t.cuda() for t in k), kf.cuda(), *(t.cuda() for t in v), vf.cuda(), kb, vb, group)
        self.book = kv.PageBook(table.cuda(), length.cuda(), npk.cuda(), refs.cuda(), free.cuda(),
                                torch.tensor([len(perm), len(perm16), 0, 0], dtype=torch.int32).cuda(), n)

    def dense(self, i):
        """K, V [Hkv, length, 128] of sequence i in 64 bits."""
        h, a, n = self.host, self.n_packed_of[i], self.lengths[i]
        ids = h["table"][h["rows"][i]].tolist()
        out = []
        for side, full, bits, by_token in ((h["k"], h["kf"], self.kb, False), (h["v"], h["vf"], self.vb, True)):
            parts = []
            for j in range(-(-n // P)):
                if j < a:
                    x = unpack(*(t[ids[j]] for t in side), bits, self.group)
                    parts.append(x if by_token else x.transpose(0, 2, 1))
                else:
                    parts.append(full[ids[j]].double().numpy())
            out.append(np.concatenate(parts, 1)[:, :n] if parts else np.zeros((self.Hkv, 0, 128)))
        return out


def unpack(code, scale, mn, bits, group):
    """[.., words], [.., groups] x 2 -> [.., 128] in 64 bits."""
    c = code.numpy().astype(np.int64) & 0xffffffff
    fpi, size = (11, 11) if bits == 3 else (32 // bits, group)
    i = np.arange(P)
    f = (c[..., i // fpi] >> (bits * (i % fpi))) & (2 ** bits - 1)
    if bits == 3:
        f = np.where(i % 11 == 10, f & 3, f)
    return f * scale.double().numpy()[..., i // size] + mn.double().numpy()[..., i // size]


def plain(cache, q, counts, causal=True, window=0, prefix=None, first=None, softcap=0.0, slopes=None, scale=None):
    """Attention from its definition in 64 bits, and beside it a bound for the kernels' roundings (see tolerance())."""
    q = q.double().cpu().numpy()
    out, slack, at = np.zeros(q.shape), np.zeros(q.shape), 0
    scale = 1 / math.sqrt(128) if scale is None else scale
    rep = q.shape[1] // cache.Hkv
    for i, new in enumerate(counts):
        n = cache.lengths[i]
        K, V = cache.dense(i)
        for u in range(new):
            pos = n - new + u
            lo = max(0 if first is None else int(first[at + u]), pos + 1 - window if window else 0, 0)
            hi = n if not causal else min(n, max(pos + 1, 0 if prefix is None else int(prefix[i])))
            for h in range(q.shape[1]):
                if lo >= hi:
                    continue
                k, v = K[h // rep, lo:hi], V[h // rep, lo:hi]
                raw = k @ q[at + u, h]
                s = raw * scale
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                if slopes is not None:
                    s = s + float(slopes[h]) * (np.arange(lo, hi) - pos)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[at + u, h] = p @ v
                # each key element, weight and value element is rounded to fp16 once: half a step, 2^-11 relative (subnormals: 2^-25)
                eps = 2.0 ** -11
                ds = (np.abs(k) @ np.abs(q[at + u, h])) * abs(scale) * eps + 1e-5 * max(1.0, softcap) + np.abs(s) * 2e-6
                rel = ds + 2 * eps                                    # of a weight, and of a value
                slack[at + u, h] = 1.05 * ((p * rel) @ np.abs(v) + (p @ rel) * np.abs(out[at + u, h])) + eps * np.abs(out[at + u, h]) + 2.0 ** -24 * np.abs(v).sum(0) + 2.0 ** -24
        at += new
    return out, slack


def check(cache, q, counts, got, **opt):
    want, slack = plain(cache, q, counts, **opt)
    n = want.shape[0]
    err = np.abs(got[:n].double().cpu().numpy() - want)
    assert np.isfinite(err).all()
    worst = (err / np.maximum(slack, 1e-30)).max()
    assert worst <= 1.0, f"{worst:.2f} times the bound; largest error {err.max():.3e}"
    # the bound adds every rounding up; they hardly ever do: rows as a whole stay far below it
    norm = np.sqrt((want ** 2).sum(-1))
    row = np.sqrt((err ** 2).sum(-1)) / np.maximum(norm, 1e-3)
    assert row.max() <= 5e-3, f"row error {row.max():.3e}"


def starts(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32).cuda()


def queries(tokens, nh, seed=1):
    return torch.randn(tokens, nh, 128, generator=torch.Generator().manual_seed(seed)).half().cuda()


def attend(cache, q, counts, **opt):
    for k in ("prefix", "first"):
        if opt.get(k) is not None:
            opt[k] = torch.tensor(opt[k], dtype=torch.int32).cuda()
    if opt.get("slopes") is not None:
        opt["alibi_slopes"] = torch.tensor(opt.pop("slopes"), dtype=torch.float32).cuda()
    out = kv.paged_attention(q, starts(counts), cache.rows, cache.book, cache.layer, softmax_scale=opt.pop("scale", None), **opt)
    torch.cuda.synchronize()
    assert int(cache.book.count[2]) == 0
    return out


# ---- one new token ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kb", [1, 2, 3, 4])
@pytest.mark.parametrize("vb", [1, 2, 3, 4])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_one_token_bits(cuda, kb, vb, group):
    c = Cache([700, 300], [4, 1], 2, kb, vb, group, seed=kb * 16 + vb)
    q = queries(2, 8)
    check(c, q, [1, 1], attend(c, q, [1, 1]))


@pytest.mark.parametrize("length,packed", [(1, 0), (2, 0), (127, 0), (128, 0), (128, 1), (129, 1), (255, 1), (256, 2), (640, 5), (641, 3), (4300, 32), (9000, 70)])
@pytest.mark.parametrize("rep", [1, 2, 4, 5, 8])
def test_one_token_lengths(cuda, length, packed, rep):
    c = Cache([length], [packed], 2, 4, 2, 64, seed=length)
    q = queries(1, 2 * rep)
    check(c, q, [1], attend(c, q, [1]))


OPTIONS = [dict(window=1), dict(window=130), dict(window=128), dict(softcap=20.0), dict(softcap=2.0, window=300), dict(slopes=[0.25, 0.5, 0.01, 1.0]),
           dict(scale=0.3), dict(scale=-0.1), dict(causal=False), dict(slopes=[-0.01, 0.5, 0.01, 1.0], softcap=10.0)]


@pytest.mark.parametrize("opt", OPTIONS)
@pytest.mark.parametrize("kb,vb", [(2, 4), (3, 3)])
def test_one_token_options(cuda, opt, kb, vb):
    c = Cache([700, 301, 1], [4, 2, 0], 2, kb, vb, 32, seed=3)
    q = queries(3, 4)
    check(c, q, [1] * 3, attend(c, q, [1] * 3, **dict(opt)), **opt)


@pytest.mark.parametrize("counts", [[2, 1, 1], [1, 2, 2], [0, 2, 1]])
def test_few_tokens(cuda, counts):
    c = Cache([700, 301, 5], [4, 2, 0], 2, 2, 2, 64, seed=4)
    q = queries(sum(counts), 8)
    check(c, q, counts, attend(c, q, counts, max_new=2))


# ---- chunks ---------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("length,new,packed", [(3, 3, 0), (128, 128, 0), (300, 300, 0), (700, 3, 4), (700, 65, 5), (640, 64, 5), (1300, 129, 8), (700, 700, 0)])
@pytest.mark.parametrize("rep", [1, 4, 5])
def test_chunk_lengths(cuda, length, new, packed, rep):
    c = Cache([length], [packed], 1, 2, 4, 64, seed=length + new)
    q = queries(new, rep)
    check(c, q, [new], attend(c, q, [new]))


@pytest.mark.parametrize("kb", [1, 2, 3, 4])
@pytest.mark.parametrize("vb", [1, 2, 3, 4])
def test_chunk_bits(cuda, kb, vb):
    for group in (32, 128):
        c = Cache([430, 300], [2, 1], 2, kb, vb, group, seed=kb * 16 + vb)
        q = queries(60, 4)
        check(c, q, [40, 20], attend(c, q, [40, 20]))


@pytest.mark.parametrize("opt", OPTIONS + [dict(prefix=[690, 0, 3]), dict(first="blocks"), dict(first="nothing")])
def test_chunk_options(cuda, opt):
    counts = [100, 33, 4]
    c = Cache([700, 301, 4], [4, 2, 0], 2, 4, 2, 32, seed=3)
    opt = dict(opt)
    if opt.get("first") == "blocks":
        opt["first"] = [p // 47 * 47 for n, m in zip(c.lengths, counts) for p in range(n - m, n)]
    elif opt.get("first") == "nothing":                             # some rows see nothing: zeros
        opt["first"] = [p + 1 if p % 3 == 0 else 0 for n, m in zip(c.lengths, counts) for p in range(n - m, n)]
    q = queries(sum(counts), 4)
    check(c, q, counts, attend(c, q, counts, **dict(opt)), **opt)


@pytest.mark.parametrize("length,new,packed", [(2500, 130, 3), (2500, 130, 0), (3000, 300, 11), (2560, 2560, 0), (5000, 40, 20)])
def test_chunk_many_fp16_pages(cuda, length, new, packed):
    """Every buffer of the pipeline in use several times, and a last page that is not full."""
    c = Cache([length], [packed], 1, 4, 4, 32, seed=length)
    q = queries(new, 1)
    check(c, q, [new], attend(c, q, [new], window=2000), window=2000)


def test_mixed_step(cuda):
    counts = [1, 130, 1, 0, 7, 1]
    c = Cache([900, 500, 129, 77, 300, 1], [6, 2, 1, 0, 2, 0], 2, 3, 2, 128, seed=9)
    q = queries(sum(counts), 8)
    check(c, q, counts, attend(c, q, counts, max_new=130))


# ---- values and sizes at the edges ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("new,rep", [(1, 4), (1, 8), (60, 2)])
@pytest.mark.parametrize("kb,vb,group", [(2, 2, 32), (4, 1, 64), (3, 3, 128), (1, 4, 128)])
@pytest.mark.parametrize("k_size,v_size", [(1.0, 2e-4), (1e-3, 1.0), (1.0, 3e3), (600.0, 1.0), (1.0, 0.0)])
def test_large_and_small_values(cuda, new, rep, kb, vb, group, k_size, v_size):
    """Keys and values far from 1, constant ones (scales of zero) among them: scales and minima are multiplied, fp16 pages too.  Values below 1e-3
    are subnormal fp16: half a step there is 2^-25, which the bound carries."""
    c = Cache([500], [2], 1, kb, vb, group, seed=5, outliers=False)
    for side, full, size in ((c.host["k"], c.host["kf"], k_size), (c.host["v"], c.host["vf"], v_size)):
        for t in (*side[1:], full):
            t.mul_(size)
    c.layer = kv.PageLayer(*(t.cuda() for t in c.host["k"]), c.host["kf"].cuda(), *(t.cuda() for t in c.host["v"]), c.host["vf"].cuda(), kb, vb, group)
    q = queries(new, rep) / (k_size if k_size > 1 else 1.0)
    got, (want, slack) = attend(c, q, [new]), plain(c, q, [new])
    err = np.abs(got.double().cpu().numpy() - want)
    # of packed keys and values an element is code * scale + minimum rounded to fp16, or products rounded there: half a step of the smallest fp16
    # numbers, 2^-25, a term, and weights are scaled by 2^7 at most
    assert (err <= slack + 16 * 2.0 ** -24 * max(1.0, v_size)).all(), (err / slack).max()


def test_scales_that_grow_along_the_sequence(cuda):
    """p * scale is kept in fp16's range by a power of two that follows the largest scale: pages whose scales grow 2^24 fold, and fall again."""
    c = Cache([128 * 13], [13], 1, 2, 2, 64, seed=8, outliers=False)
    ids = c.host["table"][c.host["rows"][0]].tolist()
    for j, i in enumerate(ids):
        for t in c.host["v"][1:]:
            t[i] *= 2.0 ** (-12 + 2 * min(j, 24 - 2 * j if j > 8 else j))
    c.layer = c.layer._replace(vscale=c.host["v"][1].cuda(), vmn=c.host["v"][2].cuda())
    for nh in (1, 2, 4, 8):
        q = queries(1, nh)
        check(c, q, [1], attend(c, q, [1]))


@pytest.mark.parametrize("what", ["nan key", "inf value", "nan query"])
@pytest.mark.parametrize("new", [1, 200])
def test_not_finite(cuda, what, new):
    """A key or query that is not finite is seen by every query that sees it, and by none that sees no token of its page.  A value that is not
    may besides reach queries of the same tile: 64 tokens of 4 heads, so that of the chunk 500 .. 699 the tokens from 628 on share theirs with 670."""
    c = Cache([700], [0], 1, 4, 4, 64, seed=2)
    ids = c.host["table"][c.host["rows"][0]].tolist()
    q = queries(new, 4)
    if what == "nan key":
        c.layer.kfull[ids[5], 0, 30, 7] = float("nan")              # position 670
    elif what == "inf value":
        c.layer.vfull[ids[5], 0, 30, 7] = float("inf")
    else:
        q[0, 1, 3] = float("nan")
    out = attend(c, q, [new])
    if what == "nan query":
        assert out[0, 1].isnan().all() and out[:, [0, 2, 3]].isfinite().all() and out[1:].isfinite().all()
        return
    pos = torch.arange(700 - new, 700, device="cuda")
    bad = ~out.isfinite()
    assert bad[pos >= 670].any(-1).all()
    assert not bad[pos < (628 if what == "inf value" else 640)].any()
    far = attend(c, q, [new], first=[640 if p < 640 else 0 for p in pos.tolist()]) if new > 1 else out
    assert not far[pos < 628].any()                                  # they see nothing


def test_masked_keys_of_any_value_do_not_matter(cuda):
    """Keys behind a mask may be anything: NaN, infinities, the lowest number."""
    c = Cache([700], [3], 1, 2, 2, 64, seed=12)
    q1, q = queries(1, 4), queries(100, 4)
    want1, want = attend(c, q1, [1], window=200), attend(c, q, [100], window=200)
    ids = c.host["table"][c.host["rows"][0]].tolist()
    for j, bad in ((0, float("nan")), (1, float("inf")), (2, -65504.0)):
        c.layer.kmn[ids[j]] = bad                                    # positions below 384 are seen by nobody (700 - 100 - 200 = 400)
    c.layer.kfull[ids[3], :, :16] = float("nan")
    got1, got = attend(c, q1, [1], window=200), attend(c, q, [100], window=200)
    assert torch.equal(got1, want1) and torch.equal(got, want)


@pytest.mark.parametrize("rep,new", [(1, 1), (4, 1), (3, 40)])
def test_odd_layouts_of_queries_and_outputs(cuda, rep, new):
    c = Cache([300], [2], 2, 4, 2, 64, seed=21)
    nh = 2 * rep
    want = attend(c, queries(new, nh), [new])
    flat = torch.zeros(new * nh * 131 + 3, dtype=torch.half, device="cuda")
    q = flat[3:].view(new, nh, 131)[..., 1:129]                      # rows that begin at any fp16
    q.copy_(queries(new, nh))
    out = torch.full((new, nh + 1, 137), 5.0, dtype=torch.half, device="cuda")
    got = attend(c, q, [new], out=out[:, :nh, 3:131])
    assert torch.equal(got, want)
    assert (out[:, nh] == 5).all() and (out[:, :, :3] == 5).all() and (out[:, :, 131:] == 5).all()
    wide = torch.zeros(new, nh, 256, dtype=torch.half, device="cuda")
    wide[..., ::2] = queries(new, nh)                                # channels two apart
    assert torch.equal(attend(c, wide[..., ::2], [new]), want)


def test_no_work(cuda):
    c = Cache([300, 5], [2, 0], 1, 4, 2, 64)
    assert attend(c, queries(0, 4), [0, 0]).shape == (0, 4, 128)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    out = torch.full((3, 4, 128), 9.0, dtype=torch.half, device="cuda")
    kv.paged_attention(queries(3, 4), torch.zeros(1, dtype=torch.int32, device="cuda"), none, c.book, c.layer, out=out)
    assert (out == 9).all()
    out = attend(c, queries(2, 4), [0, 0], out=torch.full((2, 4, 128), 9.0, dtype=torch.half, device="cuda"))
    assert (out == 9).all()


@pytest.mark.parametrize("splits", [dict(max_tokens=640), dict(max_tokens=1), dict(), dict(max_new=1)])
def test_hints_lay_out_the_work_only(cuda, splits):
    """max_tokens below a sequence's length, or none given: other splits, the same sums."""
    c = Cache([5000, 640], [30, 4], 1, 2, 4, 64, seed=31, max_pages=60)
    q = queries(2, 4)
    check(c, q, [1, 1], attend(c, q, [1, 1], **splits))
    if "max_new" not in splits:
        q = queries(50, 4)
        check(c, q, [30, 20], attend(c, q, [30, 20], **splits))


def test_many_sequences(cuda):
    """More sequences than a CTA has threads, most of them one token long."""
    g = torch.Generator().manual_seed(3)
    lengths = [int(n) for n in torch.randint(1, 4, (2500,), generator=g)]
    lengths[1700], lengths[2499] = 300, 129
    c = Cache(lengths, [2 if n == 300 else 1 if n == 129 else 0 for n in lengths], 1, 4, 2, 64, seed=33)
    q = queries(2500, 2)
    check(c, q, [1] * 2500, attend(c, q, [1] * 2500, max_new=1))


def test_pages_beyond_32_bits(cuda):
    """Numbers of pages whose elements lie beyond 2^32: the first and the last of a pool of 8.6 GB."""
    n16, heads = 16500, 16                                           # 16500 * 16 * 16384 elements a tensor
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    g = torch.Generator().manual_seed(4)
    small = Cache([200], [0], heads, 2, 2, 128, seed=40)
    ids = small.host["table"][small.host["rows"][0]].tolist()
    kf, vf = (torch.empty(n16, heads, P, 128, dtype=torch.half, device="cuda") for _ in range(2))
    to = [n16 - 1, 0]
    for i, j in zip(ids, to):
        kf[j], vf[j] = small.layer.kfull[i], small.layer.vfull[i]
    layer = small.layer._replace(kfull=kf, vfull=vf)
    book = kv.PageBook(small.book.table.clone(), small.book.length, small.book.packed, torch.ones(small.book.n_packed + n16, dtype=torch.int32, device="cuda"),
                       torch.zeros(small.book.n_packed + n16, dtype=torch.int32, device="cuda"), small.book.count, small.book.n_packed)
    book.table[small.host["rows"][0], :2] = torch.tensor(to, dtype=torch.int32, device="cuda")
    for new in (1, 150):
        q = torch.randn(new, 2 * heads, 128, generator=g).half().cuda()
        got = kv.paged_attention(q, starts([new]), small.rows, book, layer)
        assert torch.equal(got, kv.paged_attention(q, starts([new]), small.rows, small.book, small.layer))
    x, y = (torch.randn(150, heads, 128, generator=g).half().cuda() for _ in range(2))
    kv.page_write(x, y, starts([150]), small.rows, book, layer)      # positions 50 .. 199
    assert torch.equal(kf[n16 - 1, :, 50:], x[:78].transpose(0, 1)) and torch.equal(vf[0, :, :72], y[78:].transpose(0, 1))


@pytest.mark.parametrize("n,chunks", [(9, [8]), (900, [0, 767, 768, 899]), (1600, [1599])])
def test_few_chunks_among_many_sequences(cuda, n, chunks):
    """The tile kernel finds its sequences among single tokens, with and without being told how many there are."""
    lengths, counts = [3] * n, [1] * n
    for i in chunks:
        lengths[i], counts[i] = 270, 90
    c = Cache(lengths, [1 if m == 270 else 0 for m in lengths], 1, 4, 2, 64, seed=n)
    q = queries(sum(counts), 4)
    got = attend(c, q, counts, max_new=90, max_chunks=len(chunks))
    check(c, q, counts, got)
    assert torch.equal(attend(c, q, counts, max_new=90), got)


def test_weights_on_values_of_a_small_scale(cuda):
    """Pages of large values whose weights are next to nothing before pages of small ones that have them: the small ones keep their precision."""
    c = Cache([128 * 6], [6], 1, 4, 2, 64, seed=14, outliers=False)
    ids = c.host["table"][c.host["rows"][0]].tolist()
    for j, i in enumerate(ids):
        for t in c.host["v"][1:]:
            t[i] *= 2.0 ** (6 if j < 4 else -8)
    c.layer = c.layer._replace(vscale=c.host["v"][1].cuda(), vmn=c.host["v"][2].cuda())
    slopes = [0.25] * 4                                              # positions 256 and more away: 2^-92
    q = queries(1, 4)
    got, (want, _) = attend(c, q, [1], slopes=slopes), plain(c, q, [1], slopes=slopes)
    err = np.abs(got.double().cpu().numpy() - want)
    # keys are exact to 2^-20; a weight, its product with a scale and the output are rounded once each (the minima's products share the weight's):
    # 3 * 2^-11 of codes and minima, which are up to 4 times the values here
    assert err.max() <= 3 * 2.0 ** -11 * 4 * 2.0 ** -8 * 2, err.max()
