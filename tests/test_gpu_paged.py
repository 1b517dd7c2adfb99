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
