"""Differential attention over the paged cache against its definition in 64 bits, and a search that appends, attends and reorders."""
import math

import numpy as np
import pytest
import torch

import kvmix_b200 as kv
from test_gpu_paged import P, Cache, plain, queries, starts
from test_gpu_paged_book import ints

pytestmark = pytest.mark.gpu
NORM = torch.linspace(0.5, -1.5, 128)


def definition(cache, q, lambdas, counts, norm_weight=None, norm_eps=1e-5, scale=0.125, **opt):
    """The two maps are attentions of one half of the channels each, with the bound of their roundings; a difference adds the bounds up and is rounded
    once; a norm passes a change of its input on, and that of the row's size."""
    zero = torch.zeros_like(q)
    first, second = zero.clone(), zero.clone()
    first[..., :64], second[..., 64:] = q[..., :64], q[..., 64:]
    (a, da), (b, db) = (plain(cache, x, counts, scale=scale, **opt) for x in (first, second))
    lam = lambdas.double().cpu().numpy()[:, None]
    out, slack = a - lam * b, da + np.abs(lam) * db + 2.0 ** -22 * (np.abs(a) + np.abs(lam * b))
    size = np.sqrt((a ** 2).sum(-1)) + np.abs(lam[:, 0]) * np.sqrt((b ** 2).sum(-1))
    if norm_weight is not None:
        w, by = norm_weight.double().cpu().numpy(), 1 / np.sqrt((out ** 2).mean(-1, keepdims=True) + norm_eps)
        grow = (np.abs(out) * slack).mean(-1, keepdims=True) * by ** 2
        slack = np.abs(w) * by * 1.1 * (slack + np.abs(out) * grow) + 2.0 ** -20 * np.abs(w * by * out)
        size, out = size * by[..., 0] * np.abs(w).max(), out * by * w
    # two more steps of the maps' own output rounding are in `slack` already where it is not normed
    return out, slack + 2.0 ** -11 * np.abs(out) + 2.0 ** -24, size


def call(cache, q, lambdas, counts, check_status=True, **opt):
    for k in ("prefix", "first"):
        if opt.get(k) is not None:
            opt[k] = torch.tensor(opt[k], dtype=torch.int32).cuda()
    if opt.get("slopes") is not None:
        opt["alibi_slopes"] = torch.tensor(opt.pop("slopes"), dtype=torch.float32).cuda()
    out = kv.paged_differential_attention(q, lambdas, starts(counts), cache.rows, cache.book, cache.layer, softmax_scale=opt.pop("scale", None), **opt)
    torch.cuda.synchronize()
    assert not check_status or int(cache.book.count[2]) == 0
    return out


def check(cache, q, counts, lambdas=None, hints=None, **opt):
    lambdas = torch.linspace(0.1, 0.9, q.shape[1]).cuda() if lambdas is None else lambdas
    got = call(cache, q, lambdas, counts, **dict(opt, **(hints or {})))
    want, slack, size = definition(cache, q, lambdas, counts, **opt)
    n = want.shape[0]
    err = np.abs(got[:n].double().cpu().numpy() - want)
    assert np.isfinite(err).all()
    worst = (err / slack).max()
    assert worst <= 1.0, f"{worst:.2f} times the bound; largest error {err.max():.3e}"
    # the bound adds every rounding up; rows as a whole stay far below it
    row = np.sqrt((err ** 2).sum(-1)) / np.maximum(size, 1e-3)
    assert row.max() <= 5e-3, f"row error {row.max():.3e}"
    return got


# ---- one new token ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kb", [1, 2, 3, 4])
@pytest.mark.parametrize("vb", [1, 2, 3, 4])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_one_token_bits(cuda, kb, vb, group):
    for rep in (1, 2, 4):
        c = Cache([900, 128, 515], [6, 1, 3], 2, kb, vb, group, seed=kb + vb + rep)
        check(c, queries(3, 2 * rep, rep), [1, 1, 1], norm_weight=NORM.cuda() if rep == 2 else None)


@pytest.mark.parametrize("length,packed", [(1, 0), (2, 0), (127, 0), (128, 1), (129, 1), (257, 2), (1025, 8), (2300, 0), (3000, 20)])
@pytest.mark.parametrize("rep", [1, 3, 4])
def test_one_token_lengths(cuda, length, packed, rep):
    c = Cache([length], [packed], 2, 4, 2, 64, seed=length)
    check(c, queries(1, 2 * rep), [1], norm_weight=NORM.cuda())
    check(c, queries(1, 2 * rep), [1])


OPTIONS = [dict(window=100), dict(window=1), dict(prefix=[700]), dict(softcap=5.0), dict(slopes=[0.1, 0.02, 0.5, 0.0]), dict(causal=False), dict(scale=-0.2), dict(first=[300]),
           dict(window=300, softcap=20.0, slopes=[0.01, 0.3, 0.0, 0.1]), dict(scale=0.0)]


@pytest.mark.parametrize("opt", OPTIONS)
@pytest.mark.parametrize("kb,vb", [(4, 2), (3, 3)])
def test_one_token_options(cuda, opt, kb, vb):
    check(Cache([700], [5], 1, kb, vb, 64, seed=3), queries(1, 4), [1], **opt)
    check(Cache([700], [5], 1, kb, vb, 32, seed=3), queries(1, 4), [1], norm_weight=NORM.cuda(), **opt)


@pytest.mark.parametrize("counts", [[2, 1, 0, 1], [4, 4, 1, 3], [0, 0, 0, 1]])
def test_few_tokens(cuda, counts):
    c = Cache([300, 40, 9, 513], [1, 0, 0, 4], 2, 2, 4, 64, seed=5)
    check(c, queries(sum(counts), 2), counts)
    check(c, queries(sum(counts), 2), counts, norm_weight=NORM.cuda(), norm_eps=0.0)


# ---- chunks ----------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("length,new,packed", [(9, 9, 0), (128, 128, 1), (129, 129, 0), (300, 200, 0), (700, 129, 4), (1000, 65, 7), (640, 128, 5), (700, 300, 2)])
@pytest.mark.parametrize("rep", [1, 4, 5])
def test_chunk_lengths(cuda, length, new, packed, rep):
    c = Cache([length], [packed], 1, 2, 4, 64, seed=length + rep)
    check(c, queries(new, rep), [new], norm_weight=NORM.cuda() if rep == 4 else None)


@pytest.mark.parametrize("kb", [1, 2, 3, 4])
@pytest.mark.parametrize("vb", [1, 2, 3, 4])
def test_chunk_bits(cuda, kb, vb):
    for group in (32, 64, 128):
        c = Cache([420], [3], 2, kb, vb, group, seed=kb * vb + group)
        check(c, queries(40, 4, group), [40], norm_weight=NORM.cuda() if group == 64 else None)


@pytest.mark.parametrize("opt", [dict(o) for o in OPTIONS if "first" not in o and "prefix" not in o] + [dict(prefix=[330]), dict(prefix=[10 ** 6])])
def test_chunk_options(cuda, opt):
    check(Cache([420], [2], 1, 4, 2, 64, seed=7), queries(150, 4), [150], norm_weight=NORM.cuda(), **opt)


@pytest.mark.parametrize("rep", [5, 8])
def test_many_heads_of_a_kv_head(cuda, rep):
    """One new token of more than four query heads a kv head is the tile kernel's."""
    c = Cache([500, 1, 260], [3, 0, 1], 2, 3, 2, 128, seed=rep)
    check(c, queries(3, 2 * rep), [1, 1, 1], norm_weight=NORM.cuda())


def test_mixed_step(cuda):
    counts = [1, 130, 0, 1, 33, 2]
    c = Cache([400, 600, 50, 1, 33, 1300], [2, 3, 0, 0, 0, 9], 2, 4, 2, 64, seed=9)
    for weight in (None, NORM.cuda()):
        for chunks in (None, 3):
            check(c, queries(sum(counts), 8), counts, norm_weight=weight, hints=dict(max_new=130, max_tokens=1300, max_chunks=chunks))


def test_splits_are_joined(cuda):
    """Contexts that are cut: one token, a chunk of a single kv head."""
    c = Cache([9000], [68], 1, 2, 2, 64, seed=10)
    for weight in (None, NORM.cuda()):
        check(c, queries(1, 4), [1], norm_weight=weight)
        check(c, queries(10, 4), [10], norm_weight=weight)
    assert kv.paged._library().kvq_paged_diff_attn_workspace_bytes(kv.paged._layer(c.book, 0, c.layer), 1, 1, 4, 1, 9000, 1) >= 2 * 8 * 520
    assert kv.paged._library().kvq_paged_diff_attn_workspace_bytes(kv.paged._layer(c.book, 0, c.layer), 1, 10, 4, 10, 9000, 1) >= 2 * 80 * 520


@pytest.mark.parametrize("counts,lengths,packed,cut", [([700], [4000], [20], True), ([650, 1, 300], [5000, 700, 2900], [30, 4, 10], False),
                                                       ([500, 0, 2, 510, 1], [4300, 10, 4000, 4200, 3000], [33, 0, 31, 0, 23], False),
                                                       ([400, 1, 230], [5000, 700, 2900], [30, 4, 10], True), ([300, 0, 2, 250, 1], [4300, 10, 4000, 4200, 3000], [33, 0, 31, 0, 23], True)])
@pytest.mark.parametrize("norm", [False, True])
def test_tiles_that_are_left_of_a_round_are_cut(cuda, counts, lengths, packed, cut, norm):
    """More tiles than SMs, over contexts that are long beside what is new: those of the last round are cut and joined, the others are not."""
    Hkv, rep = 8, 4
    c = Cache(lengths, packed, Hkv, 4, 2, 64, seed=21)
    q, lam = queries(sum(counts), Hkv * rep), torch.linspace(0.1, 0.9, Hkv * rep).cuda()
    before = kv.ops.LAUNCHES[0]
    got = call(c, q, lam, counts, norm_weight=NORM.cuda() if norm else None, max_new=max(counts), max_tokens=max(lengths))
    if cut:
        assert kv.ops.LAUNCHES[0] - before >= (2 if len(counts) == 1 else 3)      # tiles and the join, and where there are single tokens theirs
    at = 0
    for i, new in enumerate(counts):
        K, V = (torch.from_numpy(x).cuda() for x in c.dense(i))
        pos, j = torch.arange(lengths[i] - new, lengths[i], device="cuda")[:, None], torch.arange(lengths[i], device="cuda")
        for h in range(Hkv * rep if new else 0):
            x, g = q[at:at + new, h].double(), h // rep
            maps = [(x[:, o:o + 64] @ K[g][:, o:o + 64].T / 8).masked_fill(j > pos, -math.inf).softmax(-1) for o in (0, 64)]
            # a key, a weight and a value are rounded to fp16 once each, 2^-11 of themselves (test_gpu_paged has the bound)
            slack = 0.0
            for m, o, by in zip(maps, (0, 64), (1.0, float(lam[h]))):
                rel = x[:, o:o + 64].abs() @ K[g][:, o:o + 64].abs().T / 8 * 2.0 ** -11 + 1e-5 + 2 * 2.0 ** -11
                slack = slack + 1.05 * by * ((m * rel) @ V[g].abs() + (m * rel).sum(-1, keepdim=True) * (m @ V[g]).abs())
            want = (maps[0] - lam[h].double() * maps[1]) @ V[g]
            if norm:
                by = 1 / (want.square().mean(-1, keepdim=True) + 1e-5).sqrt()
                grow = (want.abs() * slack).mean(-1, keepdim=True) * by ** 2
                slack, want = NORM.cuda().abs() * by * 1.1 * (slack + want.abs() * grow), want * by * NORM.cuda()
            err = (got[at:at + new, h].double() - want).abs()
            assert (err <= slack + 2.0 ** -10 * want.abs() + 1e-5).all(), (i, h)
        at += new


# ---- rows that see nothing, weights that cancel, numbers that are none ----------------------------------------------------------------------

@pytest.mark.parametrize("counts", [[1, 1], [100, 1]])
def test_rows_that_see_nothing(cuda, counts):
    c = Cache([200, 300], [0, 1], 2, 4, 2, 64, seed=11)
    first = [10 ** 6 if i % 3 == 0 else 0 for i in range(sum(counts))]
    for eps in (1e-5, 0.0):
        got = call(c, queries(sum(counts), 4), torch.full((4,), 0.5).cuda(), counts, first=first, norm_weight=NORM.cuda(), norm_eps=eps)
        none = torch.tensor([f > 0 for f in first]).cuda()
        assert (got[none] == 0).all() and got.isfinite().all() and (got[~none] != 0).any()
    assert (call(c, queries(sum(counts), 4), torch.full((4,), 0.5).cuda(), counts, first=first)[none] == 0).all()


@pytest.mark.parametrize("new", [1, 70])
def test_lambdas(cuda, new):
    """0: the first map alone; 1 with halves alike: nothing; negative and large ones."""
    c = Cache([500], [0], 2, 4, 2, 64, seed=12)
    k = c.host["kf"]
    k[..., 64:] = k[..., :64]
    c.layer.kfull.copy_(k)
    q = queries(new, 4)
    q[..., 64:] = q[..., :64]
    assert (call(c, q, torch.ones(4).cuda(), [new]) == 0).all()
    assert (call(c, q, torch.ones(4).cuda(), [new], norm_weight=NORM.cuda()) == 0).all()
    padded = q.clone()
    padded[..., 64:] = 0
    one = kv.paged_attention(padded, starts([new]), c.rows, c.book, c.layer, softmax_scale=0.125).double()
    # The two kernels' weights stand under references of their own when they are rounded to fp16, by 2^-11 of each at most: either output is off by up to 2^-11 of
    # sum p |v|, and by 2^-11 of itself once it is rounded.  sum p |v| is the attention over |v|.
    size = kv.paged_attention(padded, starts([new]), c.rows, c.book, c.layer._replace(vfull=c.layer.vfull.abs()), softmax_scale=0.125).double()
    assert ((call(c, q, torch.zeros(4).cuda(), [new]).double() - one).abs() <= 2.0 ** -10 * (1.01 * size + one.abs()) + 2.0 ** -20).all()
    check(c, queries(new, 4), [new], lambdas=torch.tensor([-1.0, 7.0, 100.0, 0.0]).cuda())
    check(c, queries(new, 4), [new], lambdas=torch.tensor([-1.0, 7.0, 100.0, 0.0]).cuda(), norm_weight=NORM.cuda())


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("half", [0, 1])
def test_keys_that_are_no_numbers_reach_who_sees_them(cuda, new, half):
    c = Cache([300], [0], 1, 4, 2, 64, seed=13)
    at = 300 - new // 2 - 1                                      # the last position that about half of the new tokens see
    page = int(c.book.table[int(c.rows[0]), at // P])
    c.layer.kfull[page, 0, at % P, 64 * half] = math.nan
    got = call(c, queries(new, 2), torch.full((2,), 0.5).cuda(), [new])
    sees = torch.arange(300 - new, 300).cuda() >= at
    assert got[sees].isnan().all() and got[~sees].isfinite().all()


def test_masked_keys_of_any_value_do_not_matter(cuda):
    a, b = (Cache([400], [1], 2, 4, 2, 64, seed=14) for _ in range(2))
    page = int(b.book.table[int(b.rows[0]), 1])
    b.layer.kfull[page, :, :50] = 1e4
    b.layer.vfull[page, :, :50] = -6e4
    for new in (1, 60):
        outs = [call(c, queries(new, 8), torch.full((8,), 0.5).cuda(), [new], window=400 - new - 178) for c in (a, b)]
        assert torch.equal(*outs)


# ---- layouts, hints, streams, graphs ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("new", [1, 50])
def test_layouts_of_queries_and_outputs(cuda, new):
    # max_new: rows of q behind the last sequence would lay the work out for a longer chunk, whose sums are rounded at other places
    c = Cache([300], [1], 2, 4, 2, 64, seed=15)
    q, lam = queries(new + 2, 8), torch.linspace(0, 1, 8).cuda()
    want = call(c, q[:new].contiguous(), lam, [new], max_new=new, norm_weight=NORM.cuda())
    for how in range(4):
        x = q
        if how == 0:
            x = torch.cat([q[..., :1], q], -1)[..., 1:]
        elif how == 1:
            x = q.transpose(0, 1).contiguous().transpose(0, 1)
        elif how == 2:
            x = q.transpose(1, 2).contiguous().transpose(1, 2)
        out = torch.full((new + 2, 8, 130), 7.0, dtype=torch.float16, device="cuda")[..., 1:129]
        assert call(c, x, lam, [new], max_new=new, norm_weight=NORM.cuda(), out=out) is out
        assert torch.equal(out[:new], want) and (out[new:] == 7).all()
    wide = torch.full((8, new + 2, 128), 7.0, dtype=torch.float16, device="cuda").transpose(0, 1)
    call(c, q, lam, [new], max_new=new, norm_weight=NORM.cuda(), out=wide)
    assert torch.equal(wide[:new], want) and (wide[new:] == 7).all()


def test_many_sequences(cuda):
    n = 300
    c = Cache([1 + (i * 37) % 300 for i in range(n)], [0] * n, 1, 2, 2, 64, seed=16)
    counts = [i % 3 for i in range(n)]
    counts = [min(x, l) for x, l in zip(counts, c.lengths)]
    check(c, queries(sum(counts), 2), counts)
    counts = [0] * n
    counts[200], counts[7] = 30, 1
    check(c, queries(31, 4), counts, norm_weight=NORM.cuda(), hints=dict(max_chunks=1))


def test_streams_and_graphs(cuda):
    c = Cache([900, 200], [5, 0], 2, 4, 2, 64, seed=17)
    lam = torch.linspace(0, 1, 8).cuda()
    for counts in ([1, 1], [100, 1]):
        q = queries(sum(counts), 8)
        want, at = call(c, q, lam, counts), starts(counts)
        outs = [torch.zeros_like(want) for _ in range(4)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for i in range(10):
            for st, out in zip(streams, outs):
                with torch.cuda.stream(st):
                    kv.paged_differential_attention(q, lam, at, c.rows, c.book, c.layer, out=out)
        torch.cuda.synchronize()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for g, out in zip(graphs, outs[2:]):
            with torch.cuda.graph(g):
                kv.paged_differential_attention(q, lam, at, c.rows, c.book, c.layer, out=out)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_pages_beyond_32_bits(cuda):
    """A pool whose last pages lie beyond 2^32 bytes and 2^31 elements."""
    heads, n16 = 8, 16640                                        # 16640 pages of 8 heads: 2.18e9 elements
    gen = torch.Generator().manual_seed(18)
    cache = kv.KVmixPagedCache([(4, 2)], heads, 128, 2, 512, 1, n16, 64, 256)
    cache.book.free_ids[1:1 + n16] = torch.arange(n16, dtype=torch.int32)              # the last pages first
    step = cache.extend([1], [300])
    k, v, q = (torch.randn(300, h, 128, generator=gen).half().cuda() for h in (8, 8, 16))
    cos, sin = torch.ones(512, 32, device="cuda"), torch.zeros(512, 32, device="cuda")
    assert torch.equal(cache.append(0, k, v, cos, sin, step, q=q, parts=2), q)
    assert int(cache.book.table[1, 0]) == n16 - 1
    got = cache.attend_differential(0, q, torch.full((16,), 0.5).cuda(), step)
    x, y = (q.double().unflatten(-1, (2, 64)), k.double().unflatten(-1, (2, 64)).repeat_interleave(2, 1))
    s = torch.einsum("thmd,nhmd->mhtn", x, y) / 8
    p = s.masked_fill(torch.ones(300, 300, device="cuda").triu(1).bool(), -math.inf).softmax(-1)
    want = torch.einsum("htn,nhd->thd", p[0] - 0.5 * p[1], v.double().repeat_interleave(2, 1))
    # weights, outputs: two roundings of 2^-11 of every map's part, by rows
    both = torch.einsum("htn,nhd->thd", p[0] + 0.5 * p[1], v.double().abs().repeat_interleave(2, 1))
    assert ((got.double() - want).abs() <= 3 * 2.0 ** -11 * both + 1e-5).all()
    cache.check()


def test_no_work_and_refused_calls(cuda):
    c = Cache([100], [0], 2, 4, 2, 64, seed=19)
    lam, q = torch.ones(4).cuda(), queries(1, 4)
    assert call(c, q[:0], lam, [0]).shape == (0, 4, 128)
    base = dict(q=q, lambdas=lam, q_start=starts([1]), rows=c.rows, pages=c.book, layer=c.layer)
    for bad in (dict(lambdas=lam[:3]), dict(lambdas=lam.double()), dict(lambdas=lam.cpu()), dict(lambdas=lam.repeat(2)[::2]), dict(norm_weight=NORM), dict(norm_weight=NORM.cuda()[:64]),
                dict(norm_weight=NORM.cuda().half()), dict(norm_weight=NORM.cuda(), norm_eps=-1.0), dict(norm_weight=NORM.cuda(), norm_eps=math.nan), dict(q=q.float()), dict(q=q[..., :64]),
                dict(q=q[0]), dict(q=q[:, :3], lambdas=lam[:3]), dict(window=-1), dict(softcap=-1.0), dict(softmax_scale=math.nan), dict(max_new=0),
                dict(out=torch.empty(1, 4, 128, device="cuda")), dict(out=q[:, :1].expand(-1, 4, -1))):
        with pytest.raises(RuntimeError):
            kv.paged_differential_attention(**dict(base, **bad))
    assert int(c.book.count[2]) == 0


# ---- all of them together ------------------------------------------------------------------------------------------------------------------

def test_a_search_with_differential_attention(cuda):
    """A small model's beam search: keys and queries rotated on the way into the pages, differential attention, selection, reordering, pages settled.
    Every step's attention against the beams' own tokens, kept in lists."""
    gen = torch.Generator().manual_seed(20)
    beams, Hkv, nh, V, layers = 3, 2, 4, 60, 2
    cache = kv.KVmixPagedCache([(4, 4)] * layers, Hkv, 128, 8, 600, 40, 40, 32, 10 ** 6)           # nothing is packed: the tokens are as they were written
    angle = torch.arange(600, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    cos, sin, lam, weight = angle.cos().float().cuda(), angle.sin().float().cuda(), torch.linspace(0.2, 0.8, nh).cuda(), torch.ones(128).cuda()
    emb = torch.randn(V, layers, Hkv * 2 + nh, 128, generator=gen).half().cuda()                   # a token's keys, values and queries
    head = (torch.randn(nh * 128, V, generator=gen) * 0.1).cuda()
    turn = torch.complex(cos.double(), sin.double())

    def rotated(x, pos):
        z = x.double().unflatten(-1, (2, 2, 32)).transpose(-1, -2)                                  # parts of 64, partners 32 apart
        z = torch.view_as_complex(z.contiguous()) * turn[pos][:, None, None]
        return torch.view_as_real(z).transpose(-1, -2).flatten(-3)

    rows = [6, 1, 3, 0, 7, 2]
    prompts = [torch.randint(0, V, (n,), generator=gen).tolist() for n in (130, 250)]
    histories = [list(prompts[i // beams]) for i in range(6)]

    def forward(step, tokens, who):
        x = emb[torch.tensor(tokens).cuda()]
        for l in range(layers):
            k, v, q = x[:, l, :Hkv], x[:, l, Hkv:2 * Hkv], x[:, l, 2 * Hkv:]
            q = cache.append(l, k, v, cos, sin, step, q=q, parts=2)
            out = cache.attend_differential(l, q, lam, step, norm_weight=weight)
            for i, hist in who:                                   # the last token of every sequence
                e = emb[torch.tensor(hist).cuda(), l]
                pos = torch.arange(len(hist), device="cuda")
                K, Q = rotated(e[:, :Hkv], pos).half().double(), rotated(e[-1:, 2 * Hkv:], pos[-1:]).half().double()
                W = e[:, Hkv:2 * Hkv].double().repeat_interleave(nh // Hkv, 1)
                K = K.repeat_interleave(nh // Hkv, 1)
                maps = [torch.softmax(torch.einsum("hd,nhd->hn", Q[0, :, o:o + 64], K[..., o:o + 64]) / 8, -1) for o in (0, 64)]
                y = torch.einsum("hn,nhd->hd", maps[0] - lam.double()[:, None] * maps[1], W)
                want = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt()
                # roundings of 2^-11 of rotated keys and queries (a score of some units), of weights and the output, by rows
                assert (out[i].double() - want).norm() <= 2e-2 * want.norm(), (i, l)
        return out.flatten(1).float() @ head

    step = cache.extend([rows[0], rows[3]], [len(p) for p in prompts])
    logits = forward(step, prompts[0] + prompts[1], [(len(prompts[0]) - 1, prompts[0]), (len(prompts[0]) + len(prompts[1]) - 1, prompts[1])])
    last = torch.tensor([len(prompts[0]) - 1, len(prompts[0]) + len(prompts[1]) - 1]).cuda()
    logits = logits[last].repeat_interleave(beams, 0)
    cache.reorder([rows[1], rows[2], rows[4], rows[5]], [rows[0], rows[0], rows[3], rows[3]])
    scores = torch.tensor([0.0, -math.inf, -math.inf] * 2).cuda()
    for _ in range(140):
        chosen = cache.advance(rows, logits, scores, beams, ends=ints(5))
        value = scores.double()[:, None] + torch.log_softmax(logits.double(), -1)
        for r in range(2):
            flat = value[r * beams:(r + 1) * beams].clone()
            flat[:, 5] = -math.inf
            best = torch.topk(flat.flatten(), beams).values
            assert (chosen.next_scores[r].double() - best).abs().max() <= 1e-4
        histories = [histories[i // beams * beams + b] + [t] for i, (b, t) in enumerate(zip(chosen.next_beams.flatten().tolist(), chosen.next_tokens.flatten().tolist()))]
        scores = chosen.next_scores.flatten()
        step = cache.extend(rows, [1] * 6)
        logits = forward(step, [h[-1] for h in histories], list(enumerate(histories)))
    cache.check()
    assert cache.lengths == cache.book.length.tolist() and sorted(cache.lengths) == [0, 0] + [270] * 3 + [390] * 3
    cache.free(rows)
    assert cache.free_pages() == (40, 40)
