"""The paged cache over the whole range of its arguments: caps, scales and sizes of keys far from the usual, windows, shared pages, tensors that
a call has to refuse before it changes anything."""
import math

import pytest
import torch

import kvmix_b200 as kv
from kvmix_b200 import ops
from test_gpu_paged import P, Cache, attend, queries
from test_gpu_paged_book import ints, small, snapshot, unchanged

pytestmark = pytest.mark.gpu


def parts(c, i):
    """K, V [Hkv, length, 128] of sequence i and what their elements are sums of, |code * scale| + |minimum|, in 64 bits on the device."""
    K, V = (torch.from_numpy(x).cuda() for x in c.dense(i))
    kept = c.host
    signed = kept["k"], kept["v"]
    c.host = dict(kept, k=(kept["k"][0], kept["k"][1].abs(), kept["k"][2].abs()), v=(kept["v"][0], kept["v"][1].abs(), kept["v"][2].abs()))
    Ka, Va = (torch.from_numpy(x).cuda().abs() for x in c.dense(i))
    c.host = dict(kept, k=signed[0], v=signed[1])
    return K, V, Ka, Va


def attention(c, q, counts, exact_keys, scale=None, softcap=0.0, window=0):
    """Attention from its definition in 64 bits, and a bound of the kernels' roundings that does not grow with the cap:
    a score    2^-20 of the sum of its terms' sizes (pairs of fp16 or fp16 itself, sums in fp32; 2^-11 more where a key is rounded to fp16) and
               4e-6 of itself (conversion to log2 units and the cap, some roundings of 2^-24 and a polynomial of 6e-7)
    an output  three roundings to fp16 of 2^-11: of a weight, of a value or of weight * scale, of the output."""
    scale = 1 / math.sqrt(128) if scale is None else scale
    eps, rep, at = 2.0 ** -11, q.shape[1] // c.Hkv, 0
    out, slack = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for i, new in enumerate(counts):
        n = c.lengths[i]
        K, V, Ka, Va = parts(c, i)
        pos, j = torch.arange(n - new, n, device="cuda")[:, None], torch.arange(n, device="cuda")
        seen = (j <= pos) & (j > pos - window) if window else j <= pos
        for h in range(q.shape[1]):
            x, g = q[at:at + new, h].double(), h // rep
            s = x @ K[g].T * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            p = s.masked_fill(~seen, -math.inf).softmax(-1)
            rel = x.abs() @ Ka[g].T * abs(scale) * (2.0 ** -20 + (0 if exact_keys else eps)) + s.abs() * 4e-6
            out[at:at + new, h] = o = p @ V[g]
            slack[at:at + new, h] = 1.05 * ((p * (rel + 2 * eps)) @ Va[g] + (p * rel).sum(-1, keepdim=True) * o.abs()) + eps * o.abs() + 2.0 ** -24
        at += new
    return out, slack


def holds(got, want, slack):
    err = (got.double() - want).abs()
    assert err.isfinite().all()
    worst = (err / slack).max().item()
    assert worst <= 1.0, f"{worst:.2f} times the bound; largest error {err.max().item():.3e}"


def rows_hold(got, want, most):
    err = (got.double() - want).norm(dim=-1) / want.norm(dim=-1).clamp(min=1e-3)
    assert err.isfinite().all() and err.max() <= most, f"row error {err.max().item():.3e}"


def sized(c, k_size):
    """The same cache with keys of another size."""
    for t in (*c.host["k"][1:], c.host["kf"]):
        t.mul_(k_size)
    c.layer = c.layer._replace(kscale=c.host["k"][1].cuda(), kmn=c.host["k"][2].cuda(), kfull=c.host["kf"].cuda())
    return c


# ---- caps ------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("softcap", [1.0, 30.0, 1e4, 1e5, 1e6, 1e9])
@pytest.mark.parametrize("kb,vb", [(2, 4), (4, 2), (3, 3)])
def test_caps_of_one_token(cuda, softcap, kb, vb):
    """A score keeps its own precision, however large the cap is."""
    c = Cache([700, 301, 1], [4, 2, 0], 2, kb, vb, 32, seed=3)
    q = queries(3, 4)
    got, (want, slack) = attend(c, q, [1] * 3, softcap=softcap), attention(c, q, [1] * 3, kb != 3, softcap=softcap)
    holds(got, want, slack)
    rows_hold(got, want, 2e-3)                                  # the framework's own tolerance


@pytest.mark.parametrize("softcap", [1.0, 1e5, 1e6])
@pytest.mark.parametrize("new", [1, 100])
def test_small_scores_beside_large_ones(cuda, softcap, new):
    """Rows whose scores come near the cap beside rows whose do not (other heads, other tokens): each is as exact as it is alone."""
    c = Cache([700], [0], 1, 4, 4, 64, seed=6)
    q = queries(new, 4)
    scale = softcap / 2e5 if softcap > 1 else 0.2
    q = (q.float() / (11.3 * scale)).half()                               # scores of 1
    q[:, 1] *= 1e4 * scale * 11.3 if softcap > 1 else 2                   # scores of some 0.5 to 2 caps
    got = attend(c, q, [new], softcap=softcap, scale=scale)
    holds(got, *attention(c, q, [new], True, softcap=softcap, scale=scale))


@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("scale", [1e-3, 1e-4, 1e-5, 1e-6])
def test_large_raw_scores_below_the_cap(cuda, new, scale):
    """Queries and keys so large that their products are 1e4 to 5e7, a small softmax_scale, scores up to the cap's size."""
    c = sized(Cache([700], [0], 1, 4, 4, 64, seed=7, outliers=False), 60.0)
    q = (queries(new, 4) * (14 / (scale * 60 * 11.3))).half() if scale > 2e-6 else (queries(new, 4) * 1.2e4).half()
    assert q.isfinite().all()
    holds(attend(c, q, [new], softcap=50.0, scale=scale), *attention(c, q, [new], True, softcap=50.0, scale=scale))


@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("softcap", [float("inf"), 1e300, 3e38, 1e31])
def test_a_cap_beyond_all_scores_is_none(cuda, new, softcap):
    c = Cache([700], [3], 1, 2, 4, 64, seed=8)
    q = queries(new, 4)
    assert torch.equal(attend(c, q, [new], softcap=softcap), attend(c, q, [new]))


@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("softcap", [1e-25, 1e-38, 1e-42])
def test_a_cap_below_all_scores(cuda, new, softcap):
    """All scores the same to 2^-24: the mean of the values; a query of zeros among them."""
    c = Cache([300], [1], 1, 4, 4, 64, seed=8)
    q = queries(new, 4)
    q[0, 0] = 0
    holds(attend(c, q, [new], softcap=softcap), *attention(c, q, [new], True, scale=0.0))


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan"), 1e39])
def test_scales_that_are_no_numbers(cuda, bad):
    c = Cache([300], [1], 1, 4, 4, 64, seed=8)
    with pytest.raises(RuntimeError):
        attend(c, queries(1, 4), [1], scale=bad)


# ---- a stalled wait --------------------------------------------------------------------------------------------------------------------

def test_a_stalled_wait_leaves_the_cache_whole(cuda):
    """An attention that gave up waiting says so in the status.  Its own output is lost; the layers behind it are written, and later calls work."""
    gen = torch.Generator().manual_seed(5)
    cache = kv.KVmixPagedCache([(4, 2), (2, 2), (3, 3)], 2, 128, 3, 700, 8, 10, 64, 128)
    k, v = (torch.randn(3, 400, 2, 128, generator=gen).half().cuda() for _ in range(2))
    at = 0
    for n in (300, 1, 99):
        s = cache.extend([1], [n])
        for l in range(3):
            cache.write(l, k[l, at:at + n], v[l, at:at + n], s)
            if l == 0:
                cache.book.count[2] |= 16                       # what a wait of layer 0's attention leaves behind
        at += n
        ids = cache.book.table[1].tolist()
        for l in range(3):
            packed = int(cache.book.packed[1])
            for j in range(packed, -(-at // P)):
                m = min(P, at - j * P)
                assert torch.equal(cache.layers[l].kfull[ids[j], :, :m], k[l, j * P:j * P + m].transpose(0, 1))
                assert torch.equal(cache.layers[l].vfull[ids[j], :, :m], v[l, j * P:j * P + m].transpose(0, 1))
    cache.settle()
    assert cache.book.packed.tolist() == [0, 2, 0]
    with pytest.raises(RuntimeError, match="gave up"):
        cache.check()
    cache.check()
    assert cache.lengths == cache.book.length.tolist() == [0, 400, 0]
    cache.free([1])
    assert cache.free_pages() == (8, 10)


# ---- windows ---------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 40, float("inf")])
def test_windows_beyond_32_bits(cuda, window):
    cache = small()
    kv.pages_settle(ints(0), window, cache.book, cache.layers)
    assert not cache.book.packed.any()                          # nothing ends so far back
    never = kv.KVmixPagedCache([(4, 2)], 1, 128, 1, 512, 4, 4, 64, residual_length=window)
    never.extend([0], [512])
    never.settle()
    assert not never.book.packed.any()
    q = torch.randn(3, 4, 128, device="cuda").half()
    for rows in (ints(0), ints(2)):
        for n in (1, 3):
            got = kv.paged_attention(q[:n], ints(0, n), rows, cache.book, cache.layers[0], window=window)
            assert torch.equal(got, kv.paged_attention(q[:n], ints(0, n), rows, cache.book, cache.layers[0]))
    cache.check()


# ---- small keys ------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kb,vb,group", [(2, 2, 32), (4, 4, 64), (1, 4, 128), (4, 2, 128), (3, 3, 128)])
@pytest.mark.parametrize("rep", [1, 2, 4, 8])
@pytest.mark.parametrize("k_size", [1e-2, 1e-3, 1e-4, 3e3])
def test_keys_of_any_size(cuda, kb, vb, group, rep, k_size):
    """Keys far from 1 and queries that make up for it: scores of the usual size from the smallest fp16 scales, and from large ones."""
    c = sized(Cache([700], [5], 1, kb, vb, group, seed=5, outliers=False), k_size)
    q = (queries(1, rep).float() / k_size).half()
    got, (want, slack) = attend(c, q, [1]), attention(c, q, [1], kb != 3)
    holds(got, want, slack)
    rows_hold(got, want, 2e-3)                                  # the framework's own tolerance


def test_key_scales_that_grow_along_the_sequence(cuda):
    """Pages, and channels of a page, whose scales are 2^20 apart."""
    for rep, kb, group in ((1, 4, 32), (2, 2, 64), (4, 1, 128), (8, 4, 64), (4, 3, 128)):
        c = Cache([128 * 9], [9], 1, kb, 2, group, seed=8, outliers=False)
        ids = c.host["table"][c.host["rows"][0]].tolist()
        for j, i in enumerate(ids):
            for t in c.host["k"][1:]:
                t[i] *= 2.0 ** (-12 + 2 * min(j, 8 - j))
                t[i, :, 64:] *= 2.0 ** (-6 if j % 2 else 4)
        q = (queries(1, rep).float() * 8).half()
        holds(attend(sized(c, 1.0), q, [1]), *attention(c, q, [1], kb != 3))


# ---- refused before anything is changed ------------------------------------------------------------------------------------------------

def shifted(t):
    """The same tensor, contiguous, two elements behind a 16-byte boundary."""
    x = torch.zeros(t.numel() + 8, dtype=t.dtype, device=t.device)[2:2 + t.numel()].view(t.shape)
    x.copy_(t)
    assert x.is_contiguous() and x.data_ptr() % 16
    return x


@pytest.mark.parametrize("name", ["kcode", "kscale", "kmn", "kfull", "vcode", "vscale", "vmn", "vfull"])
def test_misaligned_pages_are_refused_at_once(cuda, name):
    """Pages that the kernels cannot copy are refused before the bookkeeping hands their numbers on."""
    cache = small()
    cache.settle([0])
    cache.extend([0], [1])
    cache.free([2])
    layers = [cache.layers[0], cache.layers[0]._replace(**{name: shifted(getattr(cache.layers[0], name))})]
    before = snapshot(cache)
    calls = [lambda: kv.pages_settle(ints(0), 0, cache.book, layers), lambda: kv.pages_compact(cache.book, layers),
             lambda: kv.page_write(torch.zeros(1, 1, 128, device="cuda").half(), torch.zeros(1, 1, 128, device="cuda").half(), ints(0, 1), ints(0), cache.book, layers[1]),
             lambda: kv.paged_attention(queries(1, 4), ints(0, 1), ints(0), cache.book, layers[1])]
    if name in ("kfull", "vfull"):
        calls.append(lambda: kv.pages_fork(ints(0), ints(3), cache.book, layers))
    for call in calls:
        with pytest.raises(RuntimeError):
            call()
        unchanged(cache, before)
    cache.check()


def test_outputs_that_lie_over_one_another(cuda):
    c = Cache([300], [1], 1, 4, 4, 64, seed=8)
    one = torch.zeros(1, 1, 128, dtype=torch.half, device="cuda")
    flat = torch.zeros(4000, dtype=torch.half, device="cuda")
    for out in (one.expand(2, 4, 128), torch.zeros(2, 1, 128, dtype=torch.half, device="cuda").expand(2, 4, 128), flat.as_strided((2, 4, 128), (256, 128, 1)),
                flat.as_strided((2, 4, 128), (1024, 64, 1)), flat.as_strided((2, 4, 128), (128, 200, 1))):
        with pytest.raises(RuntimeError, match="out"):
            attend(c, queries(2, 4), [2], out=out)
    want = attend(c, queries(2, 4), [2])
    for out in (flat.as_strided((2, 4, 128), (128, 256, 1)), flat.as_strided((2, 4, 128), (600, 130, 1)), torch.zeros(2, 4, 128, dtype=torch.half, device="cuda")):
        assert torch.equal(attend(c, queries(2, 4), [2], out=out), want)
    assert attend(c, queries(1, 4), [1], out=flat.as_strided((1, 4, 128), (0, 128, 1))).any()


def test_a_step_takes_its_own_tokens(cuda):
    cache = small()
    s = cache.extend([0], [3])
    x = torch.zeros(4, 1, 128, device="cuda").half()
    before = snapshot(cache)
    for k, v in ((x[:2], x[:2]), (x, x), (x[:3], x)):
        with pytest.raises(RuntimeError):
            cache.write(0, k, v, s)
    unchanged(cache, before)
    cache.write(0, x[:3], x[:3], s)


# ---- shared pages ----------------------------------------------------------------------------------------------------------------------

def test_shared_pages_are_never_written(cuda):
    """New tokens that are said to reach back into pages which other sequences hold too: what lies there stays, the rest is written."""
    gen = torch.Generator().manual_seed(9)
    cache = kv.KVmixPagedCache([(4, 4)], 2, 128, 3, 700, 2, 10, 64, 1000)
    k, v = (torch.randn(300, 2, 128, generator=gen).half().cuda() for _ in range(2))
    cache.write(0, k, v, cache.extend([0], [300]))
    cache.fork([0], [1])
    cache.extend([1], [20])
    x, y = (torch.randn(320, 2, 128, generator=gen).half().cuda() for _ in range(2))
    kv.page_write(x, y, ints(0, 320), ints(1), cache.book, cache.layers[0])           # 20 of them are new
    ids, own = cache.book.table[0].tolist(), cache.book.table[1].tolist()
    assert ids[:2] == own[:2] and ids[2] != own[2]
    for t, old, new in ((cache.layers[0].kfull, k, x), (cache.layers[0].vfull, v, y)):
        for j in range(2):
            assert torch.equal(t[ids[j]], old[j * P:j * P + P].transpose(0, 1))
        assert torch.equal(t[ids[2], :, :44], old[256:300].transpose(0, 1))
        assert torch.equal(t[own[2], :, :64], new[256:320].transpose(0, 1))
    with pytest.raises(RuntimeError, match="not written"):
        cache.check()
    cache.free([0])                                                                   # nobody else holds them now
    kv.page_write(x, y, ints(0, 320), ints(1), cache.book, cache.layers[0])
    assert torch.equal(cache.layers[0].kfull[ids[0]], x[:P].transpose(0, 1))
    cache.check()


def test_tokens_without_a_place_are_reported(cuda):
    """A step that was not counted, a sequence that is not there, a packed page: page_write says that it left them out, and holds nothing up."""
    cache = small()
    x = torch.zeros(300, 1, 128, device="cuda").half()
    for begin, rows, fine in ((ints(0, 1), ints(1), False), (ints(0, 11), ints(2), False), (ints(0, 10), ints(2), True), (ints(0, 300), ints(0), True)):
        kv.page_write(x, x, begin, rows, cache.book, cache.layers[0])
        if fine:
            cache.check()
        else:
            with pytest.raises(RuntimeError, match="not written"):
                cache.check()
    cache.settle([0])
    kv.page_write(x, x, ints(0, 300), ints(0), cache.book, cache.layers[0])            # 256 of them are packed
    assert int(cache.book.count[2]) == 32
    cache.extend([0], [1])
    assert int(cache.book.length[0]) == 301
    with pytest.raises(RuntimeError, match="not written"):
        cache.check()


# ---- launches --------------------------------------------------------------------------------------------------------------------------

def test_launches_are_counted_as_they_are(cuda):
    cache = kv.KVmixPagedCache([(2, 2)] * 3, 1, 128, 4, 9000, 140, 150, 64, 128)
    x = torch.zeros(8200, 1, 128, device="cuda").half()

    def launches(f, *args, **kw):
        n = ops.LAUNCHES[0]
        f(*args, **kw)
        return ops.LAUNCHES[0] - n
    b, l = cache.book, cache.layers[0]
    assert launches(kv.pages_extend, ints(0, 1, 2), ints(8192, 5, 3), b) == 1
    assert launches(kv.pages_extend, ints(), ints(), b) == 0
    assert launches(kv.page_write, x[:8200], x[:8200], ints(0, 8192, 8197, 8200), ints(0, 1, 2), b, l) == 1
    assert launches(kv.pages_settle, ints(0, 1, 2), 128, b, cache.layers) == 4
    q = queries(9, 4)
    assert launches(kv.paged_attention, q[:1], ints(0, 1), ints(1), b, l, max_tokens=128) == 1               # whole
    assert launches(kv.paged_attention, q[:1], ints(0, 1), ints(0), b, l) == 2                                # splits and their join
    assert launches(kv.paged_attention, q[:9], ints(0, 3, 8, 9), ints(2, 1, 0), b, l, max_new=5, max_tokens=128) == 2      # both kernels
    assert launches(kv.paged_attention, q[:9], ints(0, 3, 8, 9), ints(2, 1, 0), b, l, max_new=5) == 4
    assert launches(kv.paged_attention, q[:0], ints(0, 0), ints(0), b, l) == 0
    assert launches(kv.pages_fork, ints(1), ints(3), b, cache.layers) == 2
    assert launches(kv.pages_compact, b, cache.layers) == 3
    assert launches(kv.pages_free, ints(3), b) == 1
    cache.check()


# ---- bookkeeping that holds wrong numbers ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("what", ["length", "packed", "free_ids", "count", "table", "refs"])
@pytest.mark.parametrize("value", [-1, -2 ** 31, -2 ** 30, 2 ** 31 - 1, 2 ** 30, 5000])
def test_wrong_numbers_in_the_bookkeeping_stay_inside(cuda, what, value):
    """Bookkeeping that was never set up, or written over: every call ends without touching anything outside the tensors (they lie in one block, with
    guards between them)."""
    sizes = dict(table=(4, 4), length=(4,), packed=(4,), refs=(9,), free_ids=(9,), count=(4,))
    block = torch.full((4096,), 77, dtype=torch.int32, device="cuda")
    parts, at = {}, 256
    for name, shape in sizes.items():
        n = math.prod(shape)
        parts[name] = block[at:at + n].view(shape)
        at += n + 256
    outside = torch.ones_like(block, dtype=torch.bool)
    for t in parts.values():
        start = (t.data_ptr() - block.data_ptr()) // 4
        outside[start:start + t.numel()] = False
    cache = kv.KVmixPagedCache([(4, 2)], 1, 128, 4, 512, 4, 5, 64, 0)
    for call in range(8):
        for name, t in parts.items():
            t.copy_(getattr(cache.book, name))
        book = kv.PageBook(**parts, n_packed=4)
        kv.pages_extend(ints(0, 1), ints(300, 10), book)
        kv.pages_settle(ints(0), 130, book, cache.layers)
        assert int(book.count[2]) == 0
        if what == "count":
            book.count[:2] = value
        else:
            parts[what].fill_(value)
        x = torch.zeros(9, 1, 128, device="cuda").half()
        (lambda: kv.pages_extend(ints(0, 1, 2), ints(100, 0, 1), book), lambda: kv.pages_free(ints(0, 2), book), lambda: kv.pages_settle(ints(0, 1), 0, book, cache.layers),
         lambda: kv.pages_fork(ints(0, 1), ints(2, 3), book, cache.layers), lambda: kv.pages_compact(book, cache.layers),
         lambda: kv.page_write(x, x, ints(0, 9), ints(0), book, cache.layers[0]), lambda: kv.paged_attention(queries(9, 4), ints(0, 9), ints(0), book, cache.layers[0]),
         lambda: kv.paged_attention(queries(1, 4), ints(0, 1), ints(0), book, cache.layers[0]))[call]()
        torch.cuda.synchronize()
        assert (block[outside] == 77).all()


@pytest.mark.parametrize("bad", [[0, -2 ** 31, 9], [5, -2 ** 31, 9], [2 ** 31 - 1, 9, 9], [0, 2 ** 31 - 1, 2 ** 31 - 1], [-2 ** 31, 3, 9], [9, 4, 0], [-5, 100, 3]])
def test_wrong_numbers_of_new_tokens_stay_inside(cuda, bad):
    """q_start that does not ascend, or leads outside q: nothing outside out is written, no page but the sequences' own."""
    cache = small()
    block = torch.full((40, 4, 128), 7.0, dtype=torch.half, device="cuda")
    x = torch.zeros(9, 1, 128, device="cuda").half()
    own = cache.book.table[[0, 2]].flatten().tolist()
    for tokens, hints in ((9, {}), (9, dict(max_new=1)), (9, dict(max_new=5, max_chunks=1))):
        kv.paged_attention(queries(tokens, 4), ints(*bad), ints(0, 2), cache.book, cache.layers[0], out=block[16:16 + tokens], **hints)
        torch.cuda.synchronize()
        assert (block[:16] == 7).all() and (block[16 + tokens:] == 7).all()
    others = [p for p in range(6) if p not in own]
    before = cache.layers[0].kfull[others].clone()
    kv.page_write(x, x, ints(*bad), ints(0, 2), cache.book, cache.layers[0])
    assert torch.equal(cache.layers[0].kfull[others].view(torch.int16), before.view(torch.int16))
    assert int(cache.book.count[2]) in (0, 32)                                        # tokens without a place are reported, nothing else


# ---- long sequences, packing under replay ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kb,vb,group,rep,length", [(3, 2, 128, 4, 131072), (2, 1, 64, 4, 32768), (2, 2, 32, 1, 65433), (4, 4, 64, 8, 40001)])
def test_one_token_over_a_long_context(cuda, kb, vb, group, rep, length):
    """The framework's own tolerance, 2e-3 of a row: a weight's and an output's rounding are 2^-11 at most each, and a score's error is 2^-11 of
    its terms at 3 bits (random signs: 1e-4 of 1) and next to nothing otherwise."""
    c = Cache([length], [(length - 200) // P], 1, kb, vb, group, seed=length)
    q = queries(1, rep)
    got, (want, slack) = attend(c, q, [1]), attention(c, q, [1], kb != 3)
    holds(got, want, slack)
    rows_hold(got, want, 2e-3)


@pytest.mark.parametrize("kb,vb,group,new,length", [(2, 2, 64, 300, 34816), (4, 4, 32, 129, 20001), (3, 3, 128, 70, 9000)])
def test_a_chunk_over_a_long_context(cuda, kb, vb, group, new, length):
    """The same of chunks: keys are rounded to fp16 besides, 2^-12 of an element with random signs: 128 terms of 1 give a score 2e-4 to 5e-4."""
    c = Cache([length], [(length - new) // P], 1, kb, vb, group, seed=length)
    q = queries(new, 4)
    got, (want, slack) = attend(c, q, [new]), attention(c, q, [new], False)
    holds(got, want, slack)
    rows_hold(got, want, 2e-3)


@pytest.mark.parametrize("kb,vb,group", [(2, 2, 64), (3, 3, 128), (4, 4, 32)])
@pytest.mark.parametrize("counts", [[1, 300, 1, 2], [40, 1, 1, 0], [1, 1, 700, 1]])
def test_split_single_tokens_beside_chunks(cuda, kb, vb, group, counts):
    """Single tokens over a long context, in splits, in one call with chunks: each kernel finds its own partial sums."""
    c = Cache([9000, 4100, 2000, 300], [68, 20, 10, 0], 2, kb, vb, group, seed=kb)
    q = queries(sum(counts), 8)
    want, slack = attention(c, q, counts, False)
    for hints in ({}, dict(max_new=max(counts), max_chunks=2, max_tokens=9000)):
        holds(attend(c, q, counts, **hints), want, slack)


def test_replayed_steps_pack_what_is_due(cuda):
    """A captured step replayed over two boundaries of pages: the packed pages are those that left the window, and are as many as the steps say."""
    gen = torch.Generator().manual_seed(5)
    cache = kv.KVmixPagedCache([(2, 2)], 1, 128, 4, 700, 12, 12, 64, 128)
    rows, prompt = [3, 0, 2], [200, 127, 1]
    s = cache.extend(rows, prompt)
    x = torch.randn(s.tokens, 1, 128, generator=gen).half().cuda()
    cache.write(0, x, x, s)
    cache.settle(rows)
    at, ones, begin = ints(*rows), ints(1, 1, 1), ints(0, 1, 2, 3)
    new = torch.zeros(3, 1, 128, dtype=torch.half, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.pages_extend(at, ones, cache.book)
        kv.page_write(new, new, begin, at, cache.book, cache.layers[0])
        kv.pages_settle(at, 128, cache.book, cache.layers)
    for i in range(1, 301):
        graph.replay()
        lengths = [127 + i, 0, 1 + i, 200 + i]
        assert cache.book.length.tolist() == lengths
        assert cache.book.packed.tolist() == [max(0, n - 128) // 128 for n in lengths], i
    assert cache.book.packed.tolist() == [2, 0, 1, 2]
    cache.check()


def test_as_many_rows_as_a_table_may_have(cuda):
    """2^20 rows: a bit each in shared memory, beyond what a launch has unasked."""
    n = 1 << 20
    cache = kv.KVmixPagedCache([(2, 2)], 1, 128, n, 128, 2, 4, 128, 0)
    rows = [n - 1, 0, 131072]
    kv.pages_extend(ints(*rows), ints(128, 128, 5), cache.book)
    assert cache.book.length[rows].tolist() == [128, 128, 5] and int(cache.book.length.sum()) == 261
    kv.pages_settle(ints(*rows), 0, cache.book, cache.layers)
    kv.pages_fork(ints(n - 1, 131072), ints(n - 2, 1), cache.book, cache.layers)
    kv.pages_compact(cache.book, cache.layers)
    assert cache.book.packed[[n - 1, n - 2, 0, 131072, 1]].tolist() == [1, 1, 1, 0, 0] and cache.free_pages() == (0, 2)
    kv.pages_free(ints(n - 1, 5, n - 1), cache.book)                                  # named twice
    with pytest.raises(RuntimeError, match="bad rows"):
        cache.check()
    kv.pages_free(ints(n - 1, n - 2, 0, 131072, 1), cache.book)
    cache.check()
    assert cache.free_pages() == (2, 4) and not cache.book.length.any()


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("scale", [0.0, 1e-30, -1e-3])
def test_scales_of_next_to_nothing(cuda, new, scale):
    c = Cache([300], [1], 2, 4, 2, 64, seed=9)
    q = queries(new, 4)
    holds(attend(c, q, [new], scale=scale), *attention(c, q, [new], True, scale=scale))
