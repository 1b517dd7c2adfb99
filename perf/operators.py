"""What the paged cache is measured on: attention of new tokens over pages of packed and of fp16 keys and values, and the calls that
fill, share, free and compact those pages.

A page holds 128 tokens of one sequence.  A sequence's oldest pages are packed (1 to 4 bits, the formats of the layer cache: keys per
channel over groups of tokens, values per token over groups of channels, groups of 11 at 3 bits, the last of a page shorter), the
others are fp16.  Four kinds of pass, each through the public entry points:

    attend   attention of the last tokens of every sequence over its pages: ``paged_attention`` (one token each, chunks, or both)
    admit    prompts come in where finished sequences leave: ``pages_free``, ``pages_extend``, ``page_write``, ``pages_settle``
    branch   children that have been decoded apart are dropped and taken anew from their parents: ``pages_free``, ``pages_fork``
    compact  half of the sequences leave, the others close up, new ones come and are packed: ``pages_free``, ``pages_compact``,
             ``pages_extend``, ``pages_settle``

Keys and values are N(0, 1) with four key channels per head that are eight times larger, as the attention configurations of
``kvmix_b200.configs`` have them.  With ``own`` false everything is computed by elementary torch operations.
"""
import math
import random

import torch

own = False

D = 128                              # head dimension of every supported model
P = 128                              # tokens of a page
FIELDS = {1: 32, 2: 16, 3: 11, 4: 8}
# what the largest listed case costs, which drawn ones stay below: (query head, query, key) triples, and bytes of pages
TRIPLES = 32 * 2048 * 34816
PAGE_BYTES = 11 << 30


def listed():
    attend = dict(kind="attend", ragged=False, residual=128, softcap=0.0, alibi=False, window=0, prefix=0, documents=0, chunks=-1)
    return [
        # the smallest call: the next token of one conversation
        dict(attend, name="decode one short", seqs=1, heads=32, kv_heads=8, new=1, context=777, bits="42", group=64),
        # one layer of 64 sequences of a 32-head model, the 2-bit layers of its bit map
        dict(attend, name="decode batch 64", seqs=64, heads=32, kv_heads=32, new=1, context=4096, ragged=True, bits="22", group=32),
        # grouped queries over 32k tokens, scores capped by a tanh
        dict(attend, name="decode grouped 32k capped", seqs=8, heads=32, kv_heads=8, new=1, context=32768, bits="21", group=64, softcap=50.0),
        # one very long sequence, a bias that falls with the distance
        dict(attend, name="decode 131k distance bias", seqs=1, heads=32, kv_heads=8, new=1, context=131072, bits="32", group=128,
             residual=256, alibi=True),
        # a prompt of its own: nothing is packed yet
        dict(attend, name="prompt 4096", seqs=1, heads=32, kv_heads=8, new=4096, context=4096, bits="44", group=64, residual=4096),
        # the last chunk of a long prompt, most of it packed
        dict(attend, name="chunk 2048 over 32k", seqs=1, heads=32, kv_heads=8, new=2048, context=34816, bits="22", group=64, residual=2048),
        # second turns of four chats of a 32-head model, odd lengths, a sliding window, capped scores
        dict(attend, name="turns of 501 windowed", seqs=4, heads=32, kv_heads=32, new=501, context=5803, ragged=True, bits="44", group=32,
             residual=512, softcap=30.0, window=2000),
        # a step of a server: two chunks of several documents, the first 100 tokens in view of each other, and 22 that decode
        dict(attend, name="mixed step", seqs=24, heads=32, kv_heads=8, new=701, context=8192, ragged=True, bits="32", group=128,
             residual=768, prefix=100, documents=3, chunks=2),
        # one short prompt
        dict(kind="admit", name="admit one prompt", seqs=1, kv_heads=8, length=301, bits="42", group=64, residual=128, layers=1),
        # eight long prompts
        dict(kind="admit", name="admit eight of 8k", seqs=8, kv_heads=8, length=8191, bits="32", group=128, residual=256, layers=2),
        # four continuations each of 16 prompts, taken up again from the prompts' ends
        dict(kind="branch", name="branch 16 by 4", seqs=16, each=4, kv_heads=8, length=1500, bits="42", group=64, layers=8),
        # sequences of some 2000 tokens come and go
        dict(kind="compact", name="compact 64", seqs=64, kv_heads=8, length=2000, bits="44", group=64, layers=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "admit", "branch", "compact"])
    bits, group = "%d%d" % (rng.randint(1, 4), rng.randint(1, 4)), rng.choice([32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 32])
    if kind == "admit":
        seqs, length = _log(rng, 1, 16), _log(rng, 129, 8191)
        layers = rng.randint(1, 2)
        while seqs * length * kv_heads * layers > 8 * 8191 * 8 * 2:
            length = max(129, length // 2 + 1)
            if length == 129:
                kv_heads = max(1, kv_heads // 2)
        return dict(kind=kind, seqs=seqs, kv_heads=kv_heads, length=length, bits=bits, group=group,
                    residual=rng.choice([0, 128, 256]), layers=layers)
    if kind == "branch":
        return dict(kind=kind, seqs=_log(rng, 1, 16), each=rng.randint(1, 4), kv_heads=min(kv_heads, 8), length=_log(rng, 1, 1500), bits=bits,
                    group=group, layers=rng.randint(1, 8))
    if kind == "compact":
        return dict(kind=kind, seqs=2 * _log(rng, 1, 32), kv_heads=min(kv_heads, 8), length=_log(rng, 1, 2000), bits=bits, group=group,
                    layers=rng.randint(1, 4))
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8]) if kv_heads < 32 else 32
    new = rng.choice([1, 1, _log(rng, 2, 2048)])
    seqs = _log(rng, 1, 64) if new == 1 else _log(rng, 1, 8)
    context = new + _log(rng, 1, 131072 if new == 1 else 32768)
    # longer than the largest listed cases: shorter contexts
    while seqs * heads * new * context > TRIPLES or seqs * kv_heads * context * 4 * D > PAGE_BYTES // 2:
        context = new + (context - new) // 2
        if context <= new + 1:
            seqs, new = max(1, seqs // 2), max(1, new // 2)
            context = new + 100
    return dict(kind="attend", seqs=seqs, heads=heads, kv_heads=kv_heads, new=new, context=context, ragged=rng.random() < 0.5, bits=bits, group=group,
                residual=rng.choice([0, 128, 256]) + (new if new > 1 else 0), softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), alibi=rng.random() < 0.25,
                window=rng.choice([0, 0, _log(rng, 1, 8192)]), prefix=rng.choice([0, 0, _log(rng, 1, 500)]),
                documents=rng.choice([0, 0, 2, 5]) if new > 1 else 0, chunks=max(1, seqs // 4) if new > 1 and rng.random() < 0.5 else -1)


# ---- what the cases are made of, by their sizes alone ---------------------------------------------------------------------------------

def _pages(tokens):
    return -(-tokens // P)


def _lengths(case):
    """(length, new tokens) of every sequence of an attend case."""
    r = random.Random(case["context"] * 31 + case["seqs"])
    out = []
    for i in range(case["seqs"]):
        new = case["new"] if case["chunks"] < 0 or i < case["chunks"] else 1
        past = case["context"] - case["new"]
        if case["ragged"] and past > 1:
            past = r.randint(past // 2, past)
        out.append((past + new, new))
    return out


def _packed(length, residual):
    return max(0, length - residual) // P


def _firsts(case):
    """The first position that each new token sees, where chunks are made of several documents (each begins at a multiple of `size`); else None."""
    if not case["documents"]:
        return None
    out, size = [], max(1, case["context"] // case["documents"]) | 1
    for length, new in _lengths(case):
        out += [pos // size * size if new > 1 else 0 for pos in range(length - new, length)]
    return out


def _prefixes(case):
    """Up to which position each sequence's tokens all see each other: the chunk's first `prefix` ones do."""
    return [min(length, length - new + case["prefix"]) if case["prefix"] and new > 1 else 0 for length, new in _lengths(case)]


def _row_bytes(bits, group):
    """Bytes of one packed token of one kv head: codes, scales and minima of keys and values."""
    b = 0.0
    for bit in (int(bits[0]), int(bits[1])):
        groups = 12 if bit == 3 else D // group
        b += (48 if bit == 3 else D * bit // 8) + groups * 4
    return b


def work(case):
    if case["kind"] == "attend":
        firsts, at, flops, total = _firsts(case), 0, 0.0, 0.0
        for (length, new), prefix in zip(_lengths(case), _prefixes(case)):
            q, lo_all, pairs = _packed(length, case["residual"]) * P, length, 0
            for u in range(new):
                pos = length - new + u
                lo = 0 if firsts is None else firsts[at + u]
                if case["window"]:
                    lo = max(lo, pos + 1 - case["window"])
                hi = max(pos + 1, prefix)
                pairs += max(0, hi - lo)
                lo_all = min(lo_all, lo)
            at += new
            flops += 4.0 * D * pairs * case["heads"]
            total += case["kv_heads"] * (max(0, q - lo_all) * _row_bytes(case["bits"], case["group"]) + (length - max(q, lo_all)) * 4 * D)
            total += 4.0 * new * case["heads"] * D
        return {"bytes": total, "flops": flops}
    heads, layers = case["kv_heads"], case["layers"]
    if case["kind"] == "admit":
        full = _packed(case["length"], case["residual"]) * P
        one = case["length"] * 4 * D + full * _row_bytes(case["bits"], case["group"]) + (case["length"] - full) * 4 * D
        return {"bytes": one * heads * layers * case["seqs"], "flops": 0.0}
    if case["kind"] == "branch":
        last = P * 4 * D * 2 * heads * layers if case["length"] % P else 0
        return {"bytes": float(case["seqs"] * case["each"] * (last + 8 * _pages(case["length"]))), "flops": 0.0}
    packed = _packed(case["length"], P) * P
    moved = packed * _row_bytes(case["bits"], case["group"]) + (_pages(case["length"]) * P - packed) * 4 * D
    settled = packed * (4 * D + _row_bytes(case["bits"], case["group"]))
    return {"bytes": (2.0 * moved + settled) * heads * layers * (case["seqs"] // 2), "flops": 0.0}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------

def _kv(shape, gen, outliers):
    """[.., heads, D] fp16, N(0, 1); `outliers` [heads, D] multiplies the channels."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    return (x * outliers).half() if outliers is not None else x.half()


def _outliers(heads, gen):
    x = torch.ones(heads, D, device="cuda")
    return x.scatter_(1, torch.rand(heads, D, generator=gen, device="cuda").argsort(1)[:, :4], 8.0)


def _pool(n_packed, n_fp16, heads, bits, group):
    """Empty pages of one layer: (kcode, kscale, kmn, kfull, vcode, vscale, vmn, vfull, k_bits, v_bits, group)."""
    out = []
    for b in (int(bits[0]), int(bits[1])):
        words, groups = (12, 12) if b == 3 else (P // FIELDS[b], P // group)
        out += [torch.zeros(n_packed, heads, P, words, dtype=torch.int32, device="cuda"),
                torch.zeros(n_packed, heads, P, groups, dtype=torch.float16, device="cuda"),
                torch.zeros(n_packed, heads, P, groups, dtype=torch.float16, device="cuda"),
                torch.zeros(n_fp16, heads, P, D, dtype=torch.float16, device="cuda")]
    return tuple(out) + (int(bits[0]), int(bits[1]), group)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _book(slots, max_pages, n_packed, n_fp16):
    """Empty bookkeeping: table, length, packed, refs, free, count (free packed pages, free fp16 pages, status, 0)."""
    free = torch.cat([torch.arange(n_packed - 1, -1, -1), torch.arange(n_fp16 - 1, -1, -1)]).int().cuda()
    return (torch.full((slots, max_pages), -1, dtype=torch.int32, device="cuda"), torch.zeros(slots, dtype=torch.int32, device="cuda"),
            torch.zeros(slots, dtype=torch.int32, device="cuda"), torch.zeros(n_packed + n_fp16, dtype=torch.int32, device="cuda"), free,
            _i32([n_packed, n_fp16, 0, 0]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    heads, bits, group = case["kv_heads"], case["bits"], case["group"]
    if case["kind"] == "attend":
        sizes = _lengths(case)
        packed = [_packed(n, case["residual"]) for n, _ in sizes]
        pages = [_pages(n) for n, _ in sizes]
        n_packed, n_fp16 = sum(packed) + 3, sum(pages) - sum(packed) + 3
        layer = _pool(n_packed, n_fp16, heads, bits, group)
        out = _outliers(heads, gen)
        for at in range(0, n_packed, 512):                      # what is packed was fp16 once
            n = min(512, n_packed - at)
            for x, o in ((_kv((n, P, heads, D), gen, out).transpose(1, 2).transpose(2, 3), 0), (_kv((n, P, heads, D), gen, None).transpose(1, 2), 4)):
                for to, what in zip(layer[o:o + 3], _quantize(x.float(), layer[8 + o // 4], group)):
                    to[at:at + n] = what
        layer[3].copy_(_kv((n_fp16, P, heads, D), gen, out).transpose(1, 2))
        layer[7].normal_(generator=gen)
        perm, perm16 = (torch.randperm(n, generator=gen, device="cuda").tolist() for n in (n_packed, n_fp16))
        table = [[perm.pop() for _ in range(a)] + [perm16.pop() for _ in range(b - a)] for a, b in zip(packed, pages)]
        order = torch.randperm(len(sizes), generator=gen, device="cuda").tolist()     # sequences sit in any rows of the table
        book = _book(len(sizes), max(pages), n_packed, n_fp16)
        for i, row in enumerate(order):
            book[0][row, :pages[i]] = _i32(table[i])
        book[1][_i32(order).long()] = _i32([n for n, _ in sizes])
        book[2][_i32(order).long()] = _i32(packed)
        starts = [0]
        for _, new in sizes:
            starts.append(starts[-1] + new)
        s.update(book=book, n_packed=n_packed, layer=layer, rows=_i32(order), q_start=_i32(starts), max_new=max(new for _, new in sizes), max_tokens=max(n for n, _ in sizes),
                 q=torch.randn(starts[-1], case["heads"], D, generator=gen, device="cuda").half(), slopes=None, prefix=None, first=None)
        if case["alibi"]:
            s["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["heads"] + 1, device="cuda") / case["heads"])
        if case["prefix"]:
            s["prefix"] = _i32(_prefixes(case))
        if case["documents"]:
            s["first"] = _i32(_firsts(case))
        return s
    layers, length, seqs = case["layers"], case["length"], case["seqs"]
    pages = _pages(length)
    if case["kind"] == "admit":
        packed = _packed(length, case["residual"])
        # the prompts of the last pass are in the cache and leave
        s["n_packed"] = seqs * packed + 2
        s["book"] = _book(seqs, pages, s["n_packed"], seqs * pages + 2)
        s["layers"] = [_pool(s["n_packed"], seqs * pages + 2, heads, bits, group) for _ in range(layers)]
        out = _outliers(heads, gen)
        s["k"] = [_kv((seqs * length, heads, D), gen, out) for _ in range(layers)]
        s["v"] = [_kv((seqs * length, heads, D), gen, None) for _ in range(layers)]
        s["q_start"] = _i32([i * length for i in range(seqs + 1)])
        s["rows"] = _i32(torch.randperm(seqs, generator=gen, device="cuda").tolist())
        s["counts"] = _i32([length] * seqs)
        return s
    if case["kind"] == "branch":
        each = case["each"]
        packed, part = _packed(length, P), 1 if length % P else 0
        n_packed, n_fp16 = seqs * packed + 2, seqs * (pages - packed) + 2 * seqs * each * part + 2
        book = _book(seqs * (1 + each), pages + 1, n_packed, n_fp16)
        slots = torch.randperm(seqs * (1 + each), generator=gen, device="cuda").tolist()
        s["parents"], s["children"] = _i32([slots[i // each] for i in range(seqs * each)]), _i32(slots[seqs:])
        held = [(row, length, packed) for row in slots[:seqs]]
    else:
        packed = _packed(length, P)
        n_packed, n_fp16 = seqs * packed + 2, seqs // 2 * (2 * pages - packed) + 2
        book = _book(seqs, pages, n_packed, n_fp16)
        slots = torch.randperm(seqs, generator=gen, device="cuda").tolist()
        held = [(row, length, packed) for row in slots]
        s["turns"], s["turn"] = [_i32(slots[:seqs // 2]), _i32(slots[seqs // 2:])], [0]
        s["counts"] = _i32([length] * (seqs // 2))
    s["book"], s["n_packed"], s["layers"] = book, n_packed, [_pool(n_packed, n_fp16, heads, bits, group) for _ in range(layers)]
    for layer in s["layers"]:                                   # whatever the pages hold
        for i in (0, 4):
            layer[i].copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, layer[i].shape, generator=gen, device="cuda", dtype=torch.int32))
            for j in (1, 2, 3):
                layer[i + j].normal_(generator=gen)
    perm, perm16 = (torch.randperm(n, generator=gen, device="cuda").tolist() for n in (n_packed, n_fp16))
    used, used16, table = [], [], torch.full_like(book[0], -1).cpu()
    for row, n, a in held:
        ids, ids16 = [perm.pop() for _ in range(a)], [perm16.pop() for _ in range(_pages(n) - a)]
        table[row, :_pages(n)] = torch.tensor(ids + ids16, dtype=torch.int32)
        used, used16 = used + ids, used16 + ids16
        book[1][row], book[2][row] = n, a
    book[0].copy_(table)
    book[3][_i32(used + [n_packed + i for i in used16]).long()] = 1
    book[4][:len(perm)], book[4][n_packed:n_packed + len(perm16)] = _i32(sorted(perm, reverse=True)), _i32(sorted(perm16, reverse=True))
    book[5][:2] = _i32([len(perm), len(perm16)])
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------------------------

def _quantize(x, bits, group):
    """x [.., rows, 128] -> words, scale, minimum along the last axis."""
    size, n = (11, 12) if bits == 3 else (group, P // group)
    pad = n * size - P
    g = torch.nn.functional.pad(x, (0, pad), value=math.nan) if pad else x
    g = g.unflatten(-1, (n, size))
    there = g == g
    lo = torch.where(there, g, math.inf).amin(-1)
    hi = torch.where(there, g, -math.inf).amax(-1)
    top = 2.0 ** bits - 1
    scale = (hi - lo) / torch.full_like(lo, top)                # the true quotient: a division by a number is a product
    a = (g - lo[..., None]) / scale[..., None]
    whole = torch.trunc(a)
    code = whole + (a - whole >= 0.5)                           # halves away from zero
    code = torch.where(there & (a == a), code, 0.0).clamp_(0, top)
    if bits == 3:
        code[..., 10].clamp_(max=3.0)                           # the eleventh field has two bits
    shift = torch.arange(0, 33 if bits == 3 else 32, bits, device=x.device)
    word = (code.long() << shift).sum(-1) if bits == 3 else (code.long().flatten(-2).unflatten(-1, (-1, FIELDS[bits])) << shift).sum(-1)
    word = torch.where(word >= 2 ** 31, word - 2 ** 32, word).int()
    stored = (hi - lo) * torch.full_like(lo, 1.0).div_(torch.full_like(lo, top))
    return word, stored.half(), lo.half()


def _dequantize(word, scale, mn, bits, group):
    """[.., rows, words] -> [.., rows, 128] fp32."""
    shift = torch.arange(0, 33 if bits == 3 else 32, bits, device=word.device, dtype=torch.int32)
    code = (word[..., None] >> shift) & (2 ** bits - 1)
    if bits == 3:
        code[..., 10] &= 3
        return (code * scale[..., None].float() + mn[..., None].float()).flatten(-2)[..., :P]
    return (code.flatten(-2).unflatten(-1, (-1, group)) * scale[..., None].float() + mn[..., None].float()).flatten(-2)


def _attend_plain(s):
    table, length, packed = s["book"][:3]
    kcode, kscale, kmn, kfull, vcode, vscale, vmn, vfull, kb, vb, group = s["layer"]
    q, start, rows = s["q"], s["q_start"].long(), s["rows"].long()
    case, n = s["case"], s["rows"].numel()
    ids, j = table[rows].long(), torch.arange(table.shape[1], device="cuda")
    ids_p = torch.where(j < packed[rows][:, None], ids, 0)
    old = (j < packed[rows][:, None])[:, :, None, None, None]
    ids_f = torch.where((j >= packed[rows][:, None]) & (ids >= 0), ids, 0)
    k = torch.where(old, _dequantize(kcode[ids_p], kscale[ids_p], kmn[ids_p], kb, group).transpose(3, 4), kfull[ids_f].float())
    v = torch.where(old, _dequantize(vcode[ids_p], vscale[ids_p], vmn[ids_p], vb, group), vfull[ids_f].float())
    k, v = (x.transpose(1, 2).flatten(2, 3) for x in (k, v))    # [n, kv heads, tokens, D]
    tokens, heads, kv_heads, new = k.shape[2], q.shape[1], k.shape[1], s["max_new"]
    t = torch.arange(tokens, device="cuda")
    v = torch.where((t < length[rows][:, None])[:, None, :, None], v, 0.0)
    u = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(start, u, right=True) - 1
    pos = length[rows].long()[seq] - start[seq + 1] + u
    hi = pos + 1 if s["prefix"] is None else torch.maximum(pos + 1, s["prefix"].long()[seq])
    hi = torch.minimum(hi, length[rows].long()[seq])
    lo = torch.zeros_like(pos) if s["first"] is None else s["first"].long()
    lo = torch.maximum(lo, pos + 1 - case["window"]) if case["window"] else lo
    padded = torch.zeros(n, new, heads, D, device="cuda")
    padded[seq, u - start[seq]] = q.float()
    bounds = torch.zeros(n, new, 3, dtype=torch.long, device="cuda")
    bounds[seq, u - start[seq]] = torch.stack([lo, hi, pos], 1)
    rep = heads // kv_heads
    score = padded.unflatten(2, (kv_heads, rep)).permute(0, 2, 3, 1, 4).flatten(2, 3) @ k.transpose(2, 3)
    score = score.unflatten(2, (rep, new)).mul_(1.0 / math.sqrt(D))                    # [n, kv heads, rep, new, tokens]
    if case["softcap"]:
        score = score.div_(case["softcap"]).tanh_().mul_(case["softcap"])
    if s["slopes"] is not None:
        score += s["slopes"].view(kv_heads, rep, 1, 1) * (t - bounds[:, :, 2:])[:, None, None].float()
    seen = ((t >= bounds[:, :, :1]) & (t < bounds[:, :, 1:2]))[:, None, None]
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = e.sum(-1, keepdim=True)
    out = (e.flatten(2, 3) @ v).unflatten(2, (rep, new)) / torch.where(total > 0, total, 1.0)
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, u - start[seq]].half()


def _held(book, rows):
    """Which of the rows' table entries are packed, and which are fp16 pages."""
    table, length, packed = book[:3]
    j = torch.arange(table.shape[1], device="cuda")
    return j < packed[rows][:, None], (j >= packed[rows][:, None]) & (j < (length[rows][:, None] + P - 1) // P)


def _give_back(book, ids, where, n_packed):
    """One reference less for the pages `ids` (fp16 pages behind the packed ones) where `where`; the free ones go on their stacks by their numbers."""
    refs, free, count = book[3:]
    more = torch.zeros(refs.numel() + 1, dtype=torch.int32, device="cuda")
    more.index_add_(0, torch.where(where, ids, refs.numel()).flatten(), torch.ones(ids.numel(), dtype=torch.int32, device="cuda"))
    had = refs > 0
    refs -= more[:-1]
    gone = had & (refs <= 0)
    numbers = torch.arange(refs.numel(), device="cuda")
    packed = numbers < n_packed
    place = torch.where(packed, count[0] + (gone & packed).cumsum(0) - 1, n_packed + count[1] + (gone & ~packed).cumsum(0) - 1)
    wide = torch.cat([free, free[:1]])
    wide[torch.where(gone, place, refs.numel())] = torch.where(packed, numbers, numbers - n_packed).int()
    free.copy_(wide[:-1])
    count[:2] += torch.stack([(gone & packed).sum(), (gone & ~packed).sum()]).int()


def _free_plain(book, rows, n_packed):
    rows = rows.long()
    table, length, packed = book[:3]
    old, new = _held(book, rows)
    ids = table[rows].long()
    _give_back(book, torch.where(old, ids, ids + n_packed), old | new, n_packed)
    table[rows], length[rows], packed[rows] = -1, 0, 0


def _extend_plain(book, rows, counts, n_packed):
    rows = rows.long()
    table, length, packed, refs, free, count = book
    have = (length[rows] + P - 1) // P
    need = (length[rows] + counts + P - 1) // P - have
    before = need.cumsum(0) - need
    granted = need.sum() <= count[1]                            # all of them or none
    j = torch.arange(table.shape[1], device="cuda")
    k = j - have[:, None]
    fill = (k >= 0) & (k < need[:, None]) & granted
    ids = free[torch.where(fill, n_packed + count[1] - 1 - before[:, None] - k, 0).long()]
    table[rows] = torch.where(fill, ids, table[rows])
    wide = torch.cat([refs, refs[:1]])
    wide[torch.where(fill, ids.long() + n_packed, refs.numel())] = 1
    refs.copy_(wide[:-1])
    length[rows] += torch.where(granted, counts, 0)
    count[1] -= torch.where(granted, need, 0).sum().int()
    count[2] |= (~granted).int()


def _write_plain(book, layer, k, v, start, rows):
    table, length = book[0], book[1]
    start, rows = start.long(), rows.long()
    u = torch.arange(k.shape[0], device="cuda")
    seq = torch.searchsorted(start, u, right=True) - 1
    pos = length[rows].long()[seq] - start[seq + 1] + u
    page = table[rows[seq], pos // P].long()
    layer[3][page, :, pos % P], layer[7][page, :, pos % P] = k, v


def _settle_plain(book, layers, rows, window, n_packed):
    rows = rows.long()
    table, length, packed, refs, free, count = book
    want = torch.maximum(packed[rows], (length[rows] - window).clamp(min=0) // P)
    need = want - packed[rows]
    before = need.cumsum(0) - need
    granted = need.sum() <= count[0]
    j = torch.arange(table.shape[1], device="cuda")
    k = j - packed[rows][:, None]
    move = (k >= 0) & (k < need[:, None]) & granted
    to = free[torch.where(move, count[0] - 1 - before[:, None] - k, 0).long()].long()
    src = table[rows].long()
    table[rows] = torch.where(move, to.int(), table[rows])
    wide = torch.cat([refs, refs[:1]])
    wide[torch.where(move, to, refs.numel())] = 1
    refs.copy_(wide[:-1])
    packed[rows] = torch.where(granted, want, packed[rows])
    count[0] -= torch.where(granted, need, 0).sum().int()
    count[2] |= (~granted).int() * 2
    _give_back(book, src + n_packed, move, n_packed)
    src, dst = src[move], to[move]
    for layer in layers:
        kq, vq = _quantize(layer[3][src].float().transpose(2, 3), layer[8], layer[10]), _quantize(layer[7][src].float(), layer[9], layer[10])
        layer[0][dst], layer[1][dst], layer[2][dst], layer[4][dst], layer[5][dst], layer[6][dst] = kq + vq


def _branch_plain(book, parents, children, n_packed):
    parents, children = parents.long(), children.long()
    table, length, packed, refs, free, count = book
    need = (length[parents] % P > 0).int()
    before = need.cumsum(0) - need
    granted = need.sum() <= count[1]
    to = free[(n_packed + count[1] - 1 - before).clamp(min=n_packed).long()].long()
    old, new = _held(book, parents)
    j = torch.arange(table.shape[1], device="cuda")
    last = need.bool()[:, None] & (j == length[parents][:, None] // P)
    ids = table[parents].long()
    src = ids.gather(1, (length[parents].long() // P).clamp(max=table.shape[1] - 1)[:, None])[:, 0]
    every = torch.zeros(refs.numel() + 1, dtype=torch.int32, device="cuda")
    shared = (old | new) & ~last & granted
    every.index_add_(0, torch.where(shared, torch.where(old, ids, ids + n_packed), refs.numel()).flatten(),
                     torch.ones(ids.numel(), dtype=torch.int32, device="cuda"))
    copied = need.bool() & granted
    every.index_add_(0, torch.where(copied, to + n_packed, refs.numel()), torch.ones_like(need))
    refs += every[:-1]
    table[children] = torch.where(granted, torch.where(last, to[:, None], ids).int(), table[children])
    length[children] = torch.where(granted, length[parents], length[children])
    packed[children] = torch.where(granted, packed[parents], packed[children])
    count[1] -= torch.where(granted, need, 0).sum().int()
    count[2] |= (~granted).int()
    return src[copied], to[copied]


def _close_up(refs, free, count):
    """One pool: the live pages beyond the number of live pages go to the free ones below it.  New number of each page."""
    n = refs.numel()
    live = refs > 0
    total = live.sum()
    numbers = torch.arange(n, device="cuda")
    goes, hole = live & (numbers >= total), ~live & (numbers < total)
    holes = torch.zeros(n + 1, dtype=torch.long, device="cuda")
    holes[torch.where(hole, hole.cumsum(0) - 1, n)] = numbers
    to = torch.where(goes, holes[(goes.cumsum(0) - 1).clamp(min=0)], numbers)
    kept = refs.clone()
    refs.copy_(torch.where(numbers < total, refs, 0))
    wide = torch.cat([refs, refs[:1]])
    wide[torch.where(goes, to, n)] = kept
    refs.copy_(wide[:-1])
    free.copy_(torch.where(numbers < n - total, n - 1 - numbers, free.long()).int())
    count.copy_((n - total).int())
    return to, numbers[goes], to[goes]


def _compact_plain(book, layers, n_packed):
    table, length, packed, refs, free, count = book
    to, src, dst = _close_up(refs[:n_packed], free[:n_packed], count[0])
    to16, src16, dst16 = _close_up(refs[n_packed:], free[n_packed:], count[1])
    old, new = _held(book, torch.arange(table.shape[0], device="cuda"))
    at = table.long().clamp(min=0)
    table.copy_(torch.where(old, to[torch.where(old, at, 0)], torch.where(new, to16[torch.where(new, at, 0)], -1)).int())
    for layer in layers:
        for i in (0, 4):
            layer[i][dst], layer[i + 1][dst], layer[i + 2][dst], layer[i + 3][dst16] = layer[i][src], layer[i + 1][src], layer[i + 2][src], layer[i + 3][src16]


def run(s):
    case = s["case"]
    if own:
        import kvmix_b200 as kv
        pages = kv.PageBook(*s["book"], s["n_packed"])
        if case["kind"] == "attend":
            return kv.paged_attention(s["q"], s["q_start"], s["rows"], pages, kv.PageLayer(*s["layer"]), window=case["window"], prefix=s["prefix"],
                                      first=s["first"], softcap=case["softcap"], alibi_slopes=s["slopes"], max_new=s["max_new"], max_tokens=s["max_tokens"])
        layers = [kv.PageLayer(*layer) for layer in s["layers"]]
        if case["kind"] == "admit":
            kv.pages_free(s["rows"], pages)
            kv.pages_extend(s["rows"], s["counts"], pages)
            for layer, k, v in zip(layers, s["k"], s["v"]):
                kv.page_write(k, v, s["q_start"], s["rows"], pages, layer)
            kv.pages_settle(s["rows"], case["residual"], pages, layers)
        elif case["kind"] == "branch":
            kv.pages_free(s["children"], pages)
            kv.pages_fork(s["parents"], s["children"], pages, layers)
        else:
            rows = s["turns"][s["turn"][0]]
            kv.pages_free(rows, pages)
            kv.pages_compact(pages, layers)
            kv.pages_extend(rows, s["counts"], pages)
            kv.pages_settle(rows, P, pages, layers)
            s["turn"][0] ^= 1
    else:
        if case["kind"] == "attend":
            return _attend_plain(s)
        book, layers, n_packed = s["book"], s["layers"], s["n_packed"]
        if case["kind"] == "admit":
            _free_plain(book, s["rows"], n_packed)
            _extend_plain(book, s["rows"], s["counts"], n_packed)
            for layer, k, v in zip(layers, s["k"], s["v"]):
                _write_plain(book, layer, k, v, s["q_start"], s["rows"])
            _settle_plain(book, layers, s["rows"], case["residual"], n_packed)
        elif case["kind"] == "branch":
            _free_plain(book, s["children"], n_packed)
            src, dst = _branch_plain(book, s["parents"], s["children"], n_packed)
            for layer in layers:
                layer[3][dst], layer[7][dst] = layer[3][src], layer[7][src]
        else:
            rows = s["turns"][s["turn"][0]]
            _free_plain(book, rows, n_packed)
            _compact_plain(book, layers, n_packed)
            _extend_plain(book, rows, s["counts"], n_packed)
            _settle_plain(book, layers, rows, P, n_packed)
            s["turn"][0] ^= 1
    # of the pages that a branch takes only fp16 ones are written
    return {"book": s["book"], "layers": [layer[3:8:4] if case["kind"] == "branch" else layer[:8] for layer in s["layers"]]}


# ---- from the definition, in 64 bits ----------------------------------------------------------------------------------------------------

def _page_exact(word, scale, mn, bits, group):
    """One page of one head in 64 bits: [128 rows, 128]."""
    size = 11 if bits == 3 else group
    cols = torch.arange(P, device=word.device)
    per = FIELDS[bits]
    at = cols % per
    w = word.long()[..., cols // per] & 0xffffffff
    code = torch.div(w, torch.tensor([2 ** int(i * bits) for i in range(per)], device=word.device)[at], rounding_mode="floor") % 2 ** bits
    if bits == 3:
        code = torch.where(at == 10, code % 4, code)
    return code.double() * scale.double()[..., cols // size] + mn.double()[..., cols // size]


def _exact_attend(s):
    case = s["case"]
    kcode, kscale, kmn, kfull, vcode, vscale, vmn, vfull, kb, vb, group = s["layer"]
    table, lengths, packed = (x.cpu() for x in s["book"][:3])
    starts, rows = s["q_start"].tolist(), s["rows"].tolist()
    firsts = None if s["first"] is None else s["first"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    rep = s["q"].shape[1] // kfull.shape[1]
    for i, row in enumerate(rows):
        n, a, new = int(lengths[row]), int(packed[row]), starts[i + 1] - starts[i]
        ids = table[row].long().cuda()
        pos = torch.arange(n - new, n, device="cuda")
        key = torch.arange(n, device="cuda")
        seen = key[None] <= pos[:, None]
        if case["prefix"]:
            seen = seen | (key[None] < int(s["prefix"][i]))
        if case["window"]:
            seen = seen & (key[None] > pos[:, None] - case["window"])
        if firsts is not None:
            seen = seen & (key[None] >= torch.tensor(firsts[starts[i]:starts[i + 1]], device="cuda")[:, None])
        for g in range(kfull.shape[1]):
            one = ids[:a]
            k = torch.cat([_page_exact(kcode[one, g], kscale[one, g], kmn[one, g], kb, group).transpose(1, 2).reshape(-1, D),
                           kfull[ids[a:_pages(n)], g].double().reshape(-1, D)])[:n]
            v = torch.cat([_page_exact(vcode[one, g], vscale[one, g], vmn[one, g], vb, group).reshape(-1, D),
                           vfull[ids[a:_pages(n)], g].double().reshape(-1, D)])[:n]
            for h in range(g * rep, (g + 1) * rep):
                score = s["q"][starts[i]:starts[i + 1], h].double() @ k.T / math.sqrt(D)
                if case["softcap"]:
                    score = case["softcap"] * torch.tanh(score / case["softcap"])
                if case["alibi"]:
                    score = score - s["slopes"][h].double() * (pos[:, None] - key[None])
                score = torch.where(seen, score, -math.inf)
                weight = torch.softmax(score, -1).nan_to_num(0.0)
                out[starts[i]:starts[i + 1], h] = weight @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(s)
    if case["kind"] != "admit":
        return None
    # which packed page the settled ones went to follows from the stacks, which start in order: sequences in the order of `rows`, and their pages
    n, row_start, full = case["length"], s["q_start"].tolist(), _packed(case["length"], case["residual"])
    layers = []
    for layer, k, v in zip(s["layers"], s["k"], s["v"]):
        sides = []
        for x, bits, by_token in ((k, case["bits"][0], False), (v, case["bits"][1], True)):
            bits, scale, low = int(bits), torch.zeros(layer[1 if not by_token else 5].shape, dtype=torch.float64, device="cuda"), None
            low = scale.clone()
            size = 11 if bits == 3 else case["group"]
            for i in range(case["seqs"]):
                for p in range(full):
                    block = x[row_start[i] + p * P:row_start[i] + (p + 1) * P].double()       # [tokens, heads, channels]
                    block = block.permute(1, 0, 2) if by_token else block.permute(1, 2, 0)
                    parts = block.split(size, -1)
                    low[i * full + p] = torch.stack([t.amin(-1) for t in parts], -1)
                    scale[i * full + p] = torch.stack([(t.amax(-1) - t.amin(-1)) / (2 ** bits - 1) for t in parts], -1)
            sides += [None, scale, low, None]
        layers.append(sides)
    return {"book": [None] * 6, "layers": layers}
