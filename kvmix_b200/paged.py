"""A paged mixed-precision KV cache: sequences of any length that come, grow, branch and go in one pool of pages.

Upstream threads one tuple of tensors per batch through its forward (models/modeling_llama_KVmix.py:269-273), as ``KVmixLayerCache``
does; sequences of one batch then have one length, none can leave or join, and two that begin alike hold everything twice.  Here
a page holds 128 tokens of one sequence, the same page number in every layer.  A sequence's oldest pages are packed at the layer's
bit widths, its newest are fp16 (``include/kvmix_b200.h`` has the layouts, which are the layer cache's page by page).

    pages_extend     new tokens' pages                    page_write       their keys and values, layer by layer
    paged_attention  one new token or chunks of them      pages_settle     full pages that leave the fp16 window are quantized
    pages_fork       a sequence branches                  pages_free       a sequence goes
    pages_compact    pages in use move together           pages_reorder    rows take one another's sequences (beam search)
    page_append      page_write with the position rotation, for queries too
    paged_differential_attention  the difference of two softmax maps, over the same pages
    KVmixPagedCache  all of them with the tensors they work on

The bookkeeping (``PageBook``) lives on the device and is changed by kernels only: no call waits for the host, all can be captured in a
CUDA graph.  A call that cannot be done in full -- no page left, a row named twice -- does nothing but set a bit of ``count[2]``, and
until that is cleared every call that changes the cache does nothing (``KVmixPagedCache.check`` raises and clears).  An attention
that gave up waiting (its output is lost, the cache is whole) and a ``page_write`` or ``page_append`` that left tokens out set bits that hold nothing up.  The attention is
softmax attention over the dequantised cache with scores, softmax and sums in fp32 (scores are not narrowed to fp16 as ``decode_attention`` does by
default).  What is rounded to fp16 on the way to the tensor cores: weights; for several new tokens (and more than 8 query heads a kv head) dequantised
keys and values; for one new token those of 3 bits, and weight * scale of a value.
"""
import ctypes as C
import functools
import math
import struct
from typing import NamedTuple

import torch

from . import _lib, ops
from ._lib import check
from .beams import beam_select

PAGE_TOKENS = 128
_SCALE = 1.0 / math.sqrt(128)
_MOST = 1 << 30                  # no sequence is longer: wider windows are this one
_MOST_HEADS = 1 << 15            # what kvq_page_copy takes as one page: 1 GB
_STATUS = {1: "no free fp16 page", 2: "no free packed page", 4: "sequence longer than the table", 8: "bad rows (outside the table, named twice, "
           "a child that is not empty or also a parent)", 16: "an attention gave up waiting for its own copies, its output is not to be used",
           32: "new tokens were not written, their page is packed, shared or not there", 64: "new tokens were not written, their positions are "
           "outside the tables of angles"}

_pack_book, _pack_layer = struct.Struct("@6P4i").pack, struct.Struct("@8P6i").pack
_pack_write, _pack_attn = struct.Struct("@2P4q2P2i").pack, struct.Struct("@2P4q5P8i2fPQ").pack
_pack_diff = struct.Struct("@2P4q5P8i2fPQ2Pf").pack
_pack_append = struct.Struct("@6P10q3P8i").pack
_addresses = struct.Struct("@8P").unpack_from             # of a layer's argument block
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class PageBook(NamedTuple):
    """Who holds which page: int32 tensors on the device, shared by all layers.

    ``table`` [slots, max_pages], ``length`` [slots] tokens, ``packed`` [slots] packed pages, ``refs`` and ``free_ids`` [packed + fp16 pages],
    ``count`` [4]: free packed pages, free fp16 pages, status, 0.  ``n_packed``: packed pages in the pool."""
    table: torch.Tensor
    length: torch.Tensor
    packed: torch.Tensor
    refs: torch.Tensor
    free_ids: torch.Tensor
    count: torch.Tensor
    n_packed: int


class PageLayer(NamedTuple):
    """One layer's pages.  Keys ``kcode`` [n, Hkv, 128 channels, words], ``kscale``/``kmn`` [n, Hkv, 128 channels, groups]; values ``vcode``
    [n, Hkv, 128 tokens, words], ``vscale``/``vmn`` alike; ``kfull``/``vfull`` [n16, Hkv, 128 tokens, 128 channels] fp16; contiguous.
    words = 4 * bits, groups = 128 // group (12 and 12 at 3 bits)."""
    kcode: torch.Tensor
    kscale: torch.Tensor
    kmn: torch.Tensor
    kfull: torch.Tensor
    vcode: torch.Tensor
    vscale: torch.Tensor
    vmn: torch.Tensor
    vfull: torch.Tensor
    k_bits: int
    v_bits: int
    group: int


def page_words(bits):
    """Words of 128 packed elements."""
    return 12 if bits == 3 else 4 * bits


def page_groups(bits, group):
    """Groups of 128 elements (3 bits: groups of 11, the last of 7)."""
    return 12 if bits == 3 else PAGE_TOKENS // group


@functools.lru_cache(maxsize=None)
def _library():
    for fmt, cls in (("@6P4i", _lib.PageBookArgs), ("@8P6i", _lib.PageLayerArgs), ("@2P4q2P2i", _lib.PageWriteArgs), ("@2P4q5P8i2fPQ", _lib.PagedAttnArgs),
                     ("@6P10q3P8i", _lib.PageAppendArgs), ("@2P4q5P8i2fPQ2Pf", _lib.PagedDiffArgs)):
        assert -(-struct.calcsize(fmt) // 8) * 8 == C.sizeof(cls)
    return _lib.lib()


@functools.lru_cache(maxsize=None)
def _launch_count():
    """(the library's count of launches, what ops.LAUNCHES has of it)"""
    return C.c_uint32.in_dll(_library(), "kvq_paged_launch_count"), [0]


_i32, _f16 = torch.int32, torch.float16
_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def _ints(dev, name, t, n):
    """Address of an int32 [n] on device number `dev`."""
    if t.dtype is _i32 and t.get_device() == dev and t.dim() == 1 and t.numel() == n and t.is_contiguous():
        return t.data_ptr()
    raise RuntimeError(f"{name} must be a contiguous int32 tensor [{n}] on cuda:{dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _book(pages):
    """(device number, argument block) of a PageBook."""
    table, length, packed, refs, free_ids, count, n_packed = pages
    dev = table.get_device()
    if dev < 0:
        raise RuntimeError("kvmix_b200 operators need CUDA tensors (there is no CPU path)")
    if table.dtype is not _i32 or table.dim() != 2 or not table.is_contiguous():
        raise RuntimeError("the page table is a contiguous int32 tensor [slots, max_pages]")
    (slots, max_pages), total = table.shape, refs.numel()
    if not 0 <= n_packed <= total:
        raise RuntimeError("n_packed is the number of packed pages among refs")
    return dev, _pack_book(table.data_ptr(), _ints(dev, "length", length, slots), _ints(dev, "packed", packed, slots), _ints(dev, "refs", refs, total),
                           _ints(dev, "free_ids", free_ids, total), _ints(dev, "count", count, 4), slots, max_pages, n_packed, total - n_packed)


def _page_tensor(dev, t, dtype, shape):
    # the address is asked for in the same breath: a layer has eight such tensors, a call of many layers hundreds
    if t.dtype is dtype and t.shape == shape and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    raise RuntimeError(f"page tensor {tuple(t.shape)} {t.dtype} on {t.device}: contiguous {dtype} {shape} on cuda:{dev} expected")


def _movable(layers, addresses):
    """What kvq_page_copy and kvq_page_pack would refuse, before the bookkeeping that they come behind and that cannot be taken back."""
    low = 0
    for at in addresses:
        low |= at
    if low & 15:
        check(-13)
    if any(layer.kfull.shape[1] > _MOST_HEADS for layer in layers):
        raise RuntimeError(f"pages hold at most {_MOST_HEADS} kv heads")


def _fp16_pages(pages, dev, layer):
    """Addresses of a layer's fp16 pages."""
    kfull, vfull = layer.kfull, layer.vfull
    shape = (pages.refs.numel() - pages.n_packed, kfull.shape[1], PAGE_TOKENS, 128)
    return _page_tensor(dev, kfull, _f16, shape), _page_tensor(dev, vfull, _f16, shape)


def _layer(pages, dev, layer):
    """Argument block of a PageLayer that goes with the book."""
    kcode, kscale, kmn, kfull, vcode, vscale, vmn, vfull, kb, vb, group = layer
    if kb not in (1, 2, 3, 4) or vb not in (1, 2, 3, 4):
        check(-1)
    if group not in (32, 64, 128):
        raise RuntimeError("pages are quantized in groups of 32, 64 or 128")
    n, heads = pages.n_packed, kfull.shape[1]
    n16 = pages.refs.numel() - n
    kw, vw, kg, vg = (n, heads, PAGE_TOKENS, page_words(kb)), (n, heads, PAGE_TOKENS, page_words(vb)), (n, heads, PAGE_TOKENS, page_groups(kb, group)), \
        (n, heads, PAGE_TOKENS, page_groups(vb, group))
    full = (n16, heads, PAGE_TOKENS, 128)
    return _pack_layer(_page_tensor(dev, kcode, _i32, kw), _page_tensor(dev, kscale, _f16, kg), _page_tensor(dev, kmn, _f16, kg), _page_tensor(dev, kfull, _f16, full),
                       _page_tensor(dev, vcode, _i32, vw), _page_tensor(dev, vscale, _f16, vg), _page_tensor(dev, vmn, _f16, vg), _page_tensor(dev, vfull, _f16, full),
                       heads, kb, vb, group, n, n16)


def _rows(dev, name, rows):
    return _ints(dev, name, rows, rows.numel())


def _rows_apart(out):
    """Whether no two of the rows [tokens, heads] of 128 channels share an element (as no layout of one axis inside the other has it)."""
    (inner, n), (outer, m) = sorted((stride, size) for stride, size in zip(out.stride()[:2], out.shape[:2]))
    return (n <= 1 or inner >= 128) and (m <= 1 or outer >= (128 if n <= 1 else inner * (n - 1) + 128))


def _on_its_device(where):
    """Kernels are launched on the current stream of the tensors' device, whichever is current.  `where`: place of `pages` among the arguments."""
    def wrap(f):
        @functools.wraps(f)
        def call(*args, **kwargs):
            dev = (args[where] if len(args) > where else kwargs["pages"]).table.get_device()
            if dev < 0 or dev == _current_device():
                return f(*args, **kwargs)
            with torch.cuda.device(dev):
                return f(*args, **kwargs)
        return call
    return wrap


def _launched(rc):
    if rc:
        check(rc)
    count, seen = _launch_count()
    now = count.value
    new = (now - seen[0]) & 0xffffffff
    if new < 1 << 31:                                 # else another thread was here between
        ops.LAUNCHES[0] += new
        seen[0] = now


def _copy(tensors, moves, max_moves, how=None):
    """Pages of tensors given as (address, bytes of a page), from and to the numbers in `moves`: whole, or as `how` copies them."""
    how = how or _library().kvq_page_copy
    for at in range(0, len(tensors), 2 * _lib.MAX_PAGE_TENSORS):
        some = tensors[at:at + 2 * _lib.MAX_PAGE_TENSORS]
        _launched(how(struct.pack("@" + "Pq" * (len(some) // 2), *some), len(some) // 2, moves, max_moves, ops.raw_stream()))


@_on_its_device(2)
def pages_extend(rows, counts, pages):
    """``length[rows[i]] += counts[i]``, with the fp16 pages that takes.  rows, counts: int32 [n] on the device, no row twice."""
    dev, book = _book(pages)
    _launched(_library().kvq_pages_extend(book, _rows(dev, "rows", rows), _ints(dev, "counts", counts, rows.numel()), rows.numel(), ops.raw_stream()))


@_on_its_device(1)
def pages_free(rows, pages):
    """The rows' sequences go; pages that nobody holds any more are free."""
    dev, book = _book(pages)
    _launched(_library().kvq_pages_free(book, _rows(dev, "rows", rows), rows.numel(), ops.raw_stream()))


@_on_its_device(4)
def page_write(k, v, q_start, rows, pages, layer):
    """Keys (rotated) and values of new tokens into one layer's fp16 pages.  k, v [tokens, Hkv, 128] fp16, any strides; tokens
    [q_start[i], q_start[i+1]) are the last ones of sequence rows[i], which ``pages_extend`` has counted already.  Tokens whose page
    is packed, not there or held by another sequence too are left out, and a status bit says so."""
    dev, book = _book(pages)
    heads = layer.kfull.shape[1]
    if k.dim() != 3 or k.shape[1:] != (heads, 128) or v.shape != k.shape or k.dtype is not torch.float16 or v.dtype is not torch.float16:
        raise RuntimeError(f"page_write takes fp16 keys and values [tokens, {heads}, 128]")
    if k.get_device() != dev or v.get_device() != dev:
        raise RuntimeError(f"keys and values must be on cuda:{dev}")
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    n = rows.numel()
    a = _pack_write(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), _ints(dev, "q_start", q_start, n + 1),
                    _rows(dev, "rows", rows), n, k.shape[0])
    _launched(_library().kvq_page_write(book, _layer(pages, dev, layer), a, ops.raw_stream()))


@_on_its_device(6)
def page_append(k, v, cos, sin, q_start, rows, pages, layer, q=None, q_out=None, positions=None, interleaved=False, parts=1):
    """``page_write`` of keys and values from the projections: keys are rotated by their positions' angles on the way, and so are the step's queries.

    k, v [tokens, Hkv, 128], q [tokens, nh, 128]: fp16, bf16 or fp32, one type, any strides.  cos, sin fp32 [positions, angles], contiguous along the angles, angles a
    multiple of 8: pair i of a head's channels, (i, i + angles) or, interleaved, (2i, 2i + 1), is turned by angle i of the token's row; channels from 2 * angles on stay.
    parts = 2: the two halves of a head are turned each for itself (``paged_differential_attention``), angles up to 32 then.  A token's row is its
    place in the sequence, or positions[token] (int32 [tokens]).  Rotations are fp32 products and sums, rounded once to fp16.
    Tokens that ``page_write`` would leave out are left out; those whose position is outside the tables too, their queries with them, and a
    status bit says so.  Returns the queries, fp16 (q_out where it is given, which may be q itself; None without q); rows behind q_start[n] are left as they are, and
    all of them while an earlier call stands refused."""
    dev, book = _book(pages)
    kfull, kind, shape = layer.kfull, k.dtype, k.shape
    heads = kfull.shape[1]
    if len(shape) != 3 or shape[1] != heads or shape[2] != 128 or v.shape != shape or v.dtype is not kind or kind not in _TYPES:
        raise RuntimeError(f"page_append takes keys and values [tokens, {heads}, 128] of one type, fp16, bf16 or fp32")
    if k.get_device() != dev or v.get_device() != dev or cos.get_device() != dev or sin.get_device() != dev or (q is not None and q.get_device() != dev):
        raise RuntimeError(f"keys, values, queries and angles must be on cuda:{dev}")
    if cos.dim() != 2 or sin.shape != cos.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise RuntimeError("cos and sin must be float32 [positions, angles]")
    tokens, (angle_rows, angles), (c_sT, c_s), (s_sT, s_s) = shape[0], cos.shape, cos.stride(), sin.stride()
    if parts not in (1, 2) or angles % 8 or not 0 < angles <= 64 // parts:
        raise RuntimeError("angles must be a multiple of 8, at most 64 / parts; parts 1 or 2")
    if c_s != 1 or s_s != 1:
        raise RuntimeError("cos and sin must be contiguous along the angles")
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    at_q = at_out = nh = q_sT = q_sH = o_sT = o_sH = 0
    if q is not None:
        if q.dim() != 3 or q.shape[0] != tokens or q.shape[2] != 128 or q.dtype is not kind:
            raise RuntimeError(f"queries must be [{tokens}, heads, 128] of the keys' type")
        nh = q.shape[1]
        if q_out is None:
            q_out = q.new_empty((tokens, nh, 128)) if kind is _f16 else q.new_empty((tokens, nh, 128), dtype=_f16)
        elif q_out.shape != q.shape or q_out.dtype is not _f16 or q_out.get_device() != dev or q_out.stride(2) != 1 or not _rows_apart(q_out):
            raise RuntimeError("q_out must be fp16 like q, contiguous along the channels, its rows apart")
        if q.stride(2) != 1:
            q = q.contiguous()
        at_q, at_out, (q_sT, q_sH, _), (o_sT, o_sH, _) = q.data_ptr(), q_out.data_ptr(), q.stride(), q_out.stride()
    elif q_out is not None:
        raise RuntimeError("q_out without q")
    n, (k_sT, k_sH, _), (v_sT, v_sH, _) = rows.numel(), k.stride(), v.stride()
    at_k, at_v = _fp16_pages(pages, dev, layer)
    block = _pack_layer(0, 0, 0, at_k, 0, 0, 0, at_v, heads, layer.k_bits, layer.v_bits, layer.group, 0, kfull.shape[0])        # packed pages are not touched
    a = _pack_append(k.data_ptr(), v.data_ptr(), at_q, at_out, cos.data_ptr(), sin.data_ptr(), k_sT, k_sH, v_sT, v_sH, q_sT, q_sH, o_sT, o_sH, c_sT, s_sT,
                     _ints(dev, "q_start", q_start, n + 1), _ints(dev, "rows", rows, n), 0 if positions is None else _ints(dev, "positions", positions, tokens), n, tokens, nh,
                     _TYPES[kind], angles, angle_rows, parts, 1 if interleaved else 0)
    _launched(_library().kvq_page_append(book, block, a, ops.raw_stream()))
    return q_out


@_on_its_device(2)
def pages_settle(rows, window, pages, layers):
    """Full pages that end ``window`` tokens or more before their sequence's end are quantized in every layer and their fp16 pages given
    back.  Sequences that share an fp16 page settle it each for itself."""
    dev, book = _book(pages)
    if window < 0:
        raise RuntimeError("window must not be negative")
    moves = pages.count.new_empty(4 + 2 * pages.n_packed)
    blocks, n = [_layer(pages, dev, layer) for layer in layers], rows.numel()
    for block in blocks:
        _movable((), _addresses(block))
    L, st, at = _library(), ops.raw_stream(), moves.data_ptr()
    _launched(L.kvq_pages_settle(book, _rows(dev, "rows", rows), n, int(min(window, _MOST)), at, st))
    for block in blocks:
        _launched(L.kvq_page_pack(block, at, min(pages.n_packed, n * pages.table.shape[1]), st))


@_on_its_device(2)
def pages_fork(parents, children, pages, layers):
    """Row children[i] (empty) becomes a copy of row parents[i]: full pages are shared, a last page that is not full is copied in every
    layer.  A parent may have several children; no row is both."""
    dev, book = _book(pages)
    n, tensors = parents.numel(), []
    for layer in layers:
        size = layer.kfull.shape[1] * PAGE_TOKENS * 256
        for at in _fp16_pages(pages, dev, layer):
            tensors += (at, size)
    _movable(layers, tensors[::2])
    moves = pages.count.new_empty(4 + 2 * n)
    _launched(_library().kvq_pages_fork(book, _rows(dev, "parents", parents), _ints(dev, "children", children, n), n, moves.data_ptr(), ops.raw_stream()))
    _copy(tensors, moves.data_ptr(), n)


@_on_its_device(2)
def pages_reorder(rows, parents, pages, layers, beams=None):
    """Rows take one another's sequences, all at once: row rows[i] becomes what row parents[i] was before the call (int32 [n] each, no row twice).  With ``beams``, n
    is a multiple of it and parents[i] counts within i's group of that many rows, as ``beam_select`` gives it.  A parent may be taken by several rows, by
    none (its sequence goes), and may be a row that is not among them (it stays).  Full pages are shared; of a last page that is not full one taker keeps the page,
    the others get pages of their own with its tokens, for which the pages that the call sets free serve too."""
    dev, book = _book(pages)
    parents, n, tensors = parents.reshape(-1), rows.numel(), []
    if beams is not None and (beams <= 0 or n % beams):
        raise RuntimeError("rows must come in groups of `beams`")
    if n > pages.table.shape[0]:
        raise RuntimeError("more rows than the table has")
    for layer in layers:
        size = layer.kfull.shape[1] * PAGE_TOKENS * 256
        for at in _fp16_pages(pages, dev, layer):
            tensors += (at, size)
    _movable(layers, tensors[::2])
    L = _library()
    moves = pages.count.new_empty(L.kvq_pages_reorder_moves(book, n))
    at = moves.data_ptr()
    _launched(L.kvq_pages_reorder(book, _rows(dev, "rows", rows), _ints(dev, "parents", parents, n), n, beams or 0, at, ops.raw_stream()))
    _copy(tensors, at, n, L.kvq_page_copy_tails)


@_on_its_device(0)
def pages_compact(pages, layers):
    """The pages in use move to the lowest numbers of their pools."""
    dev, book = _book(pages)
    total, n, packed, fp16 = pages.refs.numel(), pages.n_packed, [], []
    for layer in layers:
        _layer(pages, dev, layer)
        for tensors, some in ((packed, (layer.kcode, layer.kscale, layer.kmn, layer.vcode, layer.vscale, layer.vmn)), (fp16, (layer.kfull, layer.vfull))):
            for t in some:
                tensors += (t.data_ptr(), t.numel() // max(t.shape[0], 1) * t.element_size())
    _movable(layers, packed[::2] + fp16[::2])
    moves = pages.count.new_empty(8 + 3 * total)
    _launched(_library().kvq_pages_compact(book, moves.data_ptr(), ops.raw_stream()))
    if n:
        _copy(packed, moves.data_ptr(), n)
    if total > n:
        _copy(fp16, moves.data_ptr() + 4 * (4 + 2 * n), total - n)


@_on_its_device(3)
def paged_attention(q, q_start, rows, pages, layer, causal=True, window=None, prefix=None, first=None, softcap=None, alibi_slopes=None,
                    softmax_scale=None, max_new=None, max_tokens=None, max_chunks=None, out=None):
    """Attention of the last tokens of every sequence over its pages.

    q [tokens, nh, 128] fp16: tokens [q_start[i], q_start[i+1]) are the last ones of sequence rows[i], whose keys and values are in the
    pages already; any mix of single tokens and chunks.  A token at position p sees positions j with

        max(first[token], p + 1 - window) <= j < max(p + 1, prefix[i])       (all from the lower bound on where causal is False)

    window: sliding window, None or 0 for none.  prefix int32 [n]: the first prefix[i] tokens see each other.  first int32 [tokens]: where the
    token's document begins, for documents packed behind one another.  softcap: scores become softcap * tanh(score / softcap); 1e30 and
    more, infinity too, is none.
    alibi_slopes fp32 [nh]: slopes[h] * (j - p) is added.  max_new, max_tokens, max_chunks: no sequence has more new tokens, none is longer, no
    more of them have several new tokens (host integers that lay out the work; None: whatever fits the tensors; with many sequences of
    which few have several tokens the third saves time).  Tokens that see nothing get zeros.  Cached values have
    to be finite: one that is not may reach queries that do not see it (include/kvmix_b200.h).
    Returns [tokens, nh, 128] fp16; rows behind q_start[n] are left as they are."""
    return _attend(q, q_start, rows, pages, layer, causal, window, prefix, first, softcap, alibi_slopes, _SCALE if softmax_scale is None else softmax_scale, max_new, max_tokens,
                   max_chunks, out)


def _attend(q, q_start, rows, pages, layer, causal, window, prefix, first, softcap, alibi_slopes, softmax_scale, max_new, max_tokens, max_chunks, out, diff=None):
    """``paged_attention``, or with diff -- addresses of lambdas and of the norm's weight, its eps -- the differential one."""
    dev, book = _book(pages)
    if q.dim() != 3 or q.dtype is not _f16 or q.get_device() != dev or q.shape[2] != 128:
        raise RuntimeError(f"attention over pages takes fp16 queries [tokens, heads, 128] on cuda:{dev}")
    tokens, nh, _ = q.shape
    n = rows.numel()
    block = _layer(pages, dev, layer)
    Hkv = layer.kfull.shape[1]
    if nh % Hkv:
        check(-6)
    if q.stride(2) != 1:
        q = q.contiguous()
    if out is None:
        out = q.new_empty((tokens, nh, 128))
    elif out.shape != q.shape or out.dtype is not _f16 or out.get_device() != dev or out.stride(2) != 1:
        raise RuntimeError("out must be fp16 like q, contiguous along the channels")
    elif not _rows_apart(out):
        raise RuntimeError("rows of out must not lie over one another")
    window, softcap = window or 0, softcap or 0.0
    if window < 0 or not softcap >= 0.0:
        raise RuntimeError("window and softcap must not be negative")
    if not abs(softmax_scale) <= 3.4e38:
        raise RuntimeError("softmax_scale must be a finite number")
    at_slopes = 0
    if alibi_slopes is not None:
        if alibi_slopes.dtype is not torch.float32 or alibi_slopes.shape != (nh,) or alibi_slopes.get_device() != dev or not alibi_slopes.is_contiguous():
            raise RuntimeError(f"alibi_slopes must be float32 [{nh}] on cuda:{dev}")
        at_slopes = alibi_slopes.data_ptr()
    max_new = tokens if max_new is None else min(int(max_new), tokens)
    most = pages.table.shape[1] * PAGE_TOKENS
    max_tokens = most if max_tokens is None else min(int(max_tokens), most)
    max_chunks = n if max_chunks is None else min(int(max_chunks), n)
    if tokens and n and (max_new <= 0 or max_tokens <= 0 or max_chunks < 0):
        raise RuntimeError("max_new and max_tokens must be positive, max_chunks not negative")
    L = _library()
    need = (L.kvq_paged_diff_attn_workspace_bytes if diff else L.kvq_paged_attn_workspace_bytes)(block, n, tokens, nh, max_new, max_tokens, max_chunks)
    ws = pages.count.new_empty((need + 3) // 4) if need else None
    a = (q.data_ptr(), out.data_ptr(), q.stride(0), q.stride(1), out.stride(0), out.stride(1), _ints(dev, "q_start", q_start, n + 1),
         _ints(dev, "rows", rows, n), 0 if first is None else _ints(dev, "first", first, tokens), 0 if prefix is None else _ints(dev, "prefix", prefix, n),
         at_slopes, n, tokens, nh, max_new, max_tokens, max_chunks, int(min(window, _MOST)), 1 if causal else 0,
         softmax_scale, min(softcap, 1e38), 0 if ws is None else ws.data_ptr(), need)
    if diff:
        _launched(L.kvq_paged_diff_attn(book, block, _pack_diff(*a, *diff), ops.raw_stream()))
    else:
        _launched(L.kvq_paged_attn(book, block, _pack_attn(*a), ops.raw_stream()))
    return out


@_on_its_device(4)
def paged_differential_attention(q, lambdas, q_start, rows, pages, layer, causal=True, window=None, prefix=None, first=None, softcap=None, alibi_slopes=None,
                                 softmax_scale=None, norm_weight=None, norm_eps=1e-5, max_new=None, max_tokens=None, max_chunks=None, out=None):
    """The difference of two softmax maps over the pages of every sequence: a head's 128 channels of q and of the cached keys are two halves of 64,

        out = (softmax(q1 k1^T * scale) - lambdas[head] * softmax(q2 k2^T * scale)) v,   then out / sqrt(mean(out^2) + norm_eps) * norm_weight

    lambdas fp32 [nh], finite; norm_weight fp32 [128], or None for no norm (a token that sees nothing gets zeros with one too); softmax_scale
    None: 1 / 8.  Everything else is as ``paged_attention`` has it, for both maps alike.  Both attentions are fp32 until their difference (normed) is rounded; keys, values and weights are rounded on the way as there.  Keys that ``page_append``
    rotates want parts=2."""
    dev, nh = pages.table.get_device(), q.shape[1] if q.dim() == 3 else 0
    if lambdas.dtype is not torch.float32 or lambdas.shape != (nh,) or lambdas.get_device() != dev or not lambdas.is_contiguous():
        raise RuntimeError(f"lambdas must be float32 [{nh}] on cuda:{dev}")
    at_weight = 0
    if norm_weight is not None:
        if norm_weight.dtype is not torch.float32 or norm_weight.shape != (128,) or norm_weight.get_device() != dev or not norm_weight.is_contiguous():
            raise RuntimeError(f"norm_weight must be float32 [128] on cuda:{dev}")
        if not 0.0 <= norm_eps <= 3.4e38:
            raise RuntimeError("norm_eps must not be negative")
        at_weight = norm_weight.data_ptr()
    return _attend(q, q_start, rows, pages, layer, causal, window, prefix, first, softcap, alibi_slopes, 0.125 if softmax_scale is None else softmax_scale, max_new, max_tokens,
                   max_chunks, out, (lambdas.data_ptr(), at_weight, norm_eps if at_weight else 0.0))


class PagedStep(NamedTuple):
    """The new tokens of a forward pass: tokens [q_start[i], q_start[i+1]) belong to row rows[i]."""
    rows: torch.Tensor
    q_start: torch.Tensor
    tokens: int
    max_new: int
    max_tokens: int
    max_chunks: int
    positions: int = 0                # the new tokens' are all below it


class KVmixPagedCache:
    """Pages, bookkeeping and the calls on them for a stack of layers.

    layers: [(k_bits, v_bits)] or upstream's ``quant_bits`` dict (myprofileKV.py:99-104; its ratios do not apply: the fp16 window is
    ``residual_length`` tokens and what is left of the page they begin in).  A forward pass:

        step = cache.extend(rows, counts)              # counts[i] more tokens for the sequence in row rows[i]
        for l in range(n_layers):
            cache.write(l, k, v, step)                 # [tokens, Hkv, 128] fp16 each, keys rotated
            out = cache.attend(l, q, step)             # [tokens, nh, 128]; options as paged_attention
        cache.settle(rows)                             # full pages behind the window are quantized

    ``append`` is ``write`` of keys as the projections give them, and rotates the queries too; ``attend_differential`` is the difference of two
    attentions; ``advance`` ends a step of beam search (``beam_select``, then ``reorder``).
    ``lengths`` mirrors the lengths on the host (it lays out the work); ``check()`` raises if a call had to be refused."""

    def __init__(self, layers, kv_heads, head_dim, max_seqs, max_tokens, packed_pages, fp16_pages, group_size, residual_length=128, device="cuda"):
        if head_dim != 128:
            raise RuntimeError("the paged cache holds heads of 128 channels")
        if isinstance(layers, dict):
            layers = [(layers[i]["k_bits"], layers[i]["v_bits"]) for i in sorted(layers)]
        if not layers or any(b not in (1, 2, 3, 4) for pair in layers for b in pair):
            raise RuntimeError("layers are (k_bits, v_bits) pairs of 1, 2, 3 or 4")
        if group_size not in (32, 64, 128):
            raise RuntimeError("pages are quantized in groups of 32, 64 or 128")
        if residual_length < 0 or kv_heads <= 0 or max_seqs <= 0 or max_tokens <= 0 or packed_pages < 0 or fp16_pages <= 0:
            raise RuntimeError("sizes must be positive")
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.window, self.device = int(min(residual_length, _MOST)), dev

        def packed(bits):
            w, g = page_words(bits), page_groups(bits, group_size)
            return [torch.empty(packed_pages, kv_heads, PAGE_TOKENS, w, dtype=torch.int32, device=dev)] + \
                [torch.empty(packed_pages, kv_heads, PAGE_TOKENS, g, dtype=torch.float16, device=dev) for _ in range(2)]

        def fp16():
            return torch.empty(fp16_pages, kv_heads, PAGE_TOKENS, 128, dtype=torch.float16, device=dev)

        self.layers = [PageLayer(*packed(kb), fp16(), *packed(vb), fp16(), kb, vb, group_size) for kb, vb in layers]
        i32 = dict(dtype=torch.int32, device=dev)
        self.book = PageBook(torch.empty(max_seqs, -(-max_tokens // PAGE_TOKENS), **i32), torch.empty(max_seqs, **i32), torch.empty(max_seqs, **i32),
                             torch.empty(packed_pages + fp16_pages, **i32), torch.empty(packed_pages + fp16_pages, **i32), torch.empty(4, **i32), packed_pages)
        self.reset()

    def reset(self):
        """No sequence, every page free."""
        b, n16 = self.book, self.book.refs.numel() - self.book.n_packed
        b.table.fill_(-1)
        for t in (b.length, b.packed, b.refs):
            t.zero_()
        b.free_ids.copy_(torch.cat([torch.arange(b.n_packed - 1, -1, -1, dtype=torch.int32), torch.arange(n16 - 1, -1, -1, dtype=torch.int32)]))
        b.count.copy_(torch.tensor([b.n_packed, n16, 0, 0], dtype=torch.int32))
        self.lengths = [0] * b.length.numel()

    def _row_tensor(self, rows, distinct=True):
        rows = [int(r) for r in rows]
        if any(not 0 <= r < len(self.lengths) for r in rows) or (distinct and len(set(rows)) != len(rows)):
            raise RuntimeError("rows must lie in the table, each named once")
        return rows, torch.tensor(rows, dtype=torch.int32).to(self.device, non_blocking=True)

    def extend(self, rows, counts):
        """counts[i] more tokens for the sequence in row rows[i]; returns the step to hand to ``write`` and ``attend``."""
        rows, at = self._row_tensor(rows)
        counts = [int(c) for c in counts]
        if len(counts) != len(rows) or any(c < 0 for c in counts):
            raise RuntimeError("one count of new tokens for every row")
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        both = torch.tensor(counts + starts, dtype=torch.int32).to(self.device, non_blocking=True)
        n = len(rows)
        pages_extend(at, both[:n], self.book)
        for r, c in zip(rows, counts):
            self.lengths[r] += c
        return PagedStep(at, both[n:], starts[-1], max(counts, default=0), max((self.lengths[r] for r in rows), default=0),
                         sum(c > 1 for c in counts), max((self.lengths[r] for r, c in zip(rows, counts) if c), default=0))

    def write(self, layer, k, v, step):
        if k.shape[0] != step.tokens or v.shape[0] != step.tokens:
            raise RuntimeError("keys and values for every new token of the step")
        page_write(k, v, step.q_start, step.rows, self.book, self.layers[layer])

    def attend(self, layer, q, step, **options):
        """Options as ``paged_attention``: causal, window, prefix, first, softcap, alibi_slopes, softmax_scale, out."""
        if q.shape[0] != step.tokens:
            raise RuntimeError("one query for every new token of the step")
        return paged_attention(q, step.q_start, step.rows, self.book, self.layers[layer], max_new=max(step.max_new, 1), max_tokens=max(step.max_tokens, 1),
                               max_chunks=step.max_chunks, **options)

    def attend_differential(self, layer, q, lambdas, step, **options):
        """Options as ``paged_differential_attention``: norm_weight, norm_eps and those of ``attend``."""
        if q.shape[0] != step.tokens:
            raise RuntimeError("one query for every new token of the step")
        return paged_differential_attention(q, lambdas, step.q_start, step.rows, self.book, self.layers[layer], max_new=max(step.max_new, 1),
                                            max_tokens=max(step.max_tokens, 1), max_chunks=step.max_chunks, **options)

    def append(self, layer, k, v, cos, sin, step, q=None, **options):
        """``write`` of keys that are not rotated yet, and the step's queries rotated: returns them.  Options as ``page_append``: q_out, positions, interleaved,
        parts."""
        if k.shape[0] != step.tokens or v.shape[0] != step.tokens or (q is not None and q.shape[0] != step.tokens):
            raise RuntimeError("keys, values and queries for every new token of the step")
        if options.get("positions") is None and cos.shape[0] < step.positions:
            raise RuntimeError(f"angles for {cos.shape[0]} positions, the step has new tokens up to {step.positions}")
        return page_append(k, v, cos, sin, step.q_start, step.rows, self.book, self.layers[layer], q=q, **options)

    def settle(self, rows=None):
        rows = range(len(self.lengths)) if rows is None else rows
        pages_settle(self._row_tensor(rows)[1], self.window, self.book, self.layers)

    def fork(self, parents, children):
        parents, at = self._row_tensor(parents, distinct=False)
        children, to = self._row_tensor(children)
        if len(parents) != len(children) or set(parents) & set(children) or any(self.lengths[c] for c in children):
            raise RuntimeError("one empty child for every parent")
        pages_fork(at, to, self.book, self.layers)
        for p, c in zip(parents, children):
            self.lengths[c] = self.lengths[p]

    def reorder(self, rows, parents, beams=None):
        """Row rows[i] becomes what row parents[i] was (``pages_reorder``).  With ``beams``, parents are the beams within each group of that many rows: a list or,
        as ``beam_select`` returns them, int32 on the device; the rows of a group then have one length."""
        rows, at = self._row_tensor(rows)
        if beams is not None and (beams <= 0 or len(rows) % beams):
            raise RuntimeError("rows must come in groups of `beams`")
        if isinstance(parents, torch.Tensor):
            if beams is None or parents.numel() != len(rows):
                raise RuntimeError("parents on the device are beams within groups of rows, one a row")
            if any(self.lengths[r] != self.lengths[rows[i // beams * beams]] for i, r in enumerate(rows)):
                raise RuntimeError("the rows of a group must have one length where parents are on the device")
            pages_reorder(at, parents, self.book, self.layers, beams)
            return
        parents = [int(p) for p in parents]
        if len(parents) != len(rows) or any(not 0 <= p < (len(self.lengths) if beams is None else beams) for p in parents):
            raise RuntimeError("one parent for every row")
        if beams is not None:
            parents = [rows[i // beams * beams + p] for i, p in enumerate(parents)]
        pages_reorder(at, self._row_tensor(parents, distinct=False)[1], self.book, self.layers)
        lengths = [self.lengths[p] for p in parents]
        for r, n in zip(rows, lengths):
            self.lengths[r] = n

    def advance(self, rows, logits, scores, beams, **options):
        """The end of a step of beam search: the best continuations of every group of ``beams`` rows (``beam_select``, whose options these are), which the rows
        then hold (``reorder``).  Returns the ``BeamStep``: its next_tokens are the next step's."""
        chosen = beam_select(logits, scores, beams, **options)
        self.reorder(rows, chosen.next_beams, beams)
        return chosen

    def free(self, rows):
        rows, at = self._row_tensor(rows)
        pages_free(at, self.book)
        for r in rows:
            self.lengths[r] = 0

    def compact(self):
        pages_compact(self.book, self.layers)

    def free_pages(self):
        """(packed, fp16) pages nobody holds.  Waits for the device."""
        return tuple(self.book.count[:2].tolist())

    def check(self):
        """Raises if a call since the last check had to be refused, left tokens out or lost its output, and lets the cache go on from where it
        was.  Waits for the device."""
        status = int(self.book.count[2])
        if status:
            self.book.count[2] = 0
            self.lengths = self.book.length.tolist()
            raise RuntimeError("paged cache: " + "; ".join(text for bit, text in _STATUS.items() if status & bit))

    def sequence(self, layer, row):
        """A sequence in upstream's layout: (kcode [Hkv,128,words], kscale, kmn, kfull [Hkv,tail,128], vcode [Hkv,packed,words], vscale, vmn,
        vfull, length), packed parts page behind page, None where there are none.  Waits for the device."""
        l, b = self.layers[layer], self.book
        n, a = int(b.length[row]), int(b.packed[row])
        ids = b.table[row, :-(-n // PAGE_TOKENS)].long()
        keys = [t[ids[:a]].permute(1, 2, 0, 3).flatten(2) if a else None for t in (l.kcode, l.kscale, l.kmn)]
        values = [t[ids[:a]].permute(1, 0, 2, 3).flatten(1, 2) if a else None for t in (l.vcode, l.vscale, l.vmn)]
        tails = [t[ids[a:]].permute(1, 0, 2, 3).flatten(1, 2)[:, :n - a * PAGE_TOKENS] for t in (l.kfull, l.vfull)]
        return (*keys, tails[0], *values, tails[1], n)
