"""The paged cache's host side without a GPU: argument blocks, refusals before any launch, workspace sizes."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

import kvmix_b200 as kv
from kvmix_b200 import _lib, paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_argument_blocks_match_the_header():
    names = ["kvq_page_book", "kvq_page_layer", "kvq_page_tensor", "kvq_page_write_args", "kvq_paged_attn_args"]
    src = '#include <stdio.h>\n#include "kvmix_b200.h"\nint main(void){ printf("%s", %s); return 0; }\n' % (
        " ".join(["%zu"] * len(names)), ", ".join("sizeof(%s)" % n for n in names))
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "s.c"), "w").write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), os.path.join(d, "s.c"), "-o", os.path.join(d, "s")])
        sizes = [int(x) for x in subprocess.check_output([os.path.join(d, "s")]).split()]
    assert sizes == [ctypes.sizeof(c) for c in (_lib.PageBookArgs, _lib.PageLayerArgs, _lib.PageTensor, _lib.PageWriteArgs, _lib.PagedAttnArgs)]
    paged._library()                                 # holds the packed forms to the same sizes


def book(**over):
    b = _lib.PageBookArgs(*[64] * 6, 4, 8, 10, 10)
    for k, v in over.items():
        setattr(b, k, v)
    return bytes(b)


def layer(**over):
    a = _lib.PageLayerArgs(*[64] * 8, 2, 4, 2, 64, 10, 10)
    for k, v in over.items():
        setattr(a, k, v)
    return bytes(a)


def attn(**over):
    a = _lib.PagedAttnArgs()
    a.q = a.out = a.q_start = a.rows = 64
    a.n, a.tokens, a.nh, a.max_new, a.max_tokens, a.max_chunks, a.softmax_scale = 1, 1, 4, 1, 100, 1, 0.1
    for k, v in over.items():
        setattr(a, k, v)
    return bytes(a)


def test_refusals_need_no_gpu():
    L = paged._library()
    for bad, rc in ((book(table=None), -10), (book(count=None), -10), (book(slots=0), -7), (book(max_pages=0), -7), (book(n_packed=-1), -7),
                    (book(slots=2 ** 20 + 1), -11), (book(n_packed=2 ** 30, n_fp16=1), -7)):
        assert L.kvq_pages_extend(bad, 64, 64, 1, None) == rc
        assert L.kvq_pages_free(bad, 64, 1, None) == rc
        assert L.kvq_pages_compact(bad, 64, None) == rc
        assert L.kvq_paged_attn(bad, layer(), attn(), None) == rc
    assert L.kvq_pages_extend(book(), None, 64, 1, None) == -10
    assert L.kvq_pages_extend(book(), 64, 64, -1, None) == -7
    assert L.kvq_pages_extend(book(), None, None, 0, None) == 0
    assert L.kvq_pages_settle(book(), 64, 1, -1, 64, None) == -7
    assert L.kvq_pages_settle(book(), 64, 1, 0, None, None) == -10
    assert L.kvq_pages_fork(book(), 64, None, 1, 64, None) == -10
    for bad, rc in ((layer(k_bits=5), -1), (layer(v_bits=0), -1), (layer(group=16), -11), (layer(kcode=None), -10), (layer(kfull=None), -10),
                    (layer(kscale=66), -13), (layer(Hkv=0), -7)):
        assert L.kvq_page_pack(bad, 64, 1, None) == rc
        assert L.kvq_page_write(book(), bad, bytes(_lib.PageWriteArgs()), None) == rc
        assert L.kvq_paged_attn(book(), bad, attn(), None) == rc
    for bad, rc in ((attn(nh=3), -6), (attn(q=None), -10), (attn(n=-1), -7), (attn(max_new=0), -7), (attn(max_chunks=-1), -7), (attn(window=-1), -7), (attn(softcap=-1.0), -7),
                    (attn(softcap=float("nan")), -7), (attn(softmax_scale=float("nan")), -7), (attn(tokens=0), 0), (attn(max_tokens=100000), -12)):
        assert L.kvq_paged_attn(book(), layer(), bad, None) == rc
    one = _lib.PageTensor(64, 24)
    assert L.kvq_page_copy(bytes(one), 1, 64, 1, None) == -13
    assert L.kvq_page_copy(None, 257, 64, 1, None) == -7


def test_workspace_holds_every_split():
    L = paged._library()
    for n in (1, 3, 64):
        for tokens in (1, 7, 300, 4096):
            for nh, Hkv in ((1, 1), (32, 8), (64, 8), (40, 8)):
                for length in (1, 128, 5000, 131072):
                    b = L.kvq_paged_attn_workspace_bytes(layer(Hkv=Hkv), n, tokens, nh, tokens, length, n)
                    assert b % (tokens * nh * 520) == 0
                    splits = b // (tokens * nh * 520)
                    assert splits != 1 and splits <= -(-length // 128)
    assert L.kvq_paged_attn_workspace_bytes(layer(), 1, 1, 3, 1, 100, 1) == 0


def test_no_cpu_path():
    cache = kv.KVmixPagedCache([(4, 2)], 1, 128, 2, 256, 1, 2, 64, device="cpu")
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 128).half()
    for call in (lambda: kv.pages_extend(i, i, cache.book), lambda: kv.pages_free(i, cache.book), lambda: kv.pages_settle(i, 0, cache.book, cache.layers),
                 lambda: kv.pages_fork(i, i, cache.book, cache.layers), lambda: kv.pages_compact(cache.book, cache.layers),
                 lambda: kv.page_write(x, x, i, i, cache.book, cache.layers[0]), lambda: kv.paged_attention(x, i, i, cache.book, cache.layers[0])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_layers_of_a_profile():
    from kvmix_b200.configs import config3
    qb = config3().quant_bits
    cache = kv.KVmixPagedCache(qb, 1, 128, 1, 128, 1, 1, 64, device="cpu")
    assert [(l.k_bits, l.v_bits) for l in cache.layers] == [(qb[i]["k_bits"], qb[i]["v_bits"]) for i in sorted(qb)]
    assert cache.layers[0].kcode.shape[-1] == paged.page_words(cache.layers[0].k_bits)


def test_scales_and_caps_that_are_no_numbers():
    L = paged._library()
    for bad in (dict(softmax_scale=float("inf")), dict(softmax_scale=-float("inf")), dict(softcap=-float("inf"))):
        assert L.kvq_paged_attn(book(), layer(), attn(**bad), None) == -7


def test_workspace_of_a_long_chunk_beside_single_tokens():
    """Partial sums of single tokens over a long context do not take a place for every row of the chunk beside them in each of their splits."""
    L = paged._library()
    for bits in ((2, 2), (3, 2), (4, 4)):
        for n, tokens, max_new in ((2, 1025, 1024), (2, 8193, 8192), (2, 32769, 32768), (5, 65540, 65536), (30, 20030, 20001)):
            for chunks in (1, n):
                b = L.kvq_paged_attn_workspace_bytes(layer(Hkv=8, k_bits=bits[0], v_bits=bits[1]), n, tokens, 32, max_new, 131072, chunks)
                assert b <= 2 * tokens * 32 * 520, (n, tokens, b)
    # without a chunk the splits are as many as they pay
    assert L.kvq_paged_attn_workspace_bytes(layer(Hkv=8), 1, 1, 32, 1, 131072, 1) >= 20 * 32 * 520


def test_launch_counts_of_threads_that_cross():
    """A thread that read the library's count before another one did, and comes to add it behind that one, adds nothing; the count may wrap."""
    count, seen = paged._launch_count()
    kept = count.value, seen[0], kv.ops.LAUNCHES[0]
    try:
        for now, had, added in ((5, 3, 2), (5, 6, 0), (1, 2 ** 32 - 2, 3), (2 ** 32 - 1, 2, 0)):
            count.value, seen[0], before = now, had, kv.ops.LAUNCHES[0]
            paged._launched(0)
            assert kv.ops.LAUNCHES[0] - before == added
            paged._launched(0)
            assert kv.ops.LAUNCHES[0] - before == added
    finally:
        count.value, seen[0], kv.ops.LAUNCHES[0] = kept
