"""Appending, reordering and beam selection without a GPU: argument blocks, refusals before any launch, sizes of workspaces."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

import kvmix_b200 as kv
from kvmix_b200 import _lib, paged
from test_paged_host import book, layer

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_argument_blocks_match_the_header():
    names = ["kvq_page_append_args", "kvq_beam_args", "kvq_paged_diff_args"]
    src = '#include <stdio.h>\n#include "kvmix_b200.h"\nint main(void){ printf("%s %%d %%d", %s, KVQ_MOST_BEAMS, KVQ_MOST_BEST); return 0; }\n' % (
        " ".join(["%zu"] * len(names)), ", ".join("sizeof(%s)" % n for n in names))
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "s.c"), "w").write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), os.path.join(d, "s.c"), "-o", os.path.join(d, "s")])
        sizes = [int(x) for x in subprocess.check_output([os.path.join(d, "s")]).split()]
    assert sizes == [ctypes.sizeof(_lib.PageAppendArgs), ctypes.sizeof(_lib.BeamArgs), ctypes.sizeof(_lib.PagedDiffArgs), _lib.MOST_BEAMS, _lib.MOST_BEST]
    paged._library()


def append(**over):
    a = _lib.PageAppendArgs()
    a.k = a.v = a.q = a.q_out = a.cos = a.sin = a.q_start = a.rows = 64
    a.n, a.tokens, a.nh, a.angles, a.angle_rows, a.parts = 1, 1, 4, 64, 100, 1
    for k, v in over.items():
        setattr(a, k, v)
    return bytes(a)


def select(**over):
    a = _lib.BeamArgs()
    a.logits = a.scores = a.out_scores = a.out_beams = a.out_tokens = a.next_scores = a.next_beams = a.next_tokens = 64
    a.requests, a.beams, a.vocabulary, a.n, a.l_sR, a.workspace, a.workspace_bytes = 2, 4, 1000, 8, 1000, 64, 1 << 20
    for k, v in over.items():
        setattr(a, k, v)
    return bytes(a)


def test_refused_appends():
    L = paged._library()
    for bad, rc in ((append(angles=12), -11), (append(angles=72), -11), (append(angles=0), -7), (append(angles=40, parts=2), -11), (append(parts=3), -11), (append(parts=0), -11),
                    (append(type=3), -11), (append(type=-1), -11), (append(n=-1), -7), (append(tokens=-1), -7), (append(nh=-1), -7), (append(angle_rows=-1), -7), (append(k=None), -10),
                    (append(cos=None), -10), (append(q=None), -10), (append(q_out=None), -10), (append(rows=None), -10), (append(cos=66), -13), (append(tokens=0), 0), (append(n=0), 0)):
        assert L.kvq_page_append(book(), layer(), bad, None) == rc
    assert L.kvq_page_append(book(table=None), layer(), append(), None) == -10
    assert L.kvq_page_append(book(), layer(Hkv=0), append(), None) == -7
    assert L.kvq_page_append(book(), layer(), None, None) == -10


def test_refused_reorderings():
    L = paged._library()
    for args, rc in (((book(table=None), 64, 64, 1, 0, 64), -10), ((book(), None, 64, 1, 0, 64), -10), ((book(), 64, None, 1, 0, 64), -10), ((book(), 64, 64, 1, 0, None), -10),
                     ((book(), 64, 64, -1, 0, 64), -7), ((book(), 64, 64, 5, 0, 64), -7), ((book(), 64, 64, 3, 2, 64), -7), ((book(), 64, 64, 3, -1, 64), -7)):
        assert L.kvq_pages_reorder(*args, None) == rc
    assert L.kvq_pages_reorder_moves(book(), 3) == 4 + 3 * (5 + 8) + 4
    assert L.kvq_pages_reorder_moves(book(slots=0), 3) == 0 and L.kvq_pages_reorder_moves(book(), -1) == 0
    for tensor, n, rc in ((_lib.PageTensor(64, 32768 + 16), 1, -7), (_lib.PageTensor(66, 32768), 1, -13), (_lib.PageTensor(64, 1 << 31), 1, -7), (_lib.PageTensor(64, 32768), 257, -7),
                          (_lib.PageTensor(64, 32768), -1, -7), (_lib.PageTensor(None, 32768), 1, 0)):
        assert L.kvq_page_copy_tails(bytes(tensor), n, 64, 1, None) == rc


def test_refused_selections():
    L = paged._library()
    for bad, rc in ((select(requests=-1), -7), (select(beams=0), -7), (select(beams=65), -11), (select(vocabulary=0), -7), (select(n=0), -7), (select(n=129), -11), (select(n=3), -7),
                    (select(n_ends=2, ends=64), -7), (select(n_ends=-1), -7), (select(type=3), -11), (select(logits=None), -10), (select(scores=None), -10), (select(next_tokens=None), -10),
                    (select(n_ends=1), -10), (select(workspace=None), -12), (select(workspace_bytes=100), -12), (select(workspace=72), -13), (select(logits=65), -13),
                    (select(logits=66, type=2), -13), (select(vocabulary=1, n=8), -7), (select(requests=0), 0)):
        assert L.kvq_beam_select(bad, None) == rc
    assert L.kvq_beam_select_workspace_bytes(select(beams=0)) == 0 and L.kvq_beam_select(None, None) == -10


def test_workspace_of_a_selection():
    L = paged._library()
    for requests in (1, 3, 64, 5000):
        for beams in (1, 4, 64):
            for V in (1, 100, 32000, 1 << 20):
                for n in (beams, 2 * beams, 128):
                    if n > min(128, beams * V):
                        continue
                    b = L.kvq_beam_select_workspace_bytes(select(requests=requests, beams=beams, vocabulary=V, n=n))
                    rows = requests * beams
                    assert b and b % (rows * (8 * n + 16)) == 0
                    parts = b // (rows * (8 * n + 16))
                    assert 1 <= parts <= 32 and parts * n <= max(1024, n) and (parts == 1 or parts <= -(-V // 4096))


def test_no_cpu_path():
    cache = kv.KVmixPagedCache([(4, 2)], 1, 128, 2, 256, 1, 2, 64, device="cpu")
    i, x, t = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, 128).half(), torch.zeros(4, 64)
    for call in (lambda: kv.page_append(x, x, t, t, i, i, cache.book, cache.layers[0]), lambda: kv.pages_reorder(i, i, cache.book, cache.layers),
                 lambda: kv.beam_select(t, torch.zeros(4), 2), lambda: kv.paged_differential_attention(x, t[0, :1], i, i, cache.book, cache.layers[0])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def diff(over=None, **own):
    a = _lib.PagedDiffArgs()
    a.a.q = a.a.out = a.a.q_start = a.a.rows = a.lambdas = 64
    a.a.n, a.a.tokens, a.a.nh, a.a.max_new, a.a.max_tokens, a.a.max_chunks, a.a.softmax_scale, a.norm_eps = 1, 1, 4, 1, 100, 1, 0.1, 1e-5
    for k, v in (over or {}).items():
        setattr(a.a, k, v)
    for k, v in own.items():
        setattr(a, k, v)
    return bytes(a)


def test_refused_differential_attention():
    L = paged._library()
    for bad, rc in ((diff(dict(nh=3)), -6), (diff(dict(nh=2 ** 30 + 2 ** 29)), -11), (diff(dict(q=None)), -10), (diff(dict(n=-1)), -7), (diff(dict(max_new=0)), -7), (diff(dict(tokens=0)), 0),
                    (diff(dict(max_tokens=100000)), -12), (diff(lambdas=None), -10), (diff(norm_weight=64, norm_eps=-1.0), -7), (diff(norm_weight=64, norm_eps=float("nan")), -7),
                    (diff(norm_weight=64, norm_eps=float("inf")), -7), (diff(dict(softcap=-1.0)), -7), (None, -10)):
        assert L.kvq_paged_diff_attn(book(), layer(), bad, None) == rc
    assert L.kvq_paged_diff_attn(book(count=None), layer(), diff(), None) == -10
    assert L.kvq_paged_diff_attn(book(), layer(group=16), diff(), None) == -11
    for n in (1, 3, 64):
        for tokens in (1, 7, 300, 4096):
            for nh, Hkv in ((1, 1), (32, 8), (64, 8), (40, 8)):
                for length in (1, 128, 5000, 131072):
                    b = L.kvq_paged_diff_attn_workspace_bytes(layer(Hkv=Hkv), n, tokens, nh, tokens, length, n)
                    assert b % (2 * tokens * nh * 520) == 0 and b // (2 * tokens * nh * 520) != 1
    assert L.kvq_paged_diff_attn_workspace_bytes(layer(), 1, 1, 3, 1, 100, 1) == 0
