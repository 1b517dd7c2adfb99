"""The second look of beam search's selection at a part of a row, without a GPU: what the kernel's own rule (csrc/beam_reach.cuh) takes, pass by pass, where
more elements reach the threshold than there is room for."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
THREADS, ROOM = 256, 2048            # of a CTA; for what reaches its threshold


@pytest.fixture(scope="session")
def takes(tmp_path_factory):
    d = tmp_path_factory.mktemp("reach")
    (d / "r.cc").write_text('''
#include "beam_reach.cuh"
extern "C" void takes(const unsigned long long *piece, const unsigned long long *token, long n, unsigned long long first, int raised, unsigned long long to, unsigned char *out) {
    kvq::Reach r(first);
    if (raised) r.raise(to);
    for (long i = 0; i < n; ++i) out[i] = r.takes(piece[i], token[i]);
}
''')
    subprocess.check_call(["g++", "-O2", "-shared", "-fPIC", "-I", os.path.join(ROOT, "kvmix_b200", "csrc"), str(d / "r.cc"), "-o", str(d / "r.so")])
    f = ctypes.CDLL(str(d / "r.so")).takes
    pointer = np.ctypeslib.ndpointer(flags="C")
    f.argtypes = [pointer, pointer, ctypes.c_long, ctypes.c_uint64, ctypes.c_int, ctypes.c_uint64, pointer]

    def call(piece, token, first, raised):
        out = np.empty(len(piece), dtype=np.uint8)
        f(piece, token, len(piece), int(first), raised is not None, int(raised or 0), out)
        return out.astype(bool)
    return call


def key(x, number):
    u = (np.asarray(x, dtype=np.float32) + np.float32(0)).view(np.uint32)
    u = np.where(u >> 31, ~u, u | np.uint32(1 << 31)).astype(np.uint64)
    return u << np.uint64(32) | (np.uint64(0xffffffff) - np.asarray(number, dtype=np.uint64))


def first_threshold(x, n, of):
    """(threshold, threads that reach it) of a part that is the whole row: the n-th best of the groups of threads, by each thread's first largest piece."""
    pieces = np.arange(len(x) // of)
    keys = key(x.reshape(-1, of).max(1), pieces)
    mine = np.array([keys[t::THREADS].max() for t in range(THREADS)], dtype=np.uint64)
    if n <= 32:
        first = np.sort(mine.reshape(-1, 8 if n <= 16 else 4).max(1))[-n]
    else:
        first = min(np.sort(w)[-((n + 7) // 8)] for w in mine.reshape(8, 32))
    return first, np.nonzero(mine >= first)[0]


def walk(x, n, of, takes, rng, most=1000):
    """(n best tokens, passes)."""
    first, threads = first_threshold(x, n, of)
    tokens = np.concatenate([(np.arange(t, len(x) // of, THREADS)[:, None] * of + np.arange(of)).ravel() for t in threads])
    by_piece, by_token = key(x[tokens], tokens // of), key(x[tokens], tokens)
    raised = None
    for passes in range(1, most):
        order = np.nonzero(takes(by_piece, by_token, first, raised))[0]
        if rng is not None:                                      # those that come first find room: by tokens, or as it happens
            order = order[np.array(rng.sample(range(len(order)), len(order)))]
        kept = np.sort(by_token[order[:ROOM]])[::-1][:n]
        if len(order) <= ROOM:
            return [0xffffffff - (int(k) & 0xffffffff) for k in kept], passes
        raised = kept[-1]
    return None, most


def coinciding(n, of, V):
    """A row of -10 and 0 whose first threshold is (0, piece P) and whose n-th best token is P: eight threads have nothing but 0 from there on, one more has its
    first at piece P, and each further group (or lane) that makes P the n-th has one in between."""
    P = (2048 * 7 + 40) if of == 8 else 1024 * 14 + 24
    x = np.full(V, -10.0, dtype=np.float32)
    dense = np.nonzero(np.arange(V) // of % THREADS < 8)[0]
    x[dense[np.searchsorted(dense, P) - (n - 1):]] = 0
    x[P * of] = 0
    turn = THREADS * 40                                          # between P / of and P
    if n <= 32:
        width = 8 if n <= 16 else 4
        groups = [g for g in range(THREADS // width) if g >= 8 // width and g != P % THREADS // width]
        for g in groups[:n - 1 - 8 // width]:
            x[(turn + g * width) * of] = 0
    else:
        for w in range(8):
            lanes = [l for l in range(32) if w or l >= 8]
            if w == P % THREADS // 32:
                lanes.remove(P % 32)
            want = (n + 7) // 8 - (8 if w == 0 else 0) - (w == P % THREADS // 32)
            for l in lanes[:max(want, 0)]:
                x[(turn + 32 * w + l) * of] = 0
    return x, P


COINCIDING = [(n, 8) for n in (2, 3, 8, 15, 16, 17, 31, 32, 33, 48, 100, 128)] + [(n, 4) for n in (2, 5, 16, 24, 32)]


@pytest.mark.parametrize("n,of", COINCIDING)
def test_a_token_with_the_number_of_the_thresholds_piece(takes, n, of):
    x, P = coinciding(n, of, 131072)
    first, threads = first_threshold(x, n, of)
    assert first == key(0, P)                                    # what the row was made for
    want = np.nonzero(x == 0)[0][:n].tolist()
    assert want[-1] == P
    for rng in (None, random.Random(n)):
        got, passes = walk(x, n, of, takes, rng)
        assert got == want and passes <= 8


@pytest.mark.parametrize("seed", range(30))
def test_rows_of_few_values(takes, seed):
    rng = np.random.default_rng(seed)
    of, n, V = int(rng.choice([4, 8])), int(rng.choice([1, 2, 9, 16, 17, 32, 33, 64, 128])), int(rng.integers(20, 120)) * 2048
    thread = np.arange(V) // of % THREADS
    x = np.where(thread < rng.integers(1, 40), rng.integers(0, int(rng.integers(1, 4)), V), -10 + rng.integers(0, 2, V)).astype(np.float32)
    x[:int(rng.integers(0, V // 2))] = -20
    x[rng.integers(0, V, 40)] = 0
    got, passes = walk(x, n, of, takes, random.Random(seed))
    assert got == np.argsort(-x, kind="stable")[:n].tolist()
    assert passes <= 1 + V // (ROOM - n)
