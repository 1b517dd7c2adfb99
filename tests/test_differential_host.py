"""Differential attention over pages without a GPU: what a call asks for beside its tensors."""
import inspect

import pytest
import torch

import kvmix_b200 as kv
from kvmix_b200 import paged
from test_paged_host import layer

MB = 1 << 20


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (32, 32), (64, 8), (8, 4), (160, 32)])
@pytest.mark.parametrize("n", [1, 2, 8])
def test_sums_of_cut_tiles_take_no_gigabytes(heads, kv_heads, n):
    """Long chunks over longer contexts, of which only the tiles of a last round of CTAs are cut: half a gigabyte at most, and none where that does not do."""
    L = paged._library()
    for new in (2048, 2400, 3333, 4816, 8192, 11904, 23667):
        each = new // n
        if each * n * heads < 37888:                             # fewer CTAs than SMs: all tiles may be cut
            continue
        for context in (4 * new, 34816, 65536, 131072):
            assert L.kvq_paged_diff_attn_workspace_bytes(layer(Hkv=kv_heads), n, n * each, heads, each, context, n) <= 512 * MB, (new, context)


def test_a_cut_is_still_made():
    L = paged._library()
    assert L.kvq_paged_diff_attn_workspace_bytes(layer(Hkv=8), 1, 2048, 32, 2048, 34816, 1) == 2 * 2048 * 64 * 520
    assert 0 < L.kvq_paged_diff_attn_workspace_bytes(layer(Hkv=8), 1, 2400, 32, 2400, 34816, 1) <= 160 * MB


def test_plain_attention_takes_no_more_than_it_says():
    """Addresses of the differential form are not to be had through the plain one."""
    names = inspect.signature(kv.paged_attention).parameters
    assert not [n for n in names if n.startswith("_")]
    i = torch.zeros(1, dtype=torch.int32)
    cache = kv.KVmixPagedCache([(4, 2)], 1, 128, 2, 256, 1, 2, 64, device="cpu")
    with pytest.raises(TypeError):
        kv.paged_attention(torch.zeros(1, 1, 128).half(), i, i, cache.book, cache.layers[0], True, None, None, None, None, None, None, None, None, None, None, (1, 2, 3.0))
    with pytest.raises(TypeError):
        kv.paged_attention(torch.zeros(1, 1, 128).half(), i, i, cache.book, cache.layers[0], _diff=(1, 2, 3.0))
