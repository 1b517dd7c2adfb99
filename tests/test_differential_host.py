"""Differential attention over pages without a GPU: what a call asks for beside its tensors."""
import pytest

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
