"""The sequence operators at the limits of their arguments, as far as the host decides them: everything here runs without a GPU."""
import ctypes as C
import os

import pytest
import torch


@pytest.fixture(scope="module")
def native():
    import __graft_entry__ as ge
    from nl_vsgg_amd import _native
    if not os.path.exists(_native.LIB_PATH):
        ge.build()
    return _native


def _step(nat, n, heads, capacity, d=1):
    """a cache that all sequences share (sequence stride 0)"""
    return nat.SttranAttentionStep(struct_size=C.sizeof(nat.SttranAttentionStep), dtype=nat.DTYPE_BF16, num_seq=n, num_q_heads=heads, num_kv_heads=heads, head_dim=d,
                                   capacity=capacity, q=4096, k=4096, v=4096, q_seq_stride=heads * d, q_head_stride=d, k_row_stride=heads * d, k_head_stride=d,
                                   v_row_stride=heads * d, v_head_stride=d, lengths=4096, scale=1.0, out=4096)


@pytest.mark.parametrize("n,heads,capacity", [(16384, 1, 1 << 30), (24576, 1, 1 << 30), (65535, 1, 1 << 30), (65535, 64, 1 << 21), (65535, 4096, 1 << 30), (4096, 1, 1000)])
def test_step_of_many_sequences_over_one_cache_takes_it_whole(native, n, heads, capacity):
    """rows a workgroup are counted in 64 bits until they are known to be the cache's at most: one share, nothing to join"""
    assert native.load().sttran_attention_step_workspace_bytes(C.byref(_step(native, n, heads, capacity))) == 0


@pytest.mark.parametrize("n,heads,capacity", [(1, 1, 1 << 30), (1, 1, 193), (4095, 1, 1 << 20), (3, 2, 5000)])
def test_step_shares_cover_the_cache(native, n, heads, capacity):
    need = native.load().sttran_attention_step_workspace_bytes(C.byref(_step(native, n, heads, capacity)))
    shares, rest = divmod(need, heads * n * (1 + 2) * 4)
    assert rest == 0 and 2 <= shares <= 4096 + 1 and -(-capacity // shares) >= 97           # 192 rows a share, or what is left of them
