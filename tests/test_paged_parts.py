"""Which calls over pages with the slots first are cut into twice as many runs (the workspace has two slots a run): large ones whose
slots have rows of 1024 bytes and more, in entries of at most 128."""
import ctypes

import pytest

from test_paged_cpu import _attn, _cache, _lib


def workspace(D, Hkv, dtype, slots_first, tokens=131072):
    page = 64
    stride = (Hkv * page * D, D, Hkv * D) if slots_first else (Hkv * page * D, page * D, D)
    c = _cache(batch=4, page_size=page, table_width=tokens // page, pages=4 * tokens // page, heads_kv=Hkv, head_dim=D, dtype=dtype,
               k_stride=stride, v_stride=stride)
    p = _attn(cache=c, heads_q=8 * Hkv, max_len=tokens, window=tokens, q_stride=(8 * Hkv * D, D), o_stride=(8 * Hkv * D, D))
    n = _lib.lib().fa_paged_workspace_bytes(ctypes.byref(p))
    assert n > 256
    return n


@pytest.mark.parametrize("D,Hkv,dtype,twice", [(64, 8, 1, True), (64, 16, 2, True), (32, 16, 1, True), (16, 32, 1, True), (128, 8, 3, True),
                                               (32, 8, 4, True), (128, 4, 1, False), (128, 8, 1, False), (64, 4, 1, False), (32, 8, 1, False),
                                               (16, 16, 1, False), (64, 8, 3, False), (128, 4, 4, False)])
def test_twice_as_many_runs(D, Hkv, dtype, twice):
    assert (workspace(D, Hkv, dtype, True) > 1.5 * workspace(D, Hkv, dtype, False)) == twice


def test_small_calls_and_heads_first_are_not():
    assert workspace(64, 8, 1, True, 4096) == workspace(64, 8, 1, False, 4096)
