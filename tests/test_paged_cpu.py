"""Paged key-value caches without a GPU: the C ABI's argument checks and the Python functions' (nothing is launched)."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from conftest import ROOT, load_mod

_lib = load_mod("_lib")
_ops = load_mod("_ops")
FAKE = 1 << 20  # never dereferenced


def _cache(**over):
    c = _lib.PagedCache()
    c.k, c.v, c.table, c.lens = FAKE, FAKE, FAKE, FAKE
    c.k_stride[:] = c.v_stride[:] = (8 * 16 * 64, 16 * 64, 64)
    c.table_stride, c.batch, c.pages, c.page_size, c.table_width, c.heads_kv, c.head_dim = 10, 2, 40, 16, 10, 8, 64
    c.dtype, c.k_descale, c.v_descale = _lib.FA_DTYPE_BF16, 1.0, 1.0
    for k, v in over.items():
        if k.endswith("_stride") and k != "table_stride":
            getattr(c, k)[:] = v
        else:
            setattr(c, k, v)
    return c


CACHE_CASES = [
    (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(table=None), "NULL"), (dict(lens=None), "NULL"),
    (dict(batch=0), "SHAPE"), (dict(heads_kv=0), "SHAPE"), (dict(pages=0), "PAGES"), (dict(page_size=0), "PAGES"),
    (dict(table_width=0), "PAGES"), (dict(head_dim=48), "HEAD_DIM"), (dict(head_dim=256), "HEAD_DIM"), (dict(dtype=0), "DTYPE"),
    (dict(dtype=5), "DTYPE"), (dict(k=FAKE + 8), "ALIGN"), (dict(table=FAKE + 2), "ALIGN"), (dict(k_stride=(-8, 8, 8)), "ALIGN"),
    (dict(v_stride=(8, 12, 8)), "ALIGN"), (dict(table_stride=-1), "ALIGN"), (dict(page_size=1 << 20, table_width=1 << 10), "OVERFLOW"),
    (dict(dtype=3, head_dim=32), "HEAD_DIM"),
]


def _code(name):
    return {"NULL": -1, "SHAPE": -2, "HEAD_DIM": -3, "DTYPE": -4, "ALIGN": -5, "MASK": -6, "WORKSPACE": -7, "OVERFLOW": -9,
            "SCALE": -10, "PAGES": -12}[name]


def _append(c, k=FAKE, v=FAKE, ks=(64, 512), vs=(64, 512), rows=2, dtype=1, cu=None):
    return _lib.lib().fa_paged_append(ctypes.byref(c) if c else None, k, v, (ctypes.c_int64 * 2)(*ks), (ctypes.c_int64 * 2)(*vs), rows,
                                      dtype, cu, None)


@pytest.mark.parametrize("over,code", CACHE_CASES, ids=lambda x: str(x))
def test_cache_checks(over, code):
    assert _append(_cache(**over)) == _code(code)
    p = _attn(cache=_cache(**over))
    assert _lib.lib().fa_paged_attention(ctypes.byref(p), FAKE, 1 << 30, None) == _code(code)
    assert _lib.lib().fa_paged_workspace_bytes(ctypes.byref(p)) == 0
    e = _evict(cache=_cache(**over))
    assert _lib.lib().fa_paged_evict(ctypes.byref(e), FAKE, 1 << 30, None) == _code(code)


def test_append_checks():
    L = _lib.lib()
    assert _append(None) == _code("NULL")
    assert _append(_cache(), rows=3) == _code("SHAPE")
    assert _append(_cache(), rows=-1, cu=FAKE) == _code("SHAPE")
    assert _append(_cache(), dtype=2) == _code("DTYPE")
    assert _append(_cache(dtype=3), dtype=4) == _code("DTYPE")
    assert _append(_cache(), k=FAKE + 2) == _code("ALIGN")
    assert _append(_cache(), vs=(64, 12)) == _code("ALIGN")
    assert _append(_cache(), k=None) == _code("NULL")
    for bad in (0.0, float("nan"), float("inf"), 1e-300):
        assert _append(_cache(dtype=3, k_descale=bad)) == _code("SCALE")
    assert _append(_cache(), rows=0, cu=FAKE, k=None, v=None) == 0  # nothing to do, nothing launched
    assert L.fa_strerror(-12).decode().startswith("invalid paged cache")


def _attn(cache=None, **over):
    p = _lib.PagedAttentionParams()
    p.cache = cache if cache is not None else _cache()
    p.q, p.o, p.heads_q, p.max_len, p.window, p.sink, p.dtype, p.softmax_scale = FAKE, FAKE, 64, 160, 128, 0, p.cache.dtype, 0.125
    if p.cache.dtype == 3:
        p.dtype = 1
    p.q_stride[:] = p.o_stride[:] = (4096, 64)
    for k, v in over.items():
        if k.endswith("_stride"):
            getattr(p, k)[:] = v
        else:
            setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,code", [
    (dict(q=None), "NULL"), (dict(o=None), "NULL"), (dict(heads_q=60), "SHAPE"), (dict(heads_q=0), "SHAPE"), (dict(max_len=0), "SHAPE"),
    (dict(dtype=2), "DTYPE"), (dict(dtype=3), "DTYPE"), (dict(window=0), "MASK"), (dict(softmax_scale=float("nan")), "SCALE"),
    (dict(q=FAKE + 4), "ALIGN"), (dict(o_stride=(4096, 60)), "ALIGN"), (dict(sinks=FAKE + 1), "ALIGN"),
    (dict(weight_sums=FAKE, sums_width=159), "PAGES"), (dict(weight_sums=FAKE, sums_width=160, sums_stride=(-1, 0)), "ALIGN"),
], ids=lambda x: str(x))
def test_attention_checks(over, code):
    p = _attn(**over)
    assert _lib.lib().fa_paged_attention(ctypes.byref(p), FAKE, 1 << 30, None) == _code(code)


def test_attention_workspace():
    L = _lib.lib()
    assert L.fa_paged_workspace_bytes(None) == 0
    small = L.fa_paged_workspace_bytes(ctypes.byref(_attn()))
    assert small == 256
    big = L.fa_paged_workspace_bytes(ctypes.byref(_attn(cache=_cache(table_width=1000, pages=2000), max_len=16000, window=16000)))
    assert big > 256
    sums = _attn(weight_sums=FAKE, sums_width=160)
    need = L.fa_paged_workspace_bytes(ctypes.byref(sums))
    assert need >= 2 * 64 * 128 * 4  # a unit of 128 keys for each sequence and query head
    for ws, n in ((None, need), (FAKE + 16, need), (FAKE, need - 1)):
        assert L.fa_paged_attention(ctypes.byref(sums), ws, n, None) == _code("WORKSPACE")
    q8 = _attn(cache=_cache(dtype=3, k_descale=float("inf")))
    assert L.fa_paged_attention(ctypes.byref(q8), FAKE, 1 << 20, None) == _code("SCALE")
    # sizes past the launches' range
    wide = _attn(cache=_cache(batch=1 << 30, table_width=1 << 20, page_size=16), max_len=1 << 24, window=1 << 24)
    assert L.fa_paged_attention(ctypes.byref(wide), FAKE, 1 << 40, None) == _code("OVERFLOW")


def _evict(cache=None, **over):
    p = _lib.PagedEvictParams()
    p.cache = cache if cache is not None else _cache()
    p.sums, p.new_sums, p.new_table, p.new_lens = FAKE, FAKE, FAKE, FAKE
    p.sums_stride[:] = p.new_sums_stride[:] = (8 * 160, 160)
    p.new_table_stride, p.sums_width, p.new_table_width, p.keep, p.sink, p.recent = 4, 160, 4, 64, 4, 16
    for k, v in over.items():
        if k.endswith("sums_stride"):
            getattr(p, k)[:] = v
        else:
            setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,code", [
    (dict(sums=None), "NULL"), (dict(new_sums=None), "NULL"), (dict(new_table=None), "NULL"), (dict(new_lens=None), "NULL"),
    (dict(keep=0), "PAGES"), (dict(sink=-1), "PAGES"), (dict(recent=-1), "PAGES"), (dict(sink=40, recent=25), "PAGES"),
    (dict(sums_width=159), "PAGES"), (dict(new_table_width=3), "PAGES"), (dict(sums=FAKE + 1), "ALIGN"),
    (dict(new_sums_stride=(-1, 1)), "ALIGN"), (dict(new_table_stride=-1), "ALIGN"),
], ids=lambda x: str(x))
def test_evict_checks(over, code):
    assert _lib.lib().fa_paged_evict(ctypes.byref(_evict(**over)), FAKE, 1 << 30, None) == _code(code)


def test_evict_workspace():
    L = _lib.lib()
    need = L.fa_paged_evict_workspace_bytes(2, 8, 64, 160)
    assert need == 2 * 8 * 64 * 4 and L.fa_paged_evict_workspace_bytes(0, 8, 64, 160) == 0
    assert L.fa_paged_evict_workspace_bytes(2, 8, 64, 1 << 17) > need  # (several workgroups a head)
    for ws, n in ((None, need), (FAKE + 16, need), (FAKE, need - 1)):
        assert L.fa_paged_evict(ctypes.byref(_evict()), ws, n, None) == _code("WORKSPACE")


def test_sizes_whose_products_pass_64_bits():
    L, many = _lib.lib(), dict(batch=1 << 28, heads_kv=1 << 28, k_stride=(0, 0, 64), v_stride=(0, 0, 64))
    p = _attn(cache=_cache(**many), heads_q=1 << 28)
    assert L.fa_paged_attention(ctypes.byref(p), FAKE, 1 << 40, None) == _code("OVERFLOW")
    assert L.fa_paged_evict(ctypes.byref(_evict(_cache(**many))), FAKE, 1 << 40, None) == _code("OVERFLOW")
    # heads_kv within its own limit: batch * heads * 256 threads is 2^60 and more, the kept entries' bytes too
    q = _cache(**{**many, "heads_kv": 1 << 23, "batch": 1 << 30})
    p = _attn(cache=q, heads_q=1 << 30)
    assert L.fa_paged_attention(ctypes.byref(p), FAKE, 1 << 40, None) == _code("OVERFLOW")
    assert L.fa_paged_evict(ctypes.byref(_evict(q)), FAKE, 1 << 40, None) == _code("OVERFLOW")


def test_struct_layouts_match_header():
    src = ('#include "fa_gfx950.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){printf("%zu %zu %zu %zu %zu %zu\\n",'
           "sizeof(fa_paged_cache), sizeof(fa_paged_attention_params), sizeof(fa_paged_evict_params), offsetof(fa_paged_cache, k_descale),"
           "offsetof(fa_paged_attention_params, softmax_scale), offsetof(fa_paged_evict_params, recent));return 0;}\n")
    tmp = tempfile.mkdtemp(prefix="fa_layout_")
    cfile, exe = os.path.join(tmp, "layout.c"), os.path.join(tmp, "layout")
    with open(cfile, "w") as f:
        f.write(src)
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), cfile, "-o", exe], check=True)
    vals = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    C, A, E = _lib.PagedCache, _lib.PagedAttentionParams, _lib.PagedEvictParams
    assert vals == [ctypes.sizeof(C), ctypes.sizeof(A), ctypes.sizeof(E), C.k_descale.offset, A.softmax_scale.offset, E.recent.offset]


@pytest.mark.parametrize("binding", [True, False])
def test_cpu_tensors_are_refused(fa, monkeypatch, binding):
    if not binding:
        monkeypatch.setattr(_ops, "_BINDING", None)
    pages = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x, q = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        fa.paged_append(x, x, pages, pages, table, lens)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        fa.paged_attention(q, pages, pages, table, lens)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        fa.paged_evict(pages, pages, table, lens, torch.zeros(1, 2, 32), 16, table.clone())
    with pytest.raises(ValueError, match="cu_seqlens"):
        fa.paged_append(x, x, pages, pages, table, lens, cu_seqlens=torch.tensor([0, 2]))
