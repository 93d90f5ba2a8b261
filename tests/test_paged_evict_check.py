"""fa_check_paged_evict: what fa_paged_evict refuses, before there is a workspace (nothing is launched)."""
import ctypes

import pytest

from test_paged_cpu import CACHE_CASES, _cache, _code, _evict, _lib


@pytest.mark.parametrize("over,code", [
    (dict(), None), (dict(keep=1 << 28), "PAGES"), (dict(keep=0), "PAGES"), (dict(new_table_width=1 << 28, keep=1 << 30), "OVERFLOW"),
    (dict(sums=None), "NULL"), (dict(new_table_stride=-1), "ALIGN"), (dict(sums_width=159), "PAGES"),
    (dict(sums_width=159, max_len=159), None), (dict(sums_width=159, max_len=160), "PAGES"), (dict(max_len=1 << 30), None),
    (dict(max_len=-1), "SHAPE"),
], ids=lambda x: str(x))
def test_check(over, code):
    assert _lib.lib().fa_check_paged_evict(ctypes.byref(_evict(**over))) == (0 if code is None else _code(code))


@pytest.mark.parametrize("over,code", CACHE_CASES, ids=lambda x: str(x))
def test_cache(over, code):
    assert _lib.lib().fa_check_paged_evict(ctypes.byref(_evict(cache=_cache(**over)))) == _code(code)


def test_null():
    assert _lib.lib().fa_check_paged_evict(None) == _code("NULL")
