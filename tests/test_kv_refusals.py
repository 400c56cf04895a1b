"""Refusals of the cache's entry points beside those of tests/test_kv_plan.py; none of the
calls reaches a device."""
import ctypes as C

import pytest

from gollama_b200 import _lib
from gollama_b200._lib import KVBatchC
from tests.test_kv_plan import APPEND, ATTEND, INVALID, READ, P, cache_of, call, host, refused  # noqa: F401


@pytest.mark.parametrize("name,base", [("glc_kv_append", APPEND), ("glc_kv_read", READ), ("glc_attention_kv", ATTEND)])
@pytest.mark.parametrize("field", ["page_table", "lens", "starts"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_whole_numbers_that_are_not_aligned(call, name, base, field, off):  # noqa: F811
    batch = KVBatchC(page_table=P, lens=P, starts=P, num_seqs=4, max_pages=8, num_rows=4)
    setattr(batch, field, P + off)
    refused(call, name, base, "batch", batch, INVALID)


def test_attention_in_place_of_another_stride(call):  # noqa: F811
    """A row written would be another one's query."""
    for ld, o_ld in ((256, 260), (260, 256), (512, 1024)):
        refused(call, "glc_attention_kv", {**ATTEND, "q_ld": ld}, "o_ld", o_ld, INVALID)


@pytest.mark.parametrize("pages,page,heads,hd", [(2**31 - 1, 65536, 2**31 - 1, 128), (2**31 - 1, 65536, 2**19, 128), (2**31 - 1, 16, 2**31 - 1, 32)])
def test_pools_beyond_64_bits(call, pages, page, heads, hd):  # noqa: F811
    """The number of bytes would be cut off to a small one."""
    lib, n = _lib.lib(), C.c_size_t(7)
    cache = cache_of(pages, page, heads, hd)
    assert pages * page * heads * hd * 9 // 16 >= 2**62
    assert lib.glc_kv_cache_bytes(C.byref(cache), C.byref(n)) == INVALID and n.value == 7
    for name, base in (("glc_kv_append", APPEND), ("glc_kv_read", READ), ("glc_attention_kv", ATTEND)):
        refused(call, name, base, "cache", cache, INVALID)


def test_the_largest_pools_are_counted():
    lib, n = _lib.lib(), C.c_size_t()
    cache = cache_of(2**31 - 1, 4096, 128, 128)
    assert lib.glc_kv_cache_bytes(C.byref(cache), C.byref(n)) == 0 and n.value == (2**31 - 1) * 4096 * 128 * 128 * 9 // 16
