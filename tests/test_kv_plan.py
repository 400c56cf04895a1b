"""The paged 4-bit cache without a device: the index arithmetic that its
kernels use (gollama_b200/csrc/kv_plan.h, compiled for the host and walked as
the kernels walk it), out-of-range tables and lengths among it, and every
refusal of the generation entry points."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from gollama_b200 import _lib
from gollama_b200._lib import KVBatchC, KVCacheC

HERE = Path(__file__).parent
INVALID, UNSUPPORTED = -1, -6
BAD = 110  # the code that the device error word gets


@pytest.fixture(scope="module")
def host():
    src, lib = HERE / "native" / "kv_host.cpp", HERE / "native" / "_build" / "libkv_host.so"
    lib.parent.mkdir(exist_ok=True)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I/usr/local/cuda/include", "-o", str(lib), str(src)],
                   check=True, capture_output=True)
    h = C.CDLL(str(lib))
    h.test_context.restype = C.c_void_p
    h.test_context_free.argtypes = [C.c_void_p]
    return h


def cache_of(num_pages=64, page=16, kv_heads=2, hd=64, k=4096, v=8192):
    return KVCacheC(k=k, v=v, num_pages=num_pages, page_size=page, num_kv_heads=kv_heads, head_dim=hd)


def batch_of(table, lens, starts=None, rows=None):
    table, lens = np.ascontiguousarray(table, np.int32), np.ascontiguousarray(lens, np.int32)
    starts = None if starts is None else np.ascontiguousarray(starts, np.int32)
    b = KVBatchC(page_table=table.ctypes.data, lens=lens.ctypes.data, starts=0 if starts is None else starts.ctypes.data,
                 num_seqs=len(lens), max_pages=table.shape[1],
                 num_rows=rows if rows is not None else len(lens) if starts is None else int(starts[-1]))
    b.held = (table, lens, starts)
    return b


def walk(host, cache, batch, group, grid, rt=8, warps=16):
    err = C.c_int(0)
    return host.kv_walk(C.byref(cache), C.byref(batch), group, rt, warps, grid, C.byref(err)), err.value


def table_for(lens, page, pages, seed):
    need = max(1, max(-(-max(n, 1) // page) for n in lens))
    return np.random.default_rng(seed).integers(0, pages, (len(lens), need)).astype(np.int32)


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [16, 48, 64, 256, 4096])
@pytest.mark.parametrize("group,lens,news", [
    (1, [1], None), (8, [0, 1, 31, 32, 33, 511, 512, 513, 700], None), (7, [5000, 1, 0, 260], None),
    (4, [900, 64, 5], [5, 64, 5]), (3, [1030, 40, 7], [300, 40, 1]), (8, [700, 3, 1500], [130, 9, 0]),
    (20, [333, 17], [3, 17]), (16, [2000], [1]), (5, [10, 0, 2], [12, 4, 3])])
def test_every_key_is_read_once_by_every_item(host, hd, page, group, lens, news):
    starts = None if news is None else np.concatenate([[0], np.cumsum(news)])
    batch = batch_of(table_for(lens, page, 40, 1), lens, starts)
    for grid, rt, warps in ((1, 8, 4), (3, 8, 16), (148, 8, 16), (592, 8, 4), (148, 16, 8), (444, 32, 4)):
        assert walk(host, cache_of(40, page, 2, hd), batch, group, grid, rt, warps) == (0, 0), grid


def test_walk_of_random_batches(host):
    r = np.random.default_rng(5)
    for i in range(150):
        n = int(r.integers(1, 12))
        news = [int(x) for x in r.integers(0, [2, 9, 200][i % 3] + 1, n)]
        if sum(news) == 0:
            news[0] = 1
        lens = [x + int(r.integers(0, 900)) for x in news]
        page, hd, group = int(r.choice([16, 32, 80])), int(r.choice([32, 64, 96, 128])), int(r.integers(1, 18))
        batch = batch_of(table_for(lens, page, 64, i), lens, np.concatenate([[0], np.cumsum(news)]))
        assert walk(host, cache_of(64, page, int(r.integers(1, 4)), hd), batch, group, int(r.integers(1, 200)), int(r.choice([8, 16, 32])), int(r.choice([4, 8, 12, 16]))) == (0, 0), i


def test_bad_pages_lengths_and_rows_are_neither_read_nor_silent(host):
    cache = cache_of(8, 16, 2, 64)
    ok = np.arange(8, dtype=np.int32).reshape(2, 4)
    for bad in (-1, 8, 2**31 - 1, -2**31):
        t = ok.copy()
        t[1, 2] = bad
        assert walk(host, cache, batch_of(t, [64, 64]), 2, 4) == (0, BAD)
        assert walk(host, cache, batch_of(t, [64, 32]), 2, 4) == (0, 0)  # a page that no token needs
    for lens in ([65, 3], [-1, 3], [3, 2**31 - 1]):
        assert walk(host, cache, batch_of(ok, lens), 2, 4)[1] == BAD
        assert walk(host, cache, batch_of(ok, lens), 2, 4)[0] == 0
    for starts in ([0, 5, 4], [-1, 2, 4], [0, 2, 7]):
        assert walk(host, cache, batch_of(ok, [9, 9], starts, rows=6), 2, 4) == (0, BAD)


def test_starts_that_do_not_ascend_end_the_whole_call(host):
    """Sequences that each claim all rows would have more units than the host allowed
    for: nothing is walked, wherever the bad pair lies."""
    ok = np.zeros((6, 4), np.int32)
    for starts in ([0, 40, 0, 40, 0, 40, 0], [0, 1, 2, 3, 4, 5, 4], [3, 2, 3, 4, 5, 6, 7], [0, 40, 40, 0, 40, 40, 40]):
        got = walk(host, cache_of(8, 16, 1, 64), batch_of(ok, [64] * 6, starts, rows=40), 8, 148, 4, 4)
        assert got == (0, BAD)


def test_units_stay_within_what_the_host_allows_for(host):
    """Groups of 5 to 8 heads in tiles of 4 rows, idle sequences beside one of many rows
    (the walk compares its units with the bound)."""
    for group in (1, 3, 4, 5, 8, 9, 17):
        for lens, news in (([600, 0, 0, 0, 0], [90, 0, 0, 0, 0]), ([700, 700], [700, 1]), ([0] * 8, [1] * 8), ([512] * 3, [1] * 3)):
            batch = batch_of(table_for(lens, 16, 8, 2), lens, np.concatenate([[0], np.cumsum(news)]))
            for rt in (4, 8, 32):
                assert walk(host, cache_of(8, 16, 2, 32), batch, group, 148, rt, 4) == (0, 0), (group, news, rt)


def test_rows_find_their_sequence_and_position(host):
    cache = cache_of(8, 16, 2, 64)
    table = np.zeros((4, 4), np.int32)

    def rows(batch):
        seq, pos, err = np.zeros(batch.num_rows, np.int32), np.zeros(batch.num_rows, np.int32), C.c_int(0)
        host.kv_rows_of(C.byref(cache), C.byref(batch), seq.ctypes.data_as(C.c_void_p), pos.ctypes.data_as(C.c_void_p), C.byref(err))
        return list(zip(seq.tolist(), pos.tolist())), err.value

    # empty sequences, more new tokens than the sequence has, rows before and behind all
    got, err = rows(batch_of(table, [10, 0, 2, 5], [1, 3, 3, 6, 7], rows=9))
    assert err == 0
    assert got == [(-1, -1), (0, 8), (0, 9), (-1, -1), (2, 0), (2, 1), (3, 4), (-1, -1), (-1, -1)]
    got, err = rows(batch_of(table, [1, 0, 64, 7], rows=5))
    assert (got, err) == ([(0, 0), (-1, -1), (2, 63), (3, 6), (-1, -1)], 0)
    assert rows(batch_of(table, [65, 0, 1, 1]))[1] == BAD


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_a_piece_of_8_tokens_falls_in_different_banks(host, hd):
    assert all(host.kv_bank_quads(hd, token, ch) == 8 for token in (0, 8, 16, 24) for ch in range(hd // 32))


# ------------------------------------------------------------------ refusals


class Refused:
    def __init__(self, host):
        self.host, self.lib, self.h = host, _lib.lib(), host.test_context()

    def __call__(self, name, *args):
        rc = getattr(self.lib, name)(self.h, *args)
        buf = C.create_string_buffer(512)
        self.lib.glc_last_error(self.h, buf, 512)
        return rc, buf.value.decode()


@pytest.fixture()
def call(host):
    c = Refused(host)
    yield c
    host.test_context_free(c.h)


P = 1 << 20  # an aligned address that no refused call looks at


def good_batch(rows=4, seqs=4, max_pages=8):
    return KVBatchC(page_table=P, lens=P, starts=0, num_seqs=seqs, max_pages=max_pages, num_rows=rows)


def test_pool_bytes():
    lib, n = _lib.lib(), C.c_size_t()
    for pages, page, heads, hd in ((1, 16, 1, 32), (100, 48, 4, 64), (1 << 20, 64, 8, 128)):
        c = cache_of(pages, page, heads, hd, 0, 0)
        assert lib.glc_kv_cache_bytes(C.byref(c), C.byref(n)) == 0
        assert n.value == pages * page * heads * hd * 9 // 16
    for bad in (cache_of(0), cache_of(page=8), cache_of(page=0), cache_of(page=65552), cache_of(kv_heads=0)):
        assert lib.glc_kv_cache_bytes(C.byref(bad), C.byref(n)) == INVALID
    assert lib.glc_kv_cache_bytes(C.byref(cache_of(hd=80)), C.byref(n)) == UNSUPPORTED
    assert lib.glc_kv_cache_bytes(None, C.byref(n)) == INVALID
    assert lib.glc_kv_cache_bytes(C.byref(cache_of()), None) == INVALID


APPEND = dict(cache=cache_of(), batch=good_batch(), q=P, q_ld=256, q_out=P, q_out_ld=256, heads=4, k=P, k_ld=128, v=P, v_ld=128,
              cos=P, sin=P, rows=64)
READ = dict(cache=cache_of(), batch=good_batch(), k=P, k_ld=128, v=P, v_ld=128)
ATTEND = dict(cache=cache_of(), batch=good_batch(), q=P, q_ld=256, heads=4, o=P, o_ld=256, lse=P)
SAMPLE = dict(logits=P, ld=100, rows=2, vocab=100, t=P, k=P, p=P, m=P, u=P, tokens=P, logp=P)

CACHES = [("cache", None, INVALID), ("cache", cache_of(num_pages=0), INVALID), ("cache", cache_of(page=24), INVALID),
          ("cache", cache_of(page=-16), INVALID), ("cache", cache_of(kv_heads=-1), INVALID), ("cache", cache_of(hd=48), UNSUPPORTED),
          ("cache", cache_of(hd=256), UNSUPPORTED), ("cache", cache_of(k=0), INVALID), ("cache", cache_of(v=8), INVALID),
          ("batch", None, INVALID), ("batch", good_batch(rows=-1), INVALID), ("batch", good_batch(seqs=-1), INVALID),
          ("batch", good_batch(max_pages=0), INVALID), ("batch", good_batch(rows=3), INVALID),
          ("batch", good_batch(max_pages=(1 << 26) + 1), INVALID), ("batch", KVBatchC(num_seqs=2, max_pages=2, num_rows=2), INVALID)]


def refused(call, name, base, field, value, code):
    args = [C.byref(x) if isinstance(x, C.Structure) else x for x in {**base, field: value}.values()]
    rc, text = call(name, *args)
    assert rc == code and text.startswith(name[4:] + ": "), (rc, text)


@pytest.mark.parametrize("field,value,code", CACHES + [
    ("q", 0, INVALID), ("q_out", 0, INVALID), ("heads", 0, INVALID), ("heads", 5, INVALID), ("q_ld", 252, INVALID), ("q_ld", 258, INVALID),
    ("q_out_ld", 255, INVALID), ("k", 0, INVALID), ("v", 0, INVALID), ("k_ld", 124, INVALID), ("v_ld", 130, INVALID), ("cos", 0, INVALID),
    ("sin", 0, INVALID), ("rows", 0, INVALID), ("q", P + 4, INVALID), ("k", P + 8, INVALID), ("sin", P + 4, INVALID)])
def test_append_refuses(call, field, value, code):
    refused(call, "glc_kv_append", APPEND, field, value, code)


def test_append_refuses_queries_in_place_of_another_stride(call):
    refused(call, "glc_kv_append", {**APPEND, "q_out": P}, "q_out_ld", 260, INVALID)


@pytest.mark.parametrize("field,value,code", CACHES + [
    ("k_ld", 127, INVALID), ("v_ld", 130, INVALID), ("k", P + 4, INVALID), ("v", P + 2, INVALID)])
def test_read_refuses(call, field, value, code):
    refused(call, "glc_kv_read", READ, field, value, code)


def test_read_refuses_no_output(call):
    assert call("glc_kv_read", C.byref(cache_of()), C.byref(good_batch()), 0, 128, 0, 128)[0] == INVALID


@pytest.mark.parametrize("field,value,code", CACHES + [
    ("q", 0, INVALID), ("o", 0, INVALID), ("heads", 0, INVALID), ("heads", 3, INVALID), ("heads", -2, INVALID), ("q_ld", 252, INVALID),
    ("o_ld", 257, INVALID), ("o", P + 4, INVALID), ("lse", P + 1, INVALID)])
def test_attention_refuses(call, field, value, code):
    refused(call, "glc_attention_kv", ATTEND, field, value, code)


def test_attention_refuses_more_units_than_are_counted(call):
    # 8 heads in tiles of 4: two tiles a token, 8193 units each
    batch = KVBatchC(page_table=P, lens=P, starts=P, num_seqs=1, max_pages=65536, num_rows=200000)
    refused(call, "glc_attention_kv", {**ATTEND, "cache": cache_of(kv_heads=1), "heads": 8, "q_ld": 512, "o_ld": 512}, "batch", batch, INVALID)


@pytest.mark.parametrize("field,value,code", [
    ("rows", -1, INVALID), ("vocab", 0, INVALID), ("ld", 99, INVALID), ("logits", 0, INVALID), ("t", 0, INVALID), ("u", 0, INVALID),
    ("tokens", 0, INVALID), ("tokens", P + 4, INVALID), ("logits", P + 2, INVALID), ("k", P + 1, INVALID), ("rows", 2**31 - 1, INVALID)])
def test_sample_refuses(call, field, value, code):
    refused(call, "glc_sample", SAMPLE, field, value, code)


def test_sample_refuses_a_vocabulary_that_no_cluster_holds(call):
    refused(call, "glc_sample", {**SAMPLE, "ld": 400000}, "vocab", 344065, UNSUPPORTED)


def test_calls_without_work_return_at_once(call):
    for b in (good_batch(rows=0, seqs=0), KVBatchC(max_pages=1)):
        for name, base in (("glc_kv_append", APPEND), ("glc_kv_read", READ), ("glc_attention_kv", ATTEND)):
            args = [C.byref(x) if isinstance(x, C.Structure) else x for x in {**base, "batch": b}.values()]
            assert call(name, *args)[0] == 0
    assert call("glc_sample", *{**SAMPLE, "rows": 0}.values())[0] == 0


def test_without_a_context():
    lib = _lib.lib()
    assert lib.glc_kv_append(None, *[C.byref(x) if isinstance(x, C.Structure) else x for x in APPEND.values()]) == INVALID
    assert lib.glc_kv_read(None, *[C.byref(x) if isinstance(x, C.Structure) else x for x in READ.values()]) == INVALID
    assert lib.glc_attention_kv(None, *[C.byref(x) if isinstance(x, C.Structure) else x for x in ATTEND.values()]) == INVALID
    assert lib.glc_sample(None, *SAMPLE.values()) == INVALID


def test_struct_layout_matches_the_header():
    """The ctypes structures are what the library reads: the refusals above see
    their fields, and the sizes are those of the C declarations."""
    assert C.sizeof(KVCacheC) == 32 and C.sizeof(KVBatchC) == 40
