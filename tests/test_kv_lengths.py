"""Lengths outside the page table: such a sequence has no rows in a call, so that
nothing of the cache or the outputs is written for it.  The index arithmetic on the
host, the kernels on the device."""
import ctypes as C

import numpy as np
import pytest

from gollama_b200.device import GlcError
from tests import generation_ref as ref
from tests.test_generation_gpu import CANARY, Batch, append, attend, expect_append, make, same_bits, same_raw, tables
from tests.test_kv_plan import BAD, batch_of, cache_of, host  # noqa: F401

MOST = 64  # four pages of 16


def rows_of(host, batch):  # noqa: F811
    seq, pos, err = np.zeros(batch.num_rows, np.int32), np.zeros(batch.num_rows, np.int32), C.c_int(0)
    host.kv_rows_of(C.byref(cache_of(8, 16, 2, 64)), C.byref(batch), seq.ctypes.data_as(C.c_void_p),
                    pos.ctypes.data_as(C.c_void_p), C.byref(err))
    return list(zip(seq.tolist(), pos.tolist())), err.value


LENGTHS = [MOST + 1, MOST + 6, 10**6, 2**31 - 1, -1, -2**31]


@pytest.mark.parametrize("length", LENGTHS)
def test_a_length_outside_the_table_has_no_rows(host, length):  # noqa: F811
    table = np.zeros((3, 4), np.int32)
    assert rows_of(host, batch_of(table, [5, length, MOST])) == ([(0, 4), (-1, -1), (2, 63)], BAD)
    assert rows_of(host, batch_of(table, [5, length, 9], [0, 1, 4, 6])) == (
        [(0, 4), (-1, -1), (-1, -1), (-1, -1), (2, 7), (2, 8)], BAD)


def batches(ctx, length):
    """Three sequences that fill their tables, the middle one's length then `length`; with one new token each, and
    with several."""
    for news in (None, [2, 3, 4]):
        r = np.random.default_rng(61)
        cache, batch = make(ctx, r, [MOST] * 3, news, 2, 64, 16, spare=2)
        lens = np.array([MOST, length, MOST], np.int32)
        yield r, cache, batch, Batch(ctx, batch.table, lens, batch.starts, batch.rows), np.array([b == 1 for b, _ in batch.positions()])


@pytest.mark.gpu
@pytest.mark.parametrize("length", LENGTHS)
def test_append_of_a_length_outside_the_table_stores_nothing(ctx, length):
    for r, cache, batch, bad, rows in batches(ctx, length):
        q = r.standard_normal((batch.rows, 4 * 64), dtype=np.float32)
        k, v = (r.standard_normal((batch.rows, 128), dtype=np.float32) for _ in "kv")
        cos, sin = tables(64, MOST)
        dq, dk, dv, dc, ds = (ctx.from_numpy(x) for x in (q, k, v, cos, sin))
        out = ctx.from_numpy(np.full_like(q, CANARY))
        ctx.call("glc_kv_append", C.byref(cache.c), C.byref(bad.c), dq.addr, 256, out.addr, 256, 4, dk.addr, 128, dv.addr, 128,
                 dc.addr, ds.addr, MOST)
        with pytest.raises(GlcError, match="out of range"):
            ctx.sync()
        want, _ = expect_append(Copy(cache), batch, q, k, v, 4, cos, sin)
        want[rows] = CANARY
        assert same_bits(out.numpy(), want)
        # the pools: the other sequences' tokens stored, every byte of the middle one's as it was
        held = ref.Pools(cache.pools.pages, 16, 2, 64)
        held.raw = cache.pools.raw.copy()
        for t, (b, pos) in enumerate(batch.positions()):
            if b == 1:
                continue
            at = np.array([pos])
            held.store(0, batch.table[b, pos // 16], pos % 16, *ref.quantize(ref.rotate(k[t].reshape(1, 2, 64), cos, sin, at)[0]))
            held.store(1, batch.table[b, pos // 16], pos % 16, *ref.quantize(v[t].reshape(2, 64)))
        assert same_raw(cache.pools, cache.raw(), held.raw)
        append(ctx, cache, batch, q, k, v, 4, cos, sin)  # the next call is whole
        _, raw = expect_append(cache, batch, q, k, v, 4, cos, sin)
        assert same_raw(cache.pools, cache.raw(), raw)


class Copy:
    """A cache's host image apart from it."""

    def __init__(self, cache):
        p = cache.pools
        self.pools = ref.Pools(p.pages, p.page, p.heads, p.hd)
        self.pools.raw = p.raw.copy()


@pytest.mark.gpu
@pytest.mark.parametrize("length", LENGTHS)
def test_read_of_a_length_outside_the_table_writes_nothing(ctx, length):
    for _, cache, batch, bad, rows in batches(ctx, length):
        got = []
        for b in (batch, bad):
            k, v = (ctx.from_numpy(np.full((batch.rows, 128), CANARY)) for _ in "kv")
            ctx.call("glc_kv_read", C.byref(cache.c), C.byref(b.c), k.addr, 128, v.addr, 128)
            if b is bad:
                with pytest.raises(GlcError, match="out of range"):
                    ctx.sync()
            got.append((k.numpy(), v.numpy()))
        for whole, part in zip(*got):
            assert same_bits(part[~rows], whole[~rows]) and (part[rows] == CANARY).all()


@pytest.mark.gpu
@pytest.mark.parametrize("length", LENGTHS)
def test_attention_of_a_length_outside_the_table_writes_nothing(ctx, length):
    for r, cache, batch, bad, rows in batches(ctx, length):
        q = r.standard_normal((batch.rows, 4 * 64), dtype=np.float32)
        whole, whole_lse = attend(ctx, cache, batch, q, 4)
        dq, o, lse = ctx.from_numpy(q), ctx.from_numpy(np.full(q.shape, CANARY)), ctx.from_numpy(np.full((batch.rows, 4), CANARY))
        ctx.call("glc_attention_kv", C.byref(cache.c), C.byref(bad.c), dq.addr, 256, 4, o.addr, 256, lse.addr)
        with pytest.raises(GlcError, match="out of range"):
            ctx.sync()
        # the others' rows: the same sums, cut into other parts.  Each is within 2 (2^-19.4 s + 2^-18.5) of the
        # exact one relative to the largest value (tests/test_generation_gpu.py), s at most 8 and values at most 3
        # here: 9e-5, and 2^-12 of two
        o, lse = o.numpy(), lse.numpy()
        assert (o[rows] == CANARY).all() and (lse[rows] == CANARY).all()
        np.testing.assert_allclose(o[~rows], whole[~rows], rtol=0, atol=2**-12)
        np.testing.assert_allclose(lse[~rows], whole_lse[~rows], rtol=0, atol=2**-12)
