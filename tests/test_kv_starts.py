"""Starts that do not ascend, in the cache's append and read-back: reported wherever
the wrong pair lies, and nothing is written but what the other pairs name."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from gollama_b200.device import GlcError
from tests.test_generation_gpu import CANARY, Batch, make, same_bits
from tests.test_kv_plan import BAD, batch_of, cache_of

HERE = Path(__file__).parent
ROWS = 8
WRONG = [[0, 5, 3, 8], [0, 2, 1, 8], [0, 8, 8, 7], [0, 3, 6, 9], [-1, 2, 4, 8], [0, 8, 0, 8], [9, 9, 9, 9], [0, 8, 20, 30]]


@pytest.fixture(scope="module")
def look():
    src, lib = HERE / "native" / "kv_look_host.cpp", HERE / "native" / "_build" / "libkv_look_host.so"
    lib.parent.mkdir(exist_ok=True)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True, capture_output=True)
    return C.CDLL(str(lib)).kv_look_of


@pytest.mark.parametrize("threads", [1, 2, 100])
def test_every_wrong_pair_is_seen(look, threads):
    table = np.zeros((3, 4), np.int32)
    cache = cache_of(8, 16, 2, 64)
    for starts in WRONG:
        assert look(C.byref(cache), C.byref(batch_of(table, [20, 20, 20], starts, rows=ROWS)), threads) == BAD, starts
    for starts in ([0, 0, 0, 0], [0, 3, 3, 8], [2, 4, 6, 7]):
        assert look(C.byref(cache), C.byref(batch_of(table, [20, 20, 20], starts, rows=ROWS)), threads) == 0, starts
    assert look(C.byref(cache), C.byref(batch_of(table, [20, 65, 20], [0, 3, 3, 8], rows=ROWS)), threads) == BAD  # a length without rows


def claims(starts, lens):
    """Rows, and (sequence, position)s, that the pairs that ascend name."""
    rows, tokens = set(), set()
    for b, n in enumerate(lens):
        first, end = starts[b], starts[b + 1]
        if 0 <= first <= end <= ROWS:
            rows |= set(range(first, end))
            tokens |= {(b, n - (end - first) + i) for i in range(end - first)}
    return rows, tokens


@pytest.mark.gpu
@pytest.mark.parametrize("starts", WRONG)
def test_wrong_starts_are_reported_by_append_and_read(ctx, starts):
    r = np.random.default_rng(81)
    lens = [20, 33, 40]
    cache, good = make(ctx, r, lens, [2, 3, 3], 2, 64, 16)
    bad = Batch(ctx, good.table, lens, np.array(starts, np.int32), ROWS)
    rows, tokens = claims(starts, lens)
    k, v, q = (r.standard_normal((ROWS, n), dtype=np.float32) for n in (128, 128, 256))
    dk, dv, dq = (ctx.from_numpy(x) for x in (k, v, q))
    out = ctx.from_numpy(np.full_like(q, CANARY))
    ctx.call("glc_kv_append", C.byref(cache.c), C.byref(bad.c), dq.addr, 256, out.addr, 256, 4, dk.addr, 128, dv.addr, 128, 0, 0, 0)
    with pytest.raises(GlcError, match="out of range"):
        ctx.sync()
    out, raw = out.numpy(), cache.raw()
    for t in range(ROWS):
        assert same_bits(out[t], q[t] if t in rows else np.full_like(q[t], CANARY))
    p = cache.pools
    may = {(int(good.table[b, pos // 16]), pos % 16) for b, pos in tokens}
    before = p.raw.copy()
    for side in (0, 1):
        for page in range(p.pages):
            for slot in range(16):
                if (page, slot) in may:
                    continue
                now = []
                for x in (before, raw):
                    p.raw = x
                    now.append((p.codes[side, page, :, slot].copy(), p.scales[side, page, :, slot].copy()))
                assert same_bits(now[0][0], now[1][0]) and same_bits(now[0][1], now[1][1])
    bk, bv = (ctx.from_numpy(np.full((ROWS, 128), CANARY)) for _ in "kv")
    ctx.call("glc_kv_read", C.byref(cache.c), C.byref(bad.c), bk.addr, 128, bv.addr, 128)
    with pytest.raises(GlcError, match="out of range"):
        ctx.sync()
    for x in (bk.numpy(), bv.numpy()):
        for t in range(ROWS):
            assert (x[t] == CANARY).all() == (t not in rows)
