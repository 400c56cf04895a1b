"""Every kernel of the attention over the 4-bit cache against its definition in 64
bits, on batches that the library's own rule gives to it (tests/kv_variants.py)."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from tests.kv_variants import CASES, VARIANTS, batches
from tests.test_generation_gpu import attend, check, make, same_bits
from tests.test_kv_plan import batch_of, cache_of, table_for

HERE = Path(__file__).parent
SMS = 148


@pytest.fixture(scope="module")
def shape():
    src, lib = HERE / "native" / "kv_variant_host.cpp", HERE / "native" / "_build" / "libkv_variant_host.so"
    lib.parent.mkdir(exist_ok=True)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True, capture_output=True)
    h = C.CDLL(str(lib))

    def of(hd, kv_heads, group, page, lens, news):
        starts = None if news is None else np.concatenate([[0], np.cumsum(news)])
        table, out = table_for(lens, page, 40, 1), (C.c_int * 6)()
        assert h.kv_shape(C.byref(cache_of(40, page, kv_heads, hd)), C.byref(batch_of(table, lens, starts)), group, SMS, out) == 0
        return dict(zip(("tiles", "warps", "alone", "most", "cut", "items"), out))

    return of


@pytest.mark.parametrize("hd,tiles,warps", VARIANTS)
def test_the_batches_reach_what_they_are_for(shape, hd, tiles, warps):
    """The variant, and: a warp takes more tiles than its ring has stages (uneven), pieces of one item (even), items cut
    between CTAs and whole ones."""
    got = {name: shape(hd, *rest) for name, *rest in batches(hd, tiles, warps)}
    assert all((g["tiles"], g["warps"]) == (tiles, warps) for g in got.values()), got
    assert not got["uneven"]["alone"] and got["uneven"]["most"] > 3 and got["uneven"]["cut"] > 0, got
    assert got["even"]["alone"] and got["even"]["cut"] > 0, got
    assert got["short"]["cut"] < got["short"]["items"], got


@pytest.mark.gpu
@pytest.mark.parametrize("hd,tiles,warps,which", CASES)
def test_every_kernel_is_the_definition(ctx, hd, tiles, warps, which):
    _, kv_heads, group, page, lens, news = batches(hd, tiles, warps)[which]
    r = np.random.default_rng(hd + tiles + warps + which)
    cache, batch = make(ctx, r, lens, news, kv_heads, hd, page, extra_rows=0)
    heads = kv_heads * group
    q = 2 * r.standard_normal((batch.rows, heads * hd), dtype=np.float32)
    o, lse = attend(ctx, cache, batch, q, heads)
    check(cache, batch, q, heads, o, lse)
    o2, lse2 = attend(ctx, cache, batch, q, heads)
    assert same_bits(o, o2) and same_bits(lse, lse2)
