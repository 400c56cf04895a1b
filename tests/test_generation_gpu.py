"""The paged 4-bit cache, the attention over it and sampling on the device,
against their definitions in 64 bits (tests/generation_ref.py)."""
import ctypes as C

import numpy as np
import pytest

from gollama_b200._lib import KVBatchC, KVCacheC
from gollama_b200.device import GlcError
from tests import generation_ref as ref

pytestmark = pytest.mark.gpu

CANARY = np.float32(-7.25)


class Cache:
    def __init__(self, ctx, pools):
        self.ctx, self.pools = ctx, pools
        self.k, self.v = ctx.from_numpy(pools.raw[0]), ctx.from_numpy(pools.raw[1])
        self.c = KVCacheC(k=self.k.addr, v=self.v.addr, num_pages=pools.pages, page_size=pools.page,
                          num_kv_heads=pools.heads, head_dim=pools.hd)

    def raw(self):
        return np.stack([self.k.numpy(), self.v.numpy()])


class Batch:
    def __init__(self, ctx, table, lens, starts=None, rows=None):
        self.table, self.lens = np.ascontiguousarray(table, np.int32), np.ascontiguousarray(lens, np.int32)
        self.starts = None if starts is None else np.ascontiguousarray(starts, np.int32)
        self.rows = rows if rows is not None else len(lens) if starts is None else int(starts[-1])
        self.d = [ctx.from_numpy(self.table), ctx.from_numpy(self.lens), None if starts is None else ctx.from_numpy(self.starts)]
        self.c = KVBatchC(page_table=self.d[0].addr, lens=self.d[1].addr, starts=0 if starts is None else self.d[2].addr,
                          num_seqs=len(lens), max_pages=self.table.shape[1], num_rows=self.rows)

    def positions(self):
        """(sequence, position) of every row; position -1 where it has none."""
        out = [(-1, -1)] * self.rows
        for b, n in enumerate(self.lens):
            first, end = (b, b + 1) if self.starts is None else (self.starts[b], self.starts[b + 1])
            for t in range(first, end):
                out[t] = (b, max(-1, int(n) - (end - first) + t - first))
        return out


def make(ctx, r, lens, news=None, heads=2, hd=64, page=16, spare=3, extra_rows=0, filled=True):
    """A cache with the sequences in pages of their own, in random order."""
    need = [-(-max(int(n), 1) // page) for n in lens]
    pages = sum(need) + spare
    order = r.permutation(pages)
    table = np.full((len(lens), max(need)), -5, np.int32)  # entries that no token needs are no pages
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pools = ref.Pools(pages, page, heads, hd, r if filled else None)
    starts = None if news is None else np.concatenate([[0], np.cumsum(news)])
    rows = (len(lens) if news is None else int(starts[-1])) + extra_rows
    return Cache(ctx, pools), Batch(ctx, table, lens, starts, rows)


def tables(hd, rows):
    pos = np.arange(rows)[:, None]
    f = 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    return np.cos(pos * f).astype(np.float32), np.sin(pos * f).astype(np.float32)


def append(ctx, cache, batch, q, k, v, heads, cos=None, sin=None, q_out=None, table_rows=None):
    """Calls with operands of their own strides; returns q_out's values."""
    dq, dk, dv = (None if x is None else ctx.from_numpy(x) for x in (q, k, v))
    out = None if q is None else ctx.from_numpy(np.full_like(q, CANARY))
    dc, ds = (None if x is None else ctx.from_numpy(x) for x in (cos, sin))
    p = lambda x: 0 if x is None else x.addr  # noqa: E731
    ctx.call("glc_kv_append", C.byref(cache.c), C.byref(batch.c), p(dq), 0 if q is None else q.shape[1], p(out),
             0 if q is None else q.shape[1], heads, p(dk), k.shape[1], p(dv), v.shape[1], p(dc), p(ds),
             0 if cos is None else cos.shape[0] if table_rows is None else table_rows)
    ctx.sync()
    return None if q is None else out.numpy()


def expect_append(cache, batch, q, k, v, heads, cos, sin):
    """What append leaves: (q_out, raw pools)."""
    p = cache.pools
    want = np.full_like(q, CANARY)
    for t, (b, pos) in enumerate(batch.positions()):
        if pos < 0:
            continue
        at = np.array([pos])
        turn = (lambda x: ref.rotate(x, cos, sin, at)) if cos is not None else (lambda x: x)
        want[t] = turn(q[t].reshape(1, heads, p.hd)).reshape(-1)
        page, slot = batch.table[b, pos // p.page], pos % p.page
        p.store(0, page, slot, *ref.quantize(turn(k[t].reshape(1, p.heads, p.hd))[0]))
        p.store(1, page, slot, *ref.quantize(v[t].reshape(p.heads, p.hd)))
    return want, p.raw


def same_bits(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and np.array_equal(a.view(np.uint8), b.view(np.uint8))


def same_raw(pools, got, want):
    """Pools equal bit for bit, scales that are NaN in both counted equal."""
    p = ref.Pools(pools.pages, pools.page, pools.heads, pools.hd)
    p.raw = got
    g_codes, g_scales = p.codes.copy(), p.scales.copy()
    p.raw = want
    nan = np.isnan(g_scales) & np.isnan(p.scales)
    return np.array_equal(g_codes, p.codes) and np.array_equal(np.where(nan, 0, g_scales.view(np.uint16)), np.where(nan, 0, p.scales.view(np.uint16)))


# ------------------------------------------------------------------ append and read


@pytest.mark.parametrize("rotated", [True, False])
@pytest.mark.parametrize("hd,kv_heads,group,page", [(32, 1, 1, 16), (64, 4, 8, 16), (96, 2, 3, 48), (128, 8, 4, 64), (64, 3, 1, 256)])
@pytest.mark.parametrize("lens,news", [([1], None), ([5, 0, 33, 16, 17], None), ([40, 3, 7], [40, 1, 5]), ([100, 2, 64], [37, 0, 64])])
def test_append_is_the_definition_bit_for_bit(ctx, hd, kv_heads, group, page, lens, news, rotated):
    r = np.random.default_rng(hd + page + len(lens))
    cache, batch = make(ctx, r, lens, news, kv_heads, hd, page, extra_rows=2)
    heads = kv_heads * group
    q = r.standard_normal((batch.rows, heads * hd), dtype=np.float32)
    k, v = (r.standard_normal((batch.rows, kv_heads * hd), dtype=np.float32) for _ in "kv")
    cos, sin = tables(hd, 128) if rotated else (None, None)
    got = append(ctx, cache, batch, q, k, v, heads, cos, sin)
    want, raw = expect_append(cache, batch, q, k, v, heads, cos, sin)
    assert same_bits(got, want)  # rows of no sequence among it
    assert same_raw(cache.pools, cache.raw(), raw)  # slots of no new token among it


def test_append_of_values_at_the_edges_of_the_format(ctx):
    """Ties between codes and between magnitudes, zeros, values below and beyond
    the halves' range, infinities and NaN."""
    r = np.random.default_rng(3)
    hd, kv_heads, page = 64, 2, 16
    rows = 24
    x = r.standard_normal((rows, kv_heads * hd)).astype(np.float32)
    g = x.reshape(-1, 32)
    g[0] = 0
    g[1] = -0.0
    g[2, :] = 0
    g[2, 7] = 8.0  # scale -1: the others tie halfway between codes
    g[2, 8:20] = np.arange(12) - 5.5
    g[3, 4], g[3, 9] = 5.0, -5.0  # equal magnitudes: the first gives the sign
    g[4, 4], g[4, 9] = -5.0, 5.0
    g[5] *= 1e-7  # subnormal scales
    g[6] *= 1e-9  # scales of zero
    g[7] *= 1e6  # scales that are held to the largest half
    g[8] *= 1e30
    g[9, 3] = np.inf
    g[10, 31] = -np.inf
    g[11, 0] = np.nan
    g[12] = 3.0e38
    g[13] = 1e-45
    g[14] = np.linspace(-8, 8, 32)
    g[15] = np.linspace(8, -8, 32) * 0.3337
    g[16] = np.float32(65504 * 8) * np.linspace(-1, 1, 32)
    k, v = x.copy(), np.roll(x.reshape(-1, 32), 3, 0).reshape(x.shape).copy()
    cache, batch = make(ctx, r, [rows], [rows], kv_heads, hd, page)
    q = r.standard_normal((rows, kv_heads * hd)).astype(np.float32)
    got = append(ctx, cache, batch, q, k, v, kv_heads)
    want, raw = expect_append(cache, batch, q, k, v, kv_heads, None, None)
    assert same_bits(got, want) and same_raw(cache.pools, cache.raw(), raw)


def test_append_in_place_from_one_projection_equals_rope(ctx):
    """q, k and v as columns of one buffer, q rotated in place: glc_rope's bits."""
    r = np.random.default_rng(4)
    B, S, heads, kv_heads, hd = 3, 21, 8, 2, 64
    cache, batch = make(ctx, r, [S] * B, [S] * B, kv_heads, hd, 16)
    width = (heads + 2 * kv_heads) * hd
    x = r.standard_normal((B * S, width), dtype=np.float32)
    cos, sin = tables(hd, S)
    dx, dc, ds = ctx.from_numpy(x), ctx.from_numpy(cos), ctx.from_numpy(sin)
    a = dx.addr
    ctx.call("glc_kv_append", C.byref(cache.c), C.byref(batch.c), a, width, a, width, heads, a + 4 * heads * hd, width,
             a + 4 * (heads + kv_heads) * hd, width, dc.addr, ds.addr, S)
    q = ctx.from_numpy(np.ascontiguousarray(x[:, : heads * hd]))
    ctx.call("glc_rope", q.ptr, B * S, S, heads, hd, dc.ptr, ds.ptr, 0, 0)
    ctx.sync()
    got = dx.numpy()
    assert same_bits(np.ascontiguousarray(got[:, : heads * hd]), q.numpy())
    assert same_bits(np.ascontiguousarray(got[:, heads * hd:]), np.ascontiguousarray(x[:, heads * hd:]))
    _, raw = expect_append(cache, batch, np.ascontiguousarray(x[:, : heads * hd]), np.ascontiguousarray(x[:, heads * hd:(heads + kv_heads) * hd]),
                           np.ascontiguousarray(x[:, (heads + kv_heads) * hd:]), heads, cos, sin)
    assert same_raw(cache.pools, cache.raw(), raw)


def test_append_without_queries(ctx):
    r = np.random.default_rng(5)
    cache, batch = make(ctx, r, [9, 4], None, 2, 32, 16)
    k, v = (r.standard_normal((2, 64), dtype=np.float32) for _ in "kv")
    assert append(ctx, cache, batch, None, k, v, 0) is None
    _, raw = expect_append(cache, batch, np.zeros((2, 64), np.float32), k, v, 2, None, None)
    assert same_raw(cache.pools, cache.raw(), raw)


@pytest.mark.parametrize("hd,kv_heads,page", [(32, 1, 16), (64, 4, 16), (96, 3, 32), (128, 2, 80)])
def test_read_gives_the_stored_numbers(ctx, hd, kv_heads, page):
    r = np.random.default_rng(hd)
    lens = [50, 0, 1, 131]
    cache, _ = make(ctx, r, lens, None, kv_heads, hd, page)
    _, batch = make(ctx, np.random.default_rng(hd), lens, lens, kv_heads, hd, page, extra_rows=1)  # whole sequences
    w = kv_heads * hd
    for sides in ("kv", "k", "v"):
        out = {s: ctx.from_numpy(np.full((batch.rows, w + 4), CANARY)) for s in sides}
        a = lambda s: out[s].addr if s in out else 0  # noqa: E731
        ctx.call("glc_kv_read", C.byref(cache.c), C.byref(batch.c), a("k"), w + 4, a("v"), w + 4)
        ctx.sync()
        for i, s in enumerate("kv"):
            if s not in out:
                continue
            want = np.full((batch.rows, w + 4), CANARY)
            at = 0
            for b, n in enumerate(lens):
                if n:
                    want[at:at + n, :w] = cache.pools.sequence(i, batch.table[b], n).reshape(n, w)
                at += n
            assert same_bits(out[s].numpy(), want)


def test_bad_pages_and_positions_are_reported_and_nothing_else_is_touched(ctx):
    r = np.random.default_rng(6)
    cache, batch = make(ctx, r, [20, 20, 40], None, 2, 64, 16)
    q = r.standard_normal((3, 128), dtype=np.float32)
    k, v = (r.standard_normal((3, 128), dtype=np.float32) for _ in "kv")
    cos, sin = tables(64, 30)  # the third row's position is beyond the tables
    batch.table[1, 1] = cache.pools.pages
    batch.d[0].upload(batch.table)
    with pytest.raises(GlcError, match="out of range"):
        append(ctx, cache, batch, q, k, v, 2, cos, sin)
    # the first row alone is stored
    before = ref.Pools(cache.pools.pages, 16, 2, 64)
    before.raw = cache.pools.raw.copy()
    at = np.array([19])
    before.store(0, batch.table[0, 1], 3, *ref.quantize(ref.rotate(k[0].reshape(1, 2, 64), cos, sin, at)[0]))
    before.store(1, batch.table[0, 1], 3, *ref.quantize(v[0].reshape(2, 64)))
    assert same_raw(cache.pools, cache.raw(), before.raw)
    ctx.sync()  # reported once


# ------------------------------------------------------------------ attention


def attend(ctx, cache, batch, q, heads, pad=0, lse=True):
    hd = cache.pools.hd
    x = np.full((batch.rows, heads * hd + pad), np.nan, np.float32)
    x[:, : heads * hd] = q
    dq = ctx.from_numpy(x)
    o = ctx.from_numpy(np.full((batch.rows, heads * hd + pad), CANARY))
    dl = ctx.from_numpy(np.full((batch.rows, heads), CANARY))
    ctx.call("glc_attention_kv", C.byref(cache.c), C.byref(batch.c), dq.addr, x.shape[1], heads, o.addr, x.shape[1], dl.addr if lse else 0)
    ctx.sync()
    return o.numpy(), dl.numpy()


def check(cache, batch, q, heads, o, lse):
    """Per element, with s the sum of |q_i k_i| / sqrt(hd) of the largest key:
    a score is off by at most s (2^-22 from q's two halves, 2^-24 for each of the ~20
    roundings and cut-off sums of its products), ~2^-19.4 s; an exponential by that
    times itself and 2^-22 more; the probabilities' halves and their products with
    the scales add 2^-21, a tile's 8 cut-off sums 2^-21, and the at most 2^9 additions
    of tiles and parts, to nearest, 2^-24 each, of either sign, 2^-19.5; numerator and
    denominator both.  Hence 2 (2^-19.4 s + 2^-18.5), relative to the largest value
    (8 scales)."""
    p = cache.pools
    want, want_lse, s = ref.attend(p, batch.table, batch.lens, batch.starts, q, heads)
    none = np.isnan(want_lse).any(1)
    hd = p.hd
    assert (o[:, heads * hd:] == CANARY).all()
    o = o[:, : heads * hd]
    assert (o[none] == CANARY).all() and (lse[none] == CANARY).all()
    o, want, lse, want_lse, s = o[~none], want[~none], lse[~none], want_lse[~none], s[~none]
    tol = 2 * (2**-19.4 * s + 2**-18.5)
    big = float(np.abs(p.scales[1].astype(np.float64))[np.isfinite(p.scales[1])].max() * 8)
    err = np.abs(o - want).reshape(len(o), heads, hd).max(-1)
    assert (err <= tol * big).all(), (err / (tol * big)).max()
    empty = np.isneginf(want_lse)
    assert (o.reshape(len(o), heads, hd)[empty] == 0).all() and np.isneginf(lse[empty]).all()
    assert (np.abs(lse[~empty] - want_lse[~empty]) <= tol[~empty] + 2**-22 * np.abs(want_lse[~empty])).all()


@pytest.mark.parametrize("hd,kv_heads,group,page", [(32, 2, 8, 16), (64, 4, 8, 16), (96, 2, 3, 48), (128, 2, 4, 64), (64, 1, 1, 4096),
                                                   (128, 1, 7, 16), (64, 2, 20, 32), (32, 1, 16, 32), (96, 1, 12, 16)])
@pytest.mark.parametrize("lens", [[1], [0], [16, 31, 32, 33, 0, 1, 48], [511, 512, 513, 385, 700], [3000, 7]])
def test_attention_of_single_tokens(ctx, hd, kv_heads, group, page, lens):
    r = np.random.default_rng(hd + group + sum(lens))
    cache, batch = make(ctx, r, lens, None, kv_heads, hd, page)
    q = 2 * r.standard_normal((len(lens), kv_heads * group * hd), dtype=np.float32)
    check(cache, batch, q, kv_heads * group, *attend(ctx, cache, batch, q, kv_heads * group))


@pytest.mark.parametrize("hd,kv_heads,group,page", [(32, 2, 8, 16), (64, 2, 4, 16), (96, 1, 3, 48), (128, 2, 4, 64), (64, 2, 7, 32), (64, 1, 20, 16), (128, 1, 1, 16)])
@pytest.mark.parametrize("lens,news", [([5], [5]), ([70, 33, 5, 0], [3, 33, 0, 0]), ([100, 600, 40], [100, 9, 1]), ([300, 2], [77, 4])])
def test_attention_of_several_tokens(ctx, hd, kv_heads, group, page, lens, news):
    """Chunks of prompts, drafts, rows behind the last sequence, sequences with
    more new tokens than they have (their first rows see nothing)."""
    r = np.random.default_rng(hd + group + sum(lens))
    cache, batch = make(ctx, r, lens, news, kv_heads, hd, page, extra_rows=3)
    q = 2 * r.standard_normal((batch.rows, kv_heads * group * hd), dtype=np.float32)
    check(cache, batch, q, kv_heads * group, *attend(ctx, cache, batch, q, kv_heads * group, pad=8))


def test_attention_over_one_long_sequence(ctx):
    r = np.random.default_rng(8)
    cache, batch = make(ctx, r, [70001], None, 2, 64, 64)
    q = 2 * r.standard_normal((1, 8 * 64), dtype=np.float32)
    o, lse = attend(ctx, cache, batch, q, 8)
    check(cache, batch, q, 8, o, lse)
    for _ in range(3):  # the join of many CTAs is in one order
        o2, lse2 = attend(ctx, cache, batch, q, 8)
        assert same_bits(o, o2) and same_bits(lse, lse2)


def test_attention_of_many_sequences(ctx):
    """More sequences than a CTA has threads; most of them idle or short."""
    r = np.random.default_rng(9)
    lens = r.integers(0, 40, 1100)
    lens[::7] = 0
    lens[500] = 1500
    cache, batch = make(ctx, r, lens, None, 1, 32, 16)
    q = 2 * r.standard_normal((1100, 64), dtype=np.float32)
    check(cache, batch, q, 2, *attend(ctx, cache, batch, q, 2))


@pytest.mark.parametrize("q_size,k_size,v_size", [(1e-3, 1.0, 1e-6), (30.0, 0.03, 3e4), (1e4, 1e-4, 1.0), (1e-20, 1.0, 1.0), (0.0, 1.0, 1.0)])
def test_attention_over_the_range_of_scales(ctx, q_size, k_size, v_size):
    r = np.random.default_rng(10)
    cache, batch = make(ctx, r, [300, 77], None, 2, 64, 16, filled=False)
    p = cache.pools
    for side, size in enumerate((k_size, v_size)):
        p.codes[side] = r.integers(0, 256, p.codes[side].shape)
        grow = 2.0 ** r.integers(-4, 1, p.scales[side].shape)  # from key to key
        p.scales[side] = (r.choice([-1, 1], grow.shape) * grow * 0.26 * size).astype(np.float16)
    cache = Cache(ctx, p)
    q = (q_size * r.standard_normal((2, 8 * 64))).astype(np.float32)
    check(cache, batch, q, 8, *attend(ctx, cache, batch, q, 8))


def test_value_scales_that_grow_along_the_sequence(ctx):
    """The running size of the value scales is raised again and again, and once at the end."""
    r = np.random.default_rng(11)
    cache, batch = make(ctx, r, [2000], None, 1, 128, 16)
    p = cache.pools
    for i, page in enumerate(batch.table[0, : 2000 // 16]):
        p.scales[1, page] = np.float16(2.0 ** (-20 + 0.25 * i)) if i < 120 else np.float16(60000)
    cache = Cache(ctx, p)
    q = 2 * r.standard_normal((1, 4 * 128), dtype=np.float32)
    check(cache, batch, q, 4, *attend(ctx, cache, batch, q, 4))


@pytest.mark.parametrize("kv_heads,group,hd", [(2, 2, 64), (1, 1, 32), (2, 8, 128), (1, 20, 64), (1, 1, 96)])
@pytest.mark.parametrize("news", [[9, 1], [3, 2]])
def test_what_a_row_does_not_see_does_not_count(ctx, kv_heads, group, hd, news):
    """NaN and infinite scales behind the end of a sequence, in unused pages, and
    in tokens that only later rows see; a visible NaN reaches the rows that see it."""
    r = np.random.default_rng(12)
    heads, rows = kv_heads * group, sum(news)
    cache, batch = make(ctx, r, [40, 21], news, kv_heads, hd, 16)
    q = 2 * r.standard_normal((rows, heads * hd), dtype=np.float32)
    clean, clean_lse = attend(ctx, cache, batch, q, heads)
    check(cache, batch, q, heads, clean, clean_lse)
    p = cache.pools
    used = np.zeros((p.pages, 16), bool)
    for b, n in enumerate(batch.lens):
        for pos in range(n):
            used[batch.table[b, pos // 16], pos % 16] = True
    for side in (0, 1):
        s = p.scales[side].transpose(0, 2, 1, 3)
        s[~used] = np.array([np.nan, np.inf, -np.inf, np.nan], np.float16)[r.integers(0, 4, s[~used].shape)]
        p.scales[side] = s.transpose(0, 2, 1, 3)
    o, lse = attend(ctx, Cache(ctx, p), batch, q, heads)
    assert same_bits(o, clean) and same_bits(lse, clean_lse)
    # the first sequence's last-but-one token: of its new rows the last two see it
    at = 38
    sees = np.array([b == 0 and pos >= at for b, pos in batch.positions()])
    assert sees.sum() == 2
    for side in (0, 1):
        keep = p.raw.copy()
        p.scales[side, batch.table[0, at // 16], :, at % 16] = np.nan
        o, lse = attend(ctx, Cache(ctx, p), batch, q, heads)
        p.raw = keep
        assert np.isnan(o[sees]).all()
        assert np.isfinite(o[~sees]).all()
        np.testing.assert_allclose(o[~sees], clean[~sees], rtol=0, atol=2**-13)
        if side == 0:
            assert same_bits(np.ascontiguousarray(lse[~sees]), np.ascontiguousarray(clean_lse[~sees]))


def test_long_rows_do_not_drift(ctx):
    """Many keys for each warp: sums of hundreds of tiles stay within 2^-19 of the mean square."""
    r = np.random.default_rng(16)
    n, B = 16000, 40
    cache, batch = make(ctx, r, [n], None, 1, 32, 64)
    batch = Batch(ctx, np.repeat(batch.table, B, 0), [n] * B)
    q = np.repeat(2 * r.standard_normal((1, 8 * 32), dtype=np.float32), B, 0)
    o, lse = attend(ctx, cache, batch, q, 8)
    want, want_lse, _ = ref.attend(cache.pools, batch.table[:1], [n], None, q[:1], 8)
    for row in range(B):
        assert np.linalg.norm(o[row] - want[0]) <= 2**-19 * np.linalg.norm(want[0])
        assert np.abs(lse[row] - want_lse[0]).max() <= 2**-19


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
def test_a_bad_query_spoils_its_own_row_alone(ctx, bad):
    r = np.random.default_rng(17)
    for heads, news in ((8, None), (2, None), (8, [5, 1])):
        cache, batch = make(ctx, r, [90, 33], news, 2, 64, 16)
        q = 2 * r.standard_normal((batch.rows, heads * 64), dtype=np.float32)
        clean, clean_lse = attend(ctx, cache, batch, q, heads)
        q[0, 64 + 5] = bad
        o, lse = attend(ctx, cache, batch, q, heads)
        keep = np.ones_like(o, bool)
        keep[0, 64:128] = False
        assert same_bits(o[keep], clean[keep])
        if not bad == 3e38:  # (a score beyond fp32's range, or not)
            assert np.isnan(o[0, 64:128]).all()
        if np.isnan(bad):  # every score is NaN, and so is the sum
            assert np.isnan(lse[0, 1]) and np.isfinite(np.delete(lse.ravel(), 1)).all()


def test_attention_reports_bad_tables_and_goes_on(ctx):
    r = np.random.default_rng(13)
    cache, batch = make(ctx, r, [100, 50], None, 2, 64, 16)
    q = 2 * r.standard_normal((2, 4 * 64), dtype=np.float32)
    clean, _ = attend(ctx, cache, batch, q, 4)
    good = batch.table.copy()
    for bad in (-1, cache.pools.pages, 2**31 - 1):
        batch.table[:] = good
        batch.table[0, 3] = bad
        batch.d[0].upload(batch.table)
        with pytest.raises(GlcError, match="out of range"):
            attend(ctx, cache, batch, q, 4)
    batch.d[0].upload(good)
    for lens in ([2**31 - 1, 50], [-3, 50]):
        batch.d[1].upload(np.array(lens, np.int32))
        with pytest.raises(GlcError, match="out of range"):
            attend(ctx, cache, batch, q, 4)
    batch.d[1].upload(np.array([100, 50], np.int32))
    o, _ = attend(ctx, cache, batch, q, 4)
    assert same_bits(o, clean)


@pytest.mark.parametrize("seqs", [3, 40])
def test_starts_that_do_not_ascend_end_the_attention(ctx, seqs):
    """Reported, and no row is written; the next call is whole."""
    r = np.random.default_rng(18)
    lens, news = [20 + i for i in range(seqs)], [2] * seqs
    cache, batch = make(ctx, r, lens, news, 2, 64, 16)
    heads = 4
    q = 2 * r.standard_normal((batch.rows, heads * 64), dtype=np.float32)
    clean, _ = attend(ctx, cache, batch, q, heads)
    good = np.array(batch.starts, np.int32)
    for at, value in ((1, 5), (seqs, 1), (0, -1), (seqs, 2 * seqs + 1)):
        bad = good.copy()
        bad[at] = value
        batch.d[2].upload(bad)
        dq, o = ctx.from_numpy(q), ctx.from_numpy(np.full(q.shape, CANARY))
        ctx.call("glc_attention_kv", C.byref(cache.c), C.byref(batch.c), dq.addr, q.shape[1], heads, o.addr, q.shape[1], 0)
        with pytest.raises(GlcError, match="out of range"):
            ctx.sync()
        assert (o.numpy() == CANARY).all(), (at, value)
    batch.d[2].upload(good)
    o, _ = attend(ctx, cache, batch, q, heads)
    assert same_bits(o, clean)


def test_attention_in_place_and_on_cut_items(ctx):
    """o in the place of q, for an item that many CTAs share."""
    r = np.random.default_rng(19)
    for lens, heads in (([9000], 8), ([300, 20, 0], 4)):
        cache, batch = make(ctx, r, lens, None, 1, 64, 64)
        q = 2 * r.standard_normal((batch.rows, heads * 64), dtype=np.float32)
        clean, _ = attend(ctx, cache, batch, q, heads)
        d = ctx.from_numpy(q)
        ctx.call("glc_attention_kv", C.byref(cache.c), C.byref(batch.c), d.addr, q.shape[1], heads, d.addr, q.shape[1], 0)
        ctx.sync()
        assert same_bits(d.numpy(), clean)


def test_pools_beyond_32_bits(ctx):
    """Pages whose byte and code offsets pass 2^32, through append, read and attention."""
    heads, hd, page = 8, 128, 64
    chunk = page * hd * 9 // 16
    pages = (5 << 30) // (heads * chunk)
    r = np.random.default_rng(14)
    k, v = ctx.empty((pages * heads * chunk,), np.uint8), ctx.empty((pages * heads * chunk,), np.uint8)
    c = KVCacheC(k=k.addr, v=v.addr, num_pages=pages, page_size=page, num_kv_heads=heads, head_dim=hd)
    n = 150
    used = np.array([[pages - 1, pages - 7, pages - 3]], np.int32)
    batch = Batch(ctx, used, [n], [0, n])
    x = [r.standard_normal((n, heads * hd), dtype=np.float32) for _ in range(3)]
    d = [ctx.from_numpy(y) for y in x]
    out = ctx.empty((n, heads * hd))
    ctx.call("glc_kv_append", C.byref(c), C.byref(batch.c), d[0].addr, heads * hd, out.addr, heads * hd, heads, d[1].addr, heads * hd,
             d[2].addr, heads * hd, 0, 0, 0)
    back = [ctx.empty((n, heads * hd)) for _ in "kv"]
    ctx.call("glc_kv_read", C.byref(c), C.byref(batch.c), back[0].addr, heads * hd, back[1].addr, heads * hd)
    ctx.call("glc_attention_kv", C.byref(c), C.byref(batch.c), d[0].addr, heads * hd, heads, out.addr, heads * hd, 0)
    ctx.sync()
    small = ref.Pools(3, page, heads, hd)
    for side in (0, 1):
        codes, scales = ref.quantize(x[1 + side].reshape(n, heads, hd))
        for t in range(n):
            small.store(side, t // page, t % page, codes[t], scales[t])
        assert same_bits(back[side].numpy(), ref.numbers(codes, scales).reshape(n, -1))
    rows = [0, 1, 77, 149]
    for t in rows:
        want, _, _ = ref.attend(small, np.array([[0, 1, 2]]), [t + 1], None, x[0][t:t + 1], heads)
        assert np.abs(out.numpy()[t] - want[0]).max() < 1e-4


def test_two_contexts_and_a_grown_workspace(ctx):
    """A second context on the device runs beside the first; the workspace of one
    grows between calls; results are those of a quiet device, bit for bit."""
    from gollama_b200.device import Context

    r = np.random.default_rng(15)
    cache, batch = make(ctx, r, [900, 1200, 60], None, 2, 128, 16)
    q = 2 * r.standard_normal((3, 8 * 128), dtype=np.float32)
    want, want_lse = attend(ctx, cache, batch, q, 8)
    with Context(ctx.device) as two:
        c2, b2 = Cache(two, cache.pools), Batch(two, batch.table, batch.lens)
        q1, q2 = ctx.from_numpy(q), two.from_numpy(q)
        o1, o2 = [ctx.empty(q.shape) for _ in range(20)], [two.empty(q.shape) for _ in range(20)]
        for i in range(20):
            ctx.call("glc_attention_kv", C.byref(cache.c), C.byref(batch.c), q1.addr, q.shape[1], 8, o1[i].addr, q.shape[1], 0)
            two.call("glc_attention_kv", C.byref(c2.c), C.byref(b2.c), q2.addr, q.shape[1], 8, o2[i].addr, q.shape[1], 0)
        ctx.sync()
        two.sync()
        assert all(same_bits(o.numpy(), want) for o in o1 + o2)
        del q2, o2, c2, b2
    g = ctx.zeros((1 << 20,))
    segs = np.array([[0, 1 << 20]], np.int64)
    norm, scale = ctx.empty((1,), np.float64), ctx.empty((1,))
    ctx.call("glc_grad_clip_norm", g.ptr, segs.ctypes.data_as(C.c_void_p), 1, C.c_float(1.0), norm.ptr, scale.ptr)  # uses the workspace
    o, lse = attend(ctx, cache, batch, q, 8)
    assert same_bits(o, want) and same_bits(lse, want_lse)
    try:
        ctx.call("glc_set_pdl", 0)
        o, lse = attend(ctx, cache, batch, q, 8)
        assert same_bits(o, want) and same_bits(lse, want_lse)
    finally:
        ctx.call("glc_set_pdl", 1)


# ------------------------------------------------------------------ sampling


def sample(ctx, x, t, k=None, p=None, m=None, u=None, ld=None, shift=0):
    R, V = x.shape
    ld = ld or V
    buf = np.full(R * ld + shift, np.nan, np.float32)  # what lies between rows is not read as a logit
    for i in range(R):
        buf[shift + i * ld:shift + i * ld + V] = x[i]
    d = [ctx.from_numpy(buf)] + [None if a is None else ctx.from_numpy(np.broadcast_to(np.asarray(a, ty), (R,)).copy())
                                 for a, ty in ((t, np.float32), (k, np.int32), (p, np.float32), (m, np.float32), (u, np.float32))]
    tok, logp = ctx.from_numpy(np.full(R, -99, np.int64)), ctx.empty((R,))
    a = [0 if y is None else y.addr for y in d]
    ctx.call("glc_sample", a[0] + 4 * shift, ld, R, V, *a[1:], tok.addr, logp.addr)
    ctx.sync()
    return tok.numpy(), logp.numpy()


def check_sample(x, t, k, p, m, u, tok, logp):
    """A weight is off by at most 1.5 2^-31 of the largest (half a unit each for the
    table's entry, the correction and the shift) plus 2^-40 of itself; of V tokens
    those errors, of either sign, add up as their square root, 4 of which are taken,
    and one unit for a sum of few.  A token whose interval has u within that share of
    it is right; a token whose weight or running sum is that near to a cut may be in
    or out.  logp is that in fp32."""
    tol = 4 * np.sqrt(x.shape[1] / 3) * 1.5 * 2.0**-31 + 2.0**-31
    R, V = x.shape
    b = lambda a, none: np.broadcast_to(np.asarray(none if a is None else a, np.float64), (R,))  # noqa: E731
    f = lambda a, none: b(a, none).astype(np.float32).astype(np.float64)  # noqa: E731  (the settings are fp32)
    t, k, p, m = f(t, 1.0), b(k, 0), f(p, 1.0), f(m, 0.0)
    for i in range(R):
        ok = False
        # the settings themselves, then with the cuts moved by the tolerance
        for pp, mm in ((p[i], m[i]), (p[i] * (1 + tol), m[i]), (p[i] * (1 - tol), m[i]), (p[i], m[i] * (1 + tol)), (p[i], m[i] * (1 - tol))):
            if pp >= 1 > p[i] or (mm >= 1) != (m[i] >= 1):
                continue
            ids, w = ref.kept_tokens(x[i], np.float32(t[i]), int(k[i]), pp, mm)
            if len(ids) == 0:
                assert tok[i] == -1 and np.isneginf(logp[i])
                ok = True
                break
            at = np.searchsorted(ids, tok[i])
            if at == len(ids) or ids[at] != tok[i]:
                continue
            upto, goal = np.cumsum(w) / w.sum(), min(max(float(u[i]), 0.0), 1.0)
            low, high = upto[at] - w[at] / w.sum(), upto[at]
            close = abs(logp[i] - np.log(w[at] / w.sum())) <= 2 * tol + 2**-23 * abs(logp[i])
            if close and low - tol <= goal <= high + tol:
                ok = True
                break
        assert ok, (i, tok[i])


SETTINGS = [(1.0, None, None, None), (0.7, 40, None, None), (1.0, None, 0.9, None), (1.0, None, None, 0.05), (0.8, 50, 0.95, 0.02),
            (1.5, 1000, 0.99, None), (0.0, 5, 0.5, None), (1.0, 1, None, None), (0.3, None, 0.5, 0.1), (2.5, 600, None, None), (1.0, None, 1e-9, None)]


@pytest.mark.parametrize("t,k,p,m", SETTINGS)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (2, 1000), (300, 513), (40, 4099), (7, 32000), (3, 50257), (2, 131075), (160, 9001)])
def test_sample_is_the_definition(ctx, rows, vocab, t, k, p, m):
    r = np.random.default_rng(rows * 7 + vocab)
    x = (2.5 * r.standard_normal((rows, vocab))).astype(np.float32)
    u = r.random(rows, dtype=np.float32)
    check_sample(x, t, k, p, m, u, *sample(ctx, x, t, k, p, m, u))


def test_sample_with_settings_of_each_row_and_rows_apart(ctx):
    r = np.random.default_rng(21)
    R, V = 64, 5003
    x = (3 * r.standard_normal((R, V))).astype(np.float32)
    t = r.choice([0.0, -1.0, np.nan, 0.5, 1.0, 3.0], R)
    k = r.choice([-1, 0, 1, 2, 40, 511, 512, 513, 5003, 9999], R)
    p = r.choice([-0.5, 0.0, 0.3, 0.9, 1.0, 2.0], R)
    m = r.choice([-1.0, 0.0, 0.01, 0.5, 1.0, 7.0], R)
    u = r.random(R, dtype=np.float32)
    for ld, shift in ((V, 0), (V + 1, 0), (V + 5, 1), (V + 1, 3)):
        check_sample(x, t, k, p, m, u, *sample(ctx, x, t, k, p, m, u, ld, shift))


@pytest.mark.parametrize("t,k,p,m", SETTINGS + [(1.0, 700, 0.5, None), (1.0, 2000, None, 0.5)])
def test_sample_of_equal_and_few_distinct_logits(ctx, t, k, p, m):
    """Thousands of equals at a cut: the lower indexes are kept."""
    r = np.random.default_rng(22)
    x = np.stack([np.zeros(6001), r.integers(0, 3, 6001), np.where(np.arange(6001) % 2, -0.0, 0.0), np.repeat([1.0, -3.0], [5000, 1001]),
                  np.float32(1) + np.arange(6001) * np.float32(2**-23), np.where(np.arange(6001) == 4000, 30, r.integers(0, 2, 6001))]).astype(np.float32)
    for u in (0.0, 0.37, 0.999999):
        uu = np.full(len(x), u, np.float32)
        check_sample(x, t, k, p, m, uu, *sample(ctx, x, t, k, p, m, uu))


@pytest.mark.parametrize("t,k,p,m", SETTINGS)
def test_sample_of_masked_and_infinite_logits(ctx, t, k, p, m):
    r = np.random.default_rng(23)
    V = 3001
    x = (2 * r.standard_normal((9, V))).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, :] = -np.inf
    x[2, 1234] = -5
    x[3, r.random(V) < 0.99] = -np.inf
    x[4, r.random(V) < 0.5] = np.nan
    x[5, [7, 77, 2999]] = np.inf
    x[6, ::2] = np.finfo(np.float32).min
    x[7] = np.finfo(np.float32).min
    x[8, :1500] = np.finfo(np.float32).max
    u = r.random(9, dtype=np.float32)
    check_sample(x, t, k, p, m, u, *sample(ctx, x, t, k, p, m, u))


def test_sample_at_the_ends_of_the_random_number(ctx):
    r = np.random.default_rng(24)
    x = (2 * r.standard_normal((6, 2000))).astype(np.float32)
    u = np.array([0.0, 1.0, np.nextafter(np.float32(1), np.float32(0)), -1.0, np.nan, 2.0], np.float32)
    tok, _ = sample(ctx, x, 1.0, None, None, None, u)
    # the first token of all, or the last with any weight
    assert tok[0] == 0 and tok[3] == 0 and tok[4] == 0
    assert all(tok[i] >= 1990 for i in (1, 2, 5))


@pytest.mark.parametrize("t", [1e-45, 1e-30, 1e30, np.inf])
def test_sample_at_the_ends_of_the_temperature(ctx, t):
    """Next to none: the largest's equals share all; without bound: all are equal."""
    r = np.random.default_rng(27)
    x = (2 * r.standard_normal((4, 2000))).astype(np.float32)
    x[1, [5, 9]] = x[1].max()
    if t < 1e38:  # (infinity over infinity has no value)
        x[2, 7] = np.inf
    x[3, ::2] = -np.inf
    u = np.array([0.5, 0.75, 0.5, 0.25], np.float32)
    check_sample(x, t, None, None, None, u, *sample(ctx, x, t, None, None, None, u))


@pytest.mark.parametrize("rows,vocab", [(1, 131072), (2, 262145), (1, 344064)])
def test_sample_of_the_largest_vocabularies(ctx, rows, vocab):
    r = np.random.default_rng(vocab)
    x = (2.5 * r.standard_normal((rows, vocab))).astype(np.float32)
    u = r.random(rows, dtype=np.float32)
    for t, k, p, m in SETTINGS[1:5] + [(3.0, None, 0.99, None), (20.0, 100000, 0.7, None)]:
        check_sample(x, t, k, p, m, u, *sample(ctx, x, t, k, p, m, u))


def test_sample_follows_its_distribution(ctx):
    """The shares of 40000 draws: each within 6 standard deviations of its probability."""
    r = np.random.default_rng(25)
    n, V = 40000, 50
    x = np.broadcast_to((1.5 * r.standard_normal(V)).astype(np.float32), (n, V))
    tok, _ = sample(ctx, np.ascontiguousarray(x), 0.9, 12, 0.95, 0.0, r.random(n, dtype=np.float32))
    ids, w = ref.kept_tokens(x[0], np.float32(0.9), 12, np.float32(0.95), 0.0)
    assert set(tok) <= set(ids)
    pr = w / w.sum()
    got = np.array([(tok == i).mean() for i in ids])
    assert (np.abs(got - pr) <= 6 * np.sqrt(pr * (1 - pr) / n)).all()


def test_sample_is_the_same_each_time(ctx):
    r = np.random.default_rng(26)
    x = (2.5 * r.standard_normal((33, 32000))).astype(np.float32)
    u = r.random(33, dtype=np.float32)
    a = sample(ctx, x, 1.2, None, 0.97, None, u)
    for _ in range(3):
        b = sample(ctx, x, 1.2, None, 0.97, None, u)
        assert np.array_equal(a[0], b[0]) and same_bits(a[1], b[1])
