"""Attention where one key has nearly all of the weight and a small value, as the first
token of a sequence often has: what the other keys add is then most of the result."""
import numpy as np
import pytest

from tests import generation_ref as ref
from tests.test_generation_gpu import Cache, attend, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weight", [0.94, 0.99, 0.999])
@pytest.mark.parametrize("small", [2.0**-10, 2.0**-7, 2.0**-4])
@pytest.mark.parametrize("hd,group,news,length", [
    (64, 4, None, 32), (64, 8, None, 32), (128, 4, None, 33), (128, 8, None, 300), (64, 4, None, 4000), (32, 8, [5], 200),
    (96, 4, [5], 100), (128, 2, [40], 64)])
def test_keys_beside_a_sink_keep_their_bits(ctx, hd, group, news, length, small, weight):
    """Relative to the exact result, with scores that the products give exactly (small whole numbers and powers of
    two) and of 24 powers of two at most: those are off by 2^-24 of themselves for each of the two roundings of their
    scale, ln2 24 2^-23 = 2^-18.9 in what they weigh; an exponential by 2^-22; a probability in two halves, its product
    with the scale and a tile's cut-off sums by 2^-22 each.  2^-18 in all."""
    r = np.random.default_rng(length + hd)
    rows = 1 if news is None else news[0]
    cache, batch = make(ctx, r, [length], news, 1, hd, 16)
    p = cache.pools
    table = batch.table[0]
    # keys: scale 1/4, codes -1, 0 or 1; the first one's lie along the queries
    codes = r.integers(-1, 2, (length, 1, hd))
    sign = r.choice([-1, 1], hd)
    codes[0, 0] = 2 * sign
    # its score is 2 hd / 4 |q| / sqrt(hd) = |q| sqrt(hd) / 2, beside scores of about |q| sqrt(hd) / 5 / sqrt(hd)
    want = np.log(weight / (1 - weight) * (length - 1))
    size = np.float32(2.0 ** -6 * np.round(64 * want * 2 / np.sqrt(hd)))
    values = r.integers(-8, 8, (2, length, 1, hd))
    for t in range(length):
        page, slot = table[t // 16], t % 16
        p.store(0, page, slot, (codes[t] + 8).astype(np.uint8), np.full((1, hd // 32), 0.25, np.float16))
        p.store(1, page, slot, (values[0, t] + 8).astype(np.uint8), np.full((1, hd // 32), 0.25 if t else 0.25 * small, np.float16))
    cache = Cache(ctx, p)
    q = np.tile((size * sign).astype(np.float32), (rows, group)) * np.repeat(1 - np.arange(group) / 64, hd).astype(np.float32)
    o, _ = attend(ctx, cache, batch, q, group)
    exact, lse, _ = ref.attend(p, batch.table, batch.lens, batch.starts, q, group)
    assert np.abs(lse).max() < 24 * np.log(2)
    o, exact = o.reshape(-1, hd), exact.reshape(-1, hd)
    seen = np.repeat(np.arange(length - rows + 1, length + 1), group) > 1
    err = np.linalg.norm(o - exact, axis=1) / np.linalg.norm(exact, axis=1)
    print(err[seen].max())
    assert (err[seen] <= 2.0**-18).all(), err[seen].max()


@pytest.mark.parametrize("large", [60000.0, 900.0, np.inf, np.nan])
@pytest.mark.parametrize("size", [0.26, 0.01, 1e-3])
@pytest.mark.parametrize("group,hd,new", [(2, 64, 2), (8, 128, 3), (4, 32, 6)])
def test_a_large_value_that_a_row_does_not_see_costs_it_no_bits(ctx, group, hd, new, size, large):
    """Infinite ones cost nothing.  A finite one of 2^e: a probability times a scale is held in two halves at 2^(12 - e)
    times its size where e > 0, each rounded by 2^-25 at most, so it is off by 2^(e - 36), and by 2^-36 large / scale
    of itself, where the scales are 0.57 of `size` at least; and scales go to 2^-6 of themselves where e > 6, those below 2^-8 then
    to 2^-25, which is 2^-8 of 1e-3's smallest.  Rows have the usual errors (above, 2^-18) beside that."""
    r = np.random.default_rng(71)
    cache, batch = make(ctx, r, [70], [new], 1, hd, 16)
    p = cache.pools
    p.scales[1] = (p.scales[1].astype(np.float32) / 0.26 * size).astype(np.float16)
    p.scales[0] = (p.scales[0].astype(np.float32) / 8).astype(np.float16)
    q = r.standard_normal((new, group * hd), dtype=np.float32)
    exact, _, _ = ref.attend(p, batch.table, batch.lens, batch.starts, q, group)
    p.scales[1, batch.table[0, 69 // 16], :, 69 % 16] = np.float16(large)  # the last token's
    o, _ = attend(ctx, Cache(ctx, p), batch, q, group)
    err = [np.linalg.norm(o[t] - exact[t]) / np.linalg.norm(exact[t]) for t in range(new - 1)]
    tol = 2.0**-18
    if np.isfinite(large):
        tol += 2.0**-36 * large / (0.57 * size) + (2.0**-8 if size == 1e-3 and large > 2**6 else 0.0)
    assert max(err) <= tol, (max(err), tol)
