"""Sampling at the ends of its settings' ranges, against the definition in 64 bits."""
import numpy as np
import pytest

from tests.test_generation_gpu import check_sample, sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("p", [1e-45, 1e-38, 1e-30, 1e-20, 5.4e-20, 5.5e-20, 1e-12])
@pytest.mark.parametrize("k", [None, 5, 40, 700])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 31), (5, 4099), (2, 32000), (2, 131075)])
def test_the_smallest_nucleus_is_the_first_token(ctx, p, k, rows, vocab):
    r = np.random.default_rng(vocab + rows)
    x = (2.5 * r.standard_normal((rows, vocab))).astype(np.float32)
    x[0, vocab // 2:] = x[0].max()  # equals: the lowest index
    for t in (0.3, 1.0, 40.0):
        u = r.random(rows, dtype=np.float32)
        tok, logp = sample(ctx, x, t, k, p, None, u)
        assert np.array_equal(tok, x.argmax(1)) and (logp == 0).all()
        check_sample(x, t, k, p, None, u, tok, logp)


@pytest.mark.parametrize("t,size", [(1e-45, 1e-42), (1e-42, 1e-39), (2e-39, 3e-38), (1e-40, 1e-44), (3e-39, 1e-38), (1e-38, 1e-30)])
@pytest.mark.parametrize("k,p,m", [(None, None, None), (None, 0.9, None), (40, 0.9, None), (700, None, 0.01), (None, 0.999, 0.05)])
@pytest.mark.parametrize("rows,vocab", [(3, 1000), (2, 32000)])
def test_temperatures_whose_inverse_no_float_holds(ctx, rows, vocab, k, p, m, t, size):
    r = np.random.default_rng(vocab)
    x = (size * r.standard_normal((rows, vocab))).astype(np.float32)
    u = r.random(rows, dtype=np.float32)
    check_sample(x, t, k, p, m, u, *sample(ctx, x, t, k, p, m, u))


FLAT = [(131075, 20.0), (131075, 22.0), (131075, 22.2), (344064, 22.0), (344064, 25.0), (131075, 28.0), (5000, 14.0), (131075, 9.0)]


@pytest.mark.parametrize("vocab,below", FLAT)
@pytest.mark.parametrize("first", [0, 777])
def test_a_flat_tail_has_its_share(ctx, vocab, below, first):
    """One token over equal ones: the errors of their weights add up, to a unit (2^-45) and 2^-27 of itself for each
    and no more.  Draws over the whole row and cuts within the tail."""
    w = np.exp(-np.float64(np.float32(below)))
    tail, n = (vocab - 1) * w, vocab - 1
    tol = vocab * 2.0**-45 + tail * 2.0**-26.7  # of the sum
    x = np.full((1, vocab), -below, np.float32)
    x[0, first] = 0
    one = np.nextafter(np.float32(1), np.float32(0))
    # the draw: the head's interval begins behind `first` tail tokens
    for u in (0.0, 0.5, float(np.float32(1 - tail / 2)), float(np.float32(1 - tail / 50)), float(one)):
        tok, logp = sample(ctx, x, 1.0, None, None, None, np.float32(u))
        goal = max(float(np.float32(u)), 0.0) * (1 + tail)  # (a negative number draws as 0)
        low, high = (tok[0] * w if tok[0] <= first else 1 + (tok[0] - 1) * w), (1 + tok[0] * w if tok[0] >= first else (tok[0] + 1) * w)
        assert low - 2 * tol <= goal <= high + 2 * tol, (tok[0], low, goal, high)
        want = (0.0 if tok[0] == first else -np.float64(np.float32(below))) - np.log1p(tail)
        assert abs(logp[0] - want) <= 2 * tol + 2.0**-23 * abs(want)
    # top-p that cuts the tail: the last kept token is drawn last
    for share in (0.25, 0.75):
        p = np.float32((1 + share * tail) / (1 + tail))
        kept = np.ceil((np.float64(p) * (1 + tail) - 1) / w)
        if not 1 <= kept <= n or p >= 1:
            continue
        tok, logp = sample(ctx, x, 1.0, None, p, None, one)
        assert tok[0] != first or kept * w < 2.0**-24 + 2 * tol  # (u is 2^-24 short of the sum's end)
        most, least = kept + 2 * tol / w + 1, kept - 2 * tol / w - 1 - 2.0**-24 * (1 + tail) / w
        assert least - 1 <= tok[0] <= most, (tok[0], kept)
        assert abs(logp[0] - ((0.0 if tok[0] == first else -np.float64(np.float32(below))) - np.log1p(kept * w))) <= 4 * tol + w + 2.0**-23 * below


@pytest.mark.parametrize("k", [None, 100000])
def test_a_tail_of_few_values_is_the_definition(ctx, k):
    """Logits of few bits: thousands of equals in every step of the tail, cut by top-p at several places."""
    r = np.random.default_rng(41)
    V = 131075
    x = (np.round(r.standard_normal((6, V)) * 2) / 4 - 18).astype(np.float32)
    x[:, 5000] = 0.0
    x[1, 5001:5004] = -1.0
    x[2] -= 3
    x[3] += 6
    u = r.random(6, dtype=np.float32)
    u[4:] = np.nextafter(np.float32(1), np.float32(0))
    for p in (None, 0.9, 0.9995, 0.99999, 0.9999999):
        check_sample(x, 1.0, k, p, None, u, *sample(ctx, x, 1.0, k, p, None, u))
