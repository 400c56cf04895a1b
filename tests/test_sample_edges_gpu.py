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
