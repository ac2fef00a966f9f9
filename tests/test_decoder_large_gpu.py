"""A decoder's operators on operands of more than 2^31 elements: what lies behind that is found where it should be."""
import gc

import numpy as np
import pytest

from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
BIG = 2 ** 31


@pytest.fixture(autouse=True)
def room(thc):
    yield
    gc.collect()


def _halves(rng, *size):
    return rng.standard_normal(size).astype(np.float16)


@pytest.mark.parametrize("dim", [100, 4099, 50001])
def test_norms(thc, dim):
    rng = np.random.default_rng(dim)
    rows = BIG // dim + 60
    ends, g = _halves(rng, 40, dim), _halves(rng, 40, dim)
    t = thc.Tensor.from_numpy
    w, b = t(_halves(rng, dim)), t(_halves(rng, dim))
    x = thc.Tensor("half").resize((rows, dim)).fill(2)
    x.narrow(0, rows - 40, 40).copy(t(ends))
    y = thc.Tensor("half").layer_norm(x, w, b)
    want = thc.Tensor("half").layer_norm(t(ends), w, b).numpy()
    assert_bit_equal(y.narrow(0, rows - 40, 40).numpy(), want)
    assert_bit_equal(y.narrow(0, rows - 45, 3).numpy(), np.repeat(b.numpy()[None], 3, 0))      # rows of one value
    # the gradient: rows before the last ones add nothing, as theirs is zero
    grad = y.zero()
    grad.narrow(0, rows - 40, 40).copy(t(g))
    dw, db, dw0, db0 = (thc.Tensor("half") for _ in range(4))
    grad.layer_norm_grad(dw, db, x, grad, w)
    few = thc.Tensor("half").layer_norm_grad(dw0, db0, t(ends), t(g), w)
    assert_bit_equal(grad.narrow(0, rows - 40, 40).numpy(), few.numpy())
    assert np.all(grad.narrow(0, rows - 60, 20).numpy() == 0)
    for a, c in ((dw, dw0), (db, db0)):      # the same 40 floats in another order, rounded to half
        a, c = a.numpy().astype(np.float64), c.numpy().astype(np.float64)
        assert np.all(np.abs(a - c) <= 2.0 ** -10 * np.abs(c) + 2.0 ** -24 * 40 * 400)


def test_rotary(thc):
    rng = np.random.default_rng(1)
    heads, dim = 6, 70
    tokens = BIG // (heads * dim) + 90
    ends = _halves(rng, 50, heads, dim)
    t = thc.Tensor.from_numpy
    x = thc.Tensor("half").resize((tokens, heads, dim)).zero()
    x.narrow(0, tokens - 50, 50).copy(t(ends))
    f = thc.Tensor("double").rotary_frequencies(dim)
    at = thc.Tensor("long").resize((tokens,)).fill(3)
    places = rng.integers(0, 1 << 20, 50)
    at.narrow(0, tokens - 50, 50).copy(t(places))
    want = thc.Tensor("half").rotary(t(ends), t(places), f).numpy()
    y = thc.Tensor("half").rotary(x, at, f)
    assert_bit_equal(y.narrow(0, tokens - 50, 50).numpy(), want)
    assert np.all(y.narrow(0, tokens - 60, 10).numpy() == 0)
    x.rotary(x, at, f)
    assert_bit_equal(x.narrow(0, tokens - 50, 50).numpy(), want)
    # heads far apart in memory: strides beyond 2^31
    far = y.view_as_strided(0, (2, 1, dim), (heads * dim * (tokens - 1), dim, 1))
    far.select(0, 1).copy(t(ends[:1, 0]))
    got = thc.Tensor("half").rotary(far, t(places[:2]), f)
    assert_bit_equal(got.select(0, 1).numpy(), thc.Tensor("half").rotary(t(ends[:1, :1]), t(places[1:2]), f).select(0, 0).numpy())


@pytest.mark.parametrize("rows,cols", [(60, 100), (150, 140), (90, 300)])
def test_many_matrices(thc, rows, cols):
    rng = np.random.default_rng(rows)
    count = BIG // (rows * cols) + 50
    ends = _halves(rng, 5, rows, cols)
    t = thc.Tensor.from_numpy
    x = thc.Tensor("half").resize((count, rows, cols)).fill(1)
    x.narrow(0, count - 5, 5).copy(t(ends))
    x.orthogonalize(x)
    assert_bit_equal(x.narrow(0, count - 5, 5).numpy(), thc.Tensor("half").orthogonalize(t(ends)).numpy())
    one = thc.Tensor("half").orthogonalize(thc.Tensor("half").resize((rows, cols)).fill(1)).numpy()
    for i in (0, 1, count // 2, count - 6):
        assert_bit_equal(x.select(0, i).numpy(), one)


def test_one_matrix(thc):
    """One element a row, at the far end: the result has them there, by the polynomial of numbers."""
    rows, cols = 2100, 1 << 20
    rng = np.random.default_rng(4)
    at = cols - 1 - rng.permutation(5000)[:rows]
    values = (rng.choice([-1, 1], rows) * np.exp(rng.uniform(-2, 0, rows))).astype(np.float16)
    x = thc.Tensor("half").resize((rows, cols)).zero()
    ends = np.zeros((rows, 5000), np.float16)
    ends[np.arange(rows), at - (cols - 5000)] = values
    x.narrow(1, cols - 5000, 5000).copy(thc.Tensor.from_numpy(ends))
    x.orthogonalize(x, 2)
    s = values.astype(np.float64) / (np.linalg.norm(values.astype(np.float64)) + 1e-7)
    for _ in range(2):
        s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
    got = x.narrow(1, cols - 5000, 5000).numpy().astype(np.float64)
    mine = got[np.arange(rows), at - (cols - 5000)]
    assert np.all(np.abs(mine - s) <= 1.5 * 2.0 ** -11 * np.abs(s))      # (the rounding to half, and 2^-22 a few times)
    got[np.arange(rows), at - (cols - 5000)] = 0
    assert np.all(got == 0) and np.all(x.narrow(1, 0, 3000).numpy() == 0)
