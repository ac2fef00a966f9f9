"""How near to 64 bits results that are kept in floats come: matrices of floats, and float copies of half parameters, whose step is not rounded to halves."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
A, B, C = 3.4445, -4.7750, 2.0315


def _steps(g, kind, steps, eps=1e-7):
    """The definition with products of `kind`."""
    x = g.astype(np.float64)
    x = (x / (np.linalg.norm(x) + eps)).astype(kind)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.T
    for _ in range(steps):
        a = x @ x.T
        b = kind(B) * a + kind(C) * (a @ a)
        x = kind(A) * x + b @ x
    return (x.T if tall else x).astype(np.float64)


def _matrices(rows, cols, kind):
    """Elements alike; few directions that hold most of the norm; singular values from 1 to 1e-3."""
    rng = np.random.default_rng(rows + cols)
    m, few = min(rows, cols), min(4, rows, cols)
    yield rng.standard_normal((rows, cols)).astype(kind)
    yield ((rng.standard_normal((rows, few)) * np.logspace(0, -1, few)) @ rng.standard_normal((few, cols)) + 0.3 * rng.standard_normal((rows, cols))).astype(kind)
    u, v = np.linalg.qr(rng.standard_normal((rows, m)))[0], np.linalg.qr(rng.standard_normal((cols, m)))[0]
    yield (32 * (u * np.logspace(0, -3, m)) @ v.T).astype(kind)


def _check(got, g, steps):
    """Factors are held in 22 bits where a product of floats takes 24, and sums are of floats in both: each rounding is at most 4 times that of the
    definition in floats. The result itself, and the rate that it is multiplied by, round once more."""
    want = _steps(g, np.float64, steps)
    size = np.linalg.norm(want)
    plain, off = np.linalg.norm(_steps(g, np.float32, steps) - want) / size, np.linalg.norm(got.astype(np.float64) - want) / size
    assert off <= 4 * plain + 2.0 ** -23, (off, plain)


SIZES = [(16, 500), (23, 1024), (33, 500), (500, 33), (65, 65), (65, 513), (128, 512), (200, 400), (700, 300), (256, 1024), (300, 330)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("steps", [3, 5, 6])
def test_matrices_of_floats(thc, rows, cols, steps):
    for g in _matrices(rows, cols, np.float32):
        _check(thc.Tensor("float").orthogonalize(thc.Tensor.from_numpy(g), steps).numpy(), g, steps)


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("steps", [3, 5, 6])
def test_float_copies_of_half_parameters(thc, rows, cols, steps):
    """A first step from zeros: the copies hold the orthogonalised gradient times the rate, in floats."""
    t = thc.Tensor.from_numpy
    for g in _matrices(rows, cols, np.float16):
        copy = t(np.zeros((rows, cols), np.float32))
        thc.Muon([t(np.zeros((rows, cols), np.float16))], [t(g)], master=[copy], lr=-1.0, nesterov=False, steps=steps).step()
        _check(copy.numpy() / np.sqrt(max(1.0, rows / cols)), g, steps)
