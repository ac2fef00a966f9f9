"""Layer norm of rows without a deviation, or hardly one, far from zero: the mean of squares about the mean is not negative, whatever sums of large floats round to."""
import numpy as np
import pytest

from tests.test_layer_norm_gpu import _check_norm, _gradient, _near

pytestmark = pytest.mark.gpu
NP = {"float": np.float32, "half": np.float16}
# a length on each way through the kernels, none whose sums are exact
DIMS = [3, 7, 61, 127, 251, 509, 1021, 2039, 4093, 6798, 8191, 14957, 15437, 16381, 33331]


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("eps", [1e-5, 1e-12])
def test_rows_of_one_value(thc, kind, dim, eps):
    """The deviation is 0: results are the bias; the gradient is what is left of the output's gradient without its mean, over the root of eps."""
    rng = np.random.default_rng(dim)
    values = np.concatenate([[875835840.0, 519588704.0, 7865604.5, -3.3e7, 1e30, 1.7e-3], np.exp(rng.uniform(np.log(1e4), np.log(1e12), 26))])
    if kind == "half":
        values = rng.uniform(100, 65000, 32)
    x = np.repeat(values.astype(NP[kind])[:, None], dim, 1)
    w, b = (1 + 0.3 * rng.standard_normal(dim)).astype(NP[kind]), rng.standard_normal(dim).astype(NP[kind])
    t = thc.Tensor.from_numpy
    got = thc.Tensor(kind).layer_norm(t(x), t(w), t(b), eps).numpy()
    assert np.array_equal(got, np.repeat(b[None, :], len(x), 0)), np.argwhere(got != b)[:4]
    # eps is a float; gradients of -1, 0 and 1 and weights of ones sum exactly
    g = rng.integers(-1, 2, (len(x), dim)).astype(NP[kind])
    gw, gb = thc.Tensor(kind), thc.Tensor(kind)
    dx = thc.Tensor(kind).layer_norm_grad(gw, gb, t(x), t(g), eps=eps).numpy().astype(np.float64)
    g = g.astype(np.float64)
    want = (g - g.mean(1, keepdims=True)) / np.sqrt(np.float64(np.float32(eps)))
    if kind == "half":
        want = np.clip(want, -1e30, 1e30)
        assert np.all(np.isinf(dx[np.abs(want) > 65520])) and np.all(np.sign(dx[np.abs(want) > 65520]) == np.sign(want[np.abs(want) > 65520]))
        dx, want = dx[np.abs(want) < 65500], want[np.abs(want) < 65500]
    # the root and its instruction, the mean, two products and their difference: 8 roundings of the largest term, and the type's
    assert np.all(np.abs(dx - want) <= 8 * 2.0 ** -24 * 2 / np.sqrt(eps) + np.finfo(NP[kind]).eps / 2 * 1.01 * np.abs(want))
    assert np.all(gw.numpy() == 0)


@pytest.mark.parametrize("dim", DIMS)
def test_rows_of_nearly_one_value(thc, dim):
    """One element in three is a float's step above the others: a deviation of less than a step."""
    rng = np.random.default_rng(dim)
    values = np.exp(rng.uniform(np.log(1e5), np.log(1e9), 40)).astype(np.float32)
    x = np.repeat(values[:, None], dim, 1)
    up = rng.permuted(np.arange(dim)[None, :].repeat(40, 0), axis=1) < max(1, dim // 3)
    x = np.where(up, np.nextafter(x, np.float32(np.inf)), x)
    got = thc.Tensor("float").layer_norm(thc.Tensor.from_numpy(x), eps=1e-5).numpy().astype(np.float64)
    away = x.astype(np.float64) - x.astype(np.float64).mean(1, keepdims=True)
    want = away / np.sqrt((away ** 2).mean(1, keepdims=True) + 1e-5)
    # distances are exact multiples of a step (the first part of the mean, a float, is within one); as in the other tests, sums of 70 roundings and the lanes',
    # of squares of up to 9/2 of the variance, and of distances of up to 3 / sqrt(2) of the deviation
    steps = 70 + np.log2(dim)
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * steps * (5 * np.abs(want) + 3))


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("dim", DIMS)
def test_rows_whose_first_element_is_far_from_the_others(thc, kind, dim):
    rng = np.random.default_rng(dim)
    x, w, b, g = (rng.standard_normal(s).astype(NP[kind]) for s in ((8, dim), (dim,), (dim,), (8, dim)))
    x[:, 0] = rng.choice([-1, 1], 8) * np.array([10, 1e3, 5e4, 6.5e4] * 2 if kind == "half" else [1e2, 1e4, 1e6, 1e8] * 2)
    t = thc.Tensor.from_numpy
    _check_norm(thc, x, w, b, 1e-5, kind, thc.Tensor(kind).layer_norm(t(x), t(w), t(b), 1e-5).numpy())
    dx, bound = _gradient(x, w, g, 1e-5)[:2]
    _near(thc.Tensor(kind).layer_norm_grad(None, None, t(x), t(g), t(w)).numpy(), dx, bound, kind)
