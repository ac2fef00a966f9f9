"""AdamW with second moments of every size, down to the smallest float: bit for bit against the same operations in numpy, which keeps
subnormal numbers as the kernels do."""
import numpy as np
import pytest

from tests.test_adamw_gpu import _blocks, _f, _numpy_step, _put
from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
NOTHING = dict(lr=2e-3, beta1=0.9, beta2=0.97, eps=0.0, weight_decay=0.05)


def _every_size(rng, per=64):
    """Floats of every exponent, subnormal ones by their leading bit."""
    normal = (rng.integers(0, 1 << 23, (254, per)) | (np.arange(1, 255)[:, None] << 23)).astype(np.uint32)
    bits = np.arange(23)[:, None]
    subnormal = ((1 << bits) | (rng.integers(0, 1 << 23, (23, per)) & ((1 << bits) - 1))).astype(np.uint32)
    return np.concatenate([subnormal.reshape(-1), normal.reshape(-1)]).view(np.float32)


@pytest.mark.parametrize("eps", [0.0, 1e-30])
@pytest.mark.parametrize("kind,master", [("float", False), ("half", True)])
def test_roots_of_second_moments_of_every_size(thc, kind, master, eps):
    """The moments given, no gradient: the parameter moves by the mean over the root."""
    rng = np.random.default_rng(1)
    h = dict(NOTHING, beta2=0.5, eps=eps)
    v = _every_size(rng)
    v = v[v.view(np.uint32) > 1]           # (half of the smallest would be zero)
    m = rng.uniform(0.5, 1, v.size).astype(np.float32) * np.sqrt(v)
    p = rng.standard_normal(v.size).astype(np.float32)
    q = p.astype(np.float16 if kind == "half" else np.float32)
    g = np.zeros_like(q)
    copies = _put(thc, [p]) if master else None
    dp, dm, dv = _put(thc, [q]), _put(thc, [m]), _put(thc, [v])
    thc.AdamW(dp, _put(thc, [g]), master=copies, mean=dm, square=dv, step=2, **h).step()
    p, m, v = _numpy_step(p, g, m, v, 3, 1.0, h)
    assert_bit_equal(dm[0].numpy(), m)
    assert_bit_equal(dv[0].numpy(), v)
    assert_bit_equal((copies or dp)[0].numpy(), p)
    assert_bit_equal(dp[0].numpy(), p.astype(q.dtype))


@pytest.mark.parametrize("bits", [32, 8])
def test_first_step_of_small_gradients(thc, bits):
    """Gradients from 1e-15 to 1e-21 and no eps: every parameter moves by the rate, as far as the root's own few bits allow."""
    rng = np.random.default_rng(2)
    g = (rng.choice([-1, 1], 4099) * 10.0 ** rng.uniform(-21, -15, 4099)).astype(np.float32)
    p = rng.standard_normal(4099).astype(np.float32)
    d = _put(thc, [p])
    thc.AdamW(d, _put(thc, [g]), bits=bits, **NOTHING).step()
    want, _, v = _numpy_step(p, g, np.zeros_like(p), np.zeros_like(p), 1, 1.0, NOTHING)
    assert (v > 0).all() and (v < 2.0 ** -126).any() and (v > 2.0 ** -110).any()
    assert_bit_equal(d[0].numpy(), want)


def _codes_of_every_size(m, v):
    """8-bit states: means below 2^-120 are zeros; a square's scale is 2^-116 at least, its code 1, where it is not zero."""
    bm, bv = _blocks(m), _blocks(v)
    tm, tv = np.abs(bm).max(1), bv.max(1)
    tm = np.where(tm < 2.0 ** -120, _f(0), tm)
    tv = np.where(tv > 0, np.maximum(tv, _f(2.0 ** -116)), _f(0))
    im, iv = [np.where(t > 0, _f(1) / np.where(t > 0, t, _f(1)), _f(0)).astype(np.float32)[:, None] for t in (tm, tv)]
    cm = np.rint(np.sqrt(np.abs(bm) * im) * _f(127)) * np.sign(bm)
    cv = np.rint(np.sqrt(np.sqrt(bv * iv)) * _f(255))
    cv = np.where(bv > 0, np.maximum(cv, 1), cv)
    return cm.reshape(-1)[:m.size].astype(np.int8), tm, cv.reshape(-1)[:v.size].astype(np.uint8), tv


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("spread", ["blocks", "within"])
def test_8_bit_squares_are_not_lost(thc, kind, spread):
    """Gradients over all sizes, alike in a block or all over it: no square that is not zero comes back as zero, and a step without a
    gradient and without eps, which divides what is left of the mean by the square's root, leaves every parameter finite."""
    rng = np.random.default_rng(3)
    n = 256 * 80 + 77
    size = np.repeat(rng.uniform(-22.3, 18, n // 256 + 1), 256)[:n] if spread == "blocks" else rng.uniform(-22.3, 18, n)
    scale = 1.0
    if kind == "half":          # the type holds down to 6e-8: the rest by the gradients' factor
        size, scale = rng.uniform(-7, 0, n) if spread == "within" else np.repeat(rng.uniform(-7, 0, n // 256 + 1), 256)[:n], 1e-15
    g = (rng.choice([-1, 1], n) * 10.0 ** size).astype(np.float16 if kind == "half" else np.float32)
    p = np.zeros(n, g.dtype)
    d, dg = _put(thc, [p]), _put(thc, [g])
    opt = thc.AdamW(d, dg, bits=8, **NOTHING)
    opt.step(scale)
    _, m, v = _numpy_step(p.astype(np.float32), g, np.zeros(n, np.float32), np.zeros(n, np.float32), 1, scale, NOTHING)
    got = [x[0].numpy() for x in (opt.mean, opt.mean_scale, opt.square, opt.square_scale)]
    for a, b in zip(got, _codes_of_every_size(m, v)):
        assert np.array_equal(a, b)
    mean, square = [x[0].numpy() for x in opt.moments()]
    assert (v == 0).any() or kind == "half"
    assert np.array_equal(square > 0, v > 0)
    # a code's half step, but a whole one where the code is 1 at least, and a few roundings of numbers up to 1
    near, top = v > 2.0 ** -110, np.repeat(got[3], 256)[:n].astype(np.float64)
    off = np.abs((square[near] / top[near]) ** 0.25 - (v[near] / top[near]) ** 0.25)
    assert near.any() and np.all(off <= np.where(v[near] < top[near] * 2.0 ** -32, 1, 0.5) / 255 + 1e-6)
    dg[0].zero()
    opt.step()
    assert np.all(np.isfinite(d[0].numpy())[v > 0])
