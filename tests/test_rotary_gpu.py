"""Rotary positions against float64: both layouts, parts of heads, positions near and far, views, in place, and back."""
import numpy as np
import pytest

from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
NP = {"float": np.float32, "half": np.float16}
UNIT = {"float": 2.0 ** -24, "half": 2.0 ** -11}
TINY = {"float": 2.0 ** -149, "half": 2.0 ** -25}
F32 = 2.0 ** -24


def _turned(x, positions, f, scale, interleaved, inverse):
    """(result, what may be off of it before the last rounding); x is (tokens, heads, dim)."""
    n = 2 * len(f)
    angle = positions.astype(np.float64)[:, None, None] * f * (-1 if inverse else 1)
    c, s = np.cos(angle) * scale, np.sin(angle) * scale
    x = x.astype(np.float64)
    out, mass = x.copy(), np.zeros_like(x)
    first, second = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    # cos and sin: their angle, series and product with the scale round in float (at most 6 steps), two products and a sum follow; the angle
    # in turns has two roundings of 53 bits that the formula's has not
    each = (np.abs(a) + np.abs(b)) * abs(scale) * (9 * F32 + np.abs(angle) * 2.0 ** -52)
    mass[..., first], mass[..., second] = each, each
    return out, mass


def _check(got, x, positions, f, kind, scale=1.0, interleaved=False, inverse=False):
    want, mass = _turned(x, positions, f, np.float32(scale), interleaved, inverse)
    n = 2 * len(f)
    assert_bit_equal(got[..., n:], x[..., n:])
    off = np.abs(got.astype(np.float64) - want)[..., :n]
    bound = (mass + UNIT[kind] * np.abs(want) * 1.01 + TINY[kind])[..., :n]
    assert np.all(off <= bound), (float(np.max(off / bound)), np.argwhere(off > bound)[:3])


def _frequencies(n, base=10000.0):
    return base ** (-np.arange(n) / max(1, n))


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs", [(2, 1), (3, 1), (8, 2), (16, 8), (64, 32), (65, 32), (100, 25), (101, 50), (128, 64), (128, 16), (256, 100), (530, 260)])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (3, 5), (70, 8), (2, 40), (500, 3)])
def test_turn_and_back(thc, kind, interleaved, dim, pairs, tokens, heads):
    rng = np.random.default_rng(dim * 1000 + tokens)
    x = rng.standard_normal((tokens, heads, dim)).astype(NP[kind])
    at = rng.integers(0, 5000, tokens)
    f = _frequencies(pairs)
    t = thc.Tensor.from_numpy
    X, at_, f_ = t(x), t(at), t(f)
    got = thc.Tensor(kind).rotary(X, at_, f_, 1.25, interleaved)
    assert thc.last_kernel() == "rotary"
    _check(got.numpy(), x, at, f, kind, 1.25, interleaved)
    _check(thc.Tensor(kind).rotary(X, at_, f_, 1.0, interleaved, inverse=True).numpy(), x, at, f, kind, 1.0, interleaved, True)
    # in place: the same bits
    place = t(x)
    place.rotary(place, at_, f_, 1.25, interleaved)
    assert_bit_equal(place.numpy(), got.numpy())


@pytest.mark.parametrize("kind", ["float", "half"])
def test_far_positions(thc, kind):
    x = np.random.default_rng(1).standard_normal((7, 2, 32)).astype(NP[kind])
    at = np.array([0, 1, -5, 131071, 1 << 20, (1 << 31) + 12345, -(1 << 31)])
    for f in (_frequencies(16), _frequencies(16, 1e6), np.array([np.pi, np.pi / 2, np.pi / 4, 2 * np.pi] * 4)):
        t = thc.Tensor.from_numpy
        _check(thc.Tensor(kind).rotary(t(x), t(at), t(f)).numpy(), x, at, f, kind)


def test_the_gradient_is_the_way_back(thc):
    """<g, R x> = <R' g, x>, and the length of pairs stays."""
    rng = np.random.default_rng(2)
    x, g = (rng.standard_normal((20, 6, 48)).astype(np.float32) for _ in range(2))
    at, f = rng.integers(0, 1 << 17, 20), _frequencies(20)
    t = thc.Tensor.from_numpy
    for interleaved in (False, True):
        y = thc.Tensor("float").rotary(t(x), t(at), t(f), 0.75, interleaved).numpy().astype(np.float64)
        dx = thc.Tensor("float").rotary(t(g), t(at), t(f), 0.75, interleaved, inverse=True).numpy().astype(np.float64)
        # each of 5760 products is off by 10 roundings of its pair at most
        mass = float((np.abs(g).astype(np.float64) * np.abs(y) + np.abs(dx) * np.abs(x)).sum())
        assert abs(float((g * y).sum() - (dx * x).sum())) <= 20 * F32 * mass
        back = thc.Tensor("float").rotary(t((y / 0.75 ** 2).astype(np.float32)), t(at), t(f), 0.75, interleaved, inverse=True).numpy()
        assert np.allclose(back[..., :40], x[..., :40], rtol=0, atol=40 * F32 * 6)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_views_batches_and_places(thc, kind, interleaved):
    rng = np.random.default_rng(4)
    t = thc.Tensor.from_numpy
    b, n, h, d = 3, 11, 4, 40
    wide = rng.standard_normal((b, n, h + 3, d + 2)).astype(NP[kind])
    at, f = rng.integers(0, 900, (b, n)), _frequencies(12)
    x = wide[:, :, 1:1 + h, 1:1 + d].copy()
    want = thc.Tensor(kind).rotary(t(x), t(at), t(f), 1.0, interleaved).numpy()
    _check(want.reshape(b * n, h, d), x.reshape(b * n, h, d), at.reshape(-1), f, kind, 1.0, interleaved)
    W = t(wide)
    view = W.narrow(2, 1, h).narrow(3, 1, d)
    assert_bit_equal(thc.Tensor(kind).rotary(view, t(at), t(f), 1.0, interleaved).numpy(), want)
    # the heads within a fused projection, in place: what is around them stays
    view.rotary(view, t(at), t(f), 1.0, interleaved)
    held = W.numpy()
    assert_bit_equal(held[:, :, 1:1 + h, 1:1 + d], want)
    held[:, :, 1:1 + h, 1:1 + d] = x
    assert_bit_equal(held, wide)
    # heads before tokens in memory, in and out
    swapped = t(np.ascontiguousarray(x.transpose(0, 2, 1, 3))).t(1, 2)
    out = thc.Tensor(kind).resize((b, h, n, d)).t(1, 2)
    out.rotary(swapped, t(at), t(f), 1.0, interleaved)
    assert_bit_equal(out.numpy(), want)
    # heads whose elements lie apart, and outputs on their input elsewhere
    apart = t(np.ascontiguousarray(x.transpose(0, 1, 3, 2))).t(2, 3)
    assert_bit_equal(thc.Tensor(kind).rotary(apart, t(at), t(f), 1.0, interleaved).numpy(), want)
    flat = t(np.concatenate([x.reshape(-1), np.zeros(d, NP[kind])]))
    strides = (n * h * d, h * d, d, 1)
    moved = flat.view_as_strided(d, (b, n, h, d), strides)
    assert_bit_equal(moved.rotary(flat.view_as_strided(0, (b, n, h, d), strides), t(at), t(f), 1.0, interleaved).numpy(), want)
    # positions that the sequences share, given and counted
    for shared, given in ((at[0], t(at[0])), (np.arange(n), None)):
        got = thc.Tensor(kind).rotary(t(x), given, t(f), 1.0, interleaved).numpy()
        _check(got.reshape(b * n, h, d), x.reshape(b * n, h, d), np.tile(shared, b), f, kind, 1.0, interleaved)
    one = thc.Tensor(kind).rotary(t(x[0, 0]), t(at[0, :1]), t(f), 1.0, interleaved).numpy()
    assert_bit_equal(one, want[0, 0])
    # in pieces, as much as a launch takes
    thc.set_tuning("rotary.items", 64)
    try:
        assert_bit_equal(thc.Tensor(kind).rotary(t(x), t(at), t(f), 1.0, interleaved).numpy(), want)
    finally:
        thc.set_tuning("rotary.items", 1 << 30)


def test_frequencies(thc):
    for dim, base in ((2, 10000.0), (64, 10000.0), (128, 5e5), (130, 1e6)):
        f = base ** (-np.arange(0, dim, 2) / dim)
        got = thc.Tensor("double").rotary_frequencies(dim, base).numpy()
        assert got.shape == (dim // 2,) and np.all(np.abs(got - f) <= 1e-14 * f)
        assert np.all(np.abs(thc.Tensor("double").rotary_frequencies(dim, base, 4.0).numpy() - f / 4) <= 1e-14 * f)
        turns = 4096 * f / (2 * np.pi)
        kept = np.clip((turns - 1) / 31, 0, 1)
        want = f * (kept + (1 - kept) / 8)
        got = thc.Tensor("double").rotary_frequencies(dim, base, 8.0, 4096, 1, 32).numpy()
        assert np.all(np.abs(got - want) <= 1e-13 * f)


def test_refusals(thc):
    F = thc.Tensor
    x, f = F("float").resize((6, 2, 8)).fill(1), F.from_numpy(np.ones(4))
    for call, match in ((lambda: F("float").rotary(x, F.from_numpy(np.arange(5)), f), "5 positions for 6 tokens"),
                        (lambda: F("float").rotary(x, None, F.from_numpy(np.ones(5))), "5 frequencies turn more than heads of 8"),
                        (lambda: F("float").rotary(x, None, F("double")), "no frequencies"),
                        (lambda: F("float").rotary(x.select(0, 0).select(0, 0), None, f), "two dims at least"),
                        (lambda: F("double").rotary_frequencies(7), "even number"),
                        (lambda: F("double").rotary_frequencies(0), "even number"),
                        (lambda: F("double").rotary_frequencies(8, base=0.0), "base"),
                        (lambda: F("double").rotary_frequencies(8, factor=0.0), "factor"),
                        (lambda: F("double").rotary_frequencies(8, slow=2.0, fast=1.0), "more often")):
        with pytest.raises(thc.THCError, match=match):
            call()
    with pytest.raises(ValueError):
        F("float").rotary(x, None, F.from_numpy(np.ones(4, np.float32)))
    assert F("float").rotary(F("float"), None, f).shape == ()
