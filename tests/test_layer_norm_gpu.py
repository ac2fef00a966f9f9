"""Layer norm and its gradients against float64: rows that end inside a pack, lengths of every way through the kernels, large offsets, views,
outputs on their inputs, sums that are added to."""
import numpy as np
import pytest

from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
NP = {"float": np.float32, "half": np.float16}
UNIT = {"float": 2.0 ** -24, "half": 2.0 ** -11}      # half a step, relative
TINY = {"float": 2.0 ** -149, "half": 2.0 ** -25}
F32 = 2.0 ** -24
# lengths on both sides of every choice of lanes a row, and beyond what registers hold
DIMS = [1, 2, 3, 5, 7, 8, 9, 31, 33, 64, 65, 100, 127, 129, 257, 500, 513, 1000, 1025, 2048, 2049, 4100, 8191, 8200, 16385, 40001]


def _norm(x, eps):
    x = x.astype(np.float64)
    away = x - x.mean(-1, keepdims=True)
    r = 1 / np.sqrt((away ** 2).mean(-1, keepdims=True) + eps)
    return away * r, r, away


def _data(rng, rows, dim, kind, offset=0.0):
    x = (rng.standard_normal((rows, dim)) * np.exp(0.5 * rng.standard_normal(dim)) + offset).astype(NP[kind])
    w = (1 + 0.3 * rng.standard_normal(dim)).astype(NP[kind])
    b = (0.3 * rng.standard_normal(dim)).astype(NP[kind])
    g = rng.standard_normal((rows, dim)).astype(NP[kind])
    return x, w, b, g


def _steps(dim):
    """Roundings in a row of a sum along a row: what a lane adds, then the lanes."""
    return 70 + np.log2(max(2, dim))


def _spread(x, eps):
    """What rounding leaves of a standardised element. The distance to the mean's first part rounds once (to its own size, also far from zero), as do the
    difference to the second part and the product; that second part is a mean of distances, 1 in size at most, the deviation a sum of squares, under
    a root."""
    h, r, _ = _norm(x, eps)
    return h, r, F32 * (6 * np.abs(h) + _steps(x.shape[-1]) * (1 + np.abs(h)))


def _near(got, want, bound, kind):
    bound = bound + UNIT[kind] * np.abs(want) * 1.01 + TINY[kind]
    off = np.abs(got.astype(np.float64) - want)
    worst = float(np.max(off / bound))
    assert worst <= 1, (worst, np.argwhere(off > bound)[:3])


def _check_norm(thc, x, w, b, eps, kind, got):
    h, r, spread = _spread(x, eps)
    w64 = 1.0 if w is None else w.astype(np.float64)
    b64 = 0.0 if b is None else b.astype(np.float64)
    _near(got, h * w64 + b64, spread * np.abs(w64) + 2 * F32 * (np.abs(h * w64) + np.abs(b64)), kind)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("rows", [1, 37])
def test_forward(thc, kind, dim, rows):
    x, w, b, _ = _data(np.random.default_rng(dim * 100 + rows), rows, dim, kind)
    t = thc.Tensor.from_numpy
    got = thc.Tensor(kind).layer_norm(t(x), t(w), t(b), 1e-5)
    assert thc.last_kernel() == "layer-norm"
    _check_norm(thc, x, w, b, 1e-5, kind, got.numpy())
    _check_norm(thc, x, None, None, 1e-5, kind, thc.Tensor(kind).layer_norm(t(x)).numpy())
    _check_norm(thc, x, w, None, 1e-3, kind, thc.Tensor(kind).layer_norm(t(x), t(w), eps=1e-3).numpy())
    _check_norm(thc, x, None, b, 1e-5, kind, thc.Tensor(kind).layer_norm(t(x), None, t(b)).numpy())


def _gradient(x, w, g, eps):
    h, r, spread = _spread(x, eps)
    g = g.astype(np.float64)
    gw = g * (1.0 if w is None else w.astype(np.float64))
    dx = r * (gw - gw.mean(-1, keepdims=True) - h * (gw * h).mean(-1, keepdims=True))
    steps = _steps(x.shape[-1])
    mass, massH = np.abs(gw).mean(-1, keepdims=True), np.abs(gw * h).mean(-1, keepdims=True)
    largest = spread.max(-1, keepdims=True)
    # each of the three terms by its own roundings, h's where h is; the second part of the mean takes its share of the second sum
    bound = r * (4 * F32 * np.abs(gw) + (steps + 4) * F32 * (mass + np.abs(h) * (massH + mass)) + spread * massH + np.abs(h) * mass * largest)
    return dx, bound, (g * h).sum(0), g.sum(0), (np.abs(g * h).sum(0) * (steps + len(x)) * F32 + (np.abs(g) * spread).sum(0)), np.abs(g).sum(0) * (
        steps + len(x)) * F32


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("rows", [1, 5, 300])
def test_gradients(thc, kind, dim, rows):
    if rows * dim > 4000000:
        rows = 40
    rng = np.random.default_rng(dim * 7 + rows)
    x, w, _, g = _data(rng, rows, dim, kind)
    t = thc.Tensor.from_numpy
    dx, bound, dw, db, nearW, nearB = _gradient(x, w, g, 1e-5)
    gotX, gotW, gotB = (thc.Tensor(kind) for _ in range(3))
    gotX.layer_norm_grad(gotW, gotB, t(x), t(g), t(w))
    assert thc.last_kernel() == "layer-norm-grad"
    assert gotW.shape == gotB.shape == (dim,) and gotX.shape == x.shape
    _near(gotX.numpy(), dx, bound, kind)
    _near(gotW.numpy(), dw, nearW, kind)
    _near(gotB.numpy(), db, nearB, kind)
    # the same bits where the weights' gradients are not wanted, or one of them, and in a second call
    alone = thc.Tensor(kind).layer_norm_grad(None, None, t(x), t(g), t(w))
    assert_bit_equal(alone.numpy(), gotX.numpy())
    one = thc.Tensor(kind)
    assert_bit_equal(thc.Tensor(kind).layer_norm_grad(one, None, t(x), t(g), t(w)).numpy(), gotX.numpy())
    assert_bit_equal(one.numpy(), gotW.numpy())
    other = thc.Tensor(kind)
    thc.Tensor(kind).layer_norm_grad(None, other, t(x), t(g), t(w))
    assert_bit_equal(other.numpy(), gotB.numpy())
    # added to what is there
    was = rng.standard_normal((2, dim)).astype(NP[kind])
    addW, addB = t(was[0]), t(was[1])
    thc.Tensor(kind).layer_norm_grad(addW, addB, t(x), t(g), t(w), accumulate=True)
    _near(addW.numpy(), dw + was[0], nearW + F32 * (np.abs(dw) + np.abs(was[0])), kind)
    _near(addB.numpy(), db + was[1], nearB + F32 * (np.abs(db) + np.abs(was[1])), kind)
    # without a weight
    plain = _gradient(x, None, g, 1e-5)
    _near(thc.Tensor(kind).layer_norm_grad(None, None, t(x), t(g)).numpy(), plain[0], plain[1], kind)


def test_gradients_by_differences(thc):
    """The sum of g y, moved along random directions of x, w and b."""
    rng = np.random.default_rng(3)
    x, w, b, g = (a.astype(np.float64) for a in _data(rng, 6, 50, "float"))
    t = thc.Tensor.from_numpy
    dx, dw, db = (thc.Tensor("float") for _ in range(3))
    dx.layer_norm_grad(dw, db, t(x.astype(np.float32)), t(g.astype(np.float32)), t(w.astype(np.float32)))
    x, w, g = (a.astype(np.float32).astype(np.float64) for a in (x, w, g))

    def total(x, w, b):
        return float((g * (_norm(x, 1e-5)[0] * w + b)).sum())

    for k, (grad, size) in enumerate(((dx.numpy(), x.shape), (dw.numpy(), w.shape), (db.numpy(), b.shape))):
        d = rng.standard_normal(size)
        moved = [[v + s * 1e-5 * d if i == k else v for i, v in enumerate((x, w, b))] for s in (1, -1)]
        slope = (total(*moved[0]) - total(*moved[1])) / 2e-5
        mass = float(np.abs(grad * d).sum())
        # float gradients (70 roundings at most) and differences of a sum of 300 terms, off by 1e-10 of its third derivatives
        assert abs(slope - float((grad.astype(np.float64) * d).sum())) <= 100 * F32 * mass + 1e-6 * mass


@pytest.mark.parametrize("dim", [40, 700, 3001, 40001])
def test_large_offsets(thc, dim):
    """Rows far from zero: what is left of their digits counts, the mean does not take it."""
    rng = np.random.default_rng(dim)
    x, w, b, g = _data(rng, 9, dim, "float", offset=3e4)
    t = thc.Tensor.from_numpy
    _check_norm(thc, x, w, b, 1e-5, "float", thc.Tensor("float").layer_norm(t(x), t(w), t(b)).numpy())
    dx, bound = _gradient(x, w, g, 1e-5)[:2]
    _near(thc.Tensor("float").layer_norm_grad(None, None, t(x), t(g), t(w)).numpy(), dx, bound, "float")


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("dim", [33, 1500, 33000])
def test_views_and_places(thc, kind, dim):
    rng = np.random.default_rng(dim)
    rows = 12
    wide, w, b, gwide = _data(rng, rows, dim + 5, kind)
    w, b = w[:dim].copy(), b[:dim].copy()
    x, g = wide[:, 2:2 + dim].copy(), gwide[:, 3:3 + dim].copy()
    t = thc.Tensor.from_numpy
    want = thc.Tensor(kind).layer_norm(t(x), t(w), t(b)).numpy()
    wantX, wantW, wantB = (thc.Tensor(kind) for _ in range(3))
    wantX.layer_norm_grad(wantW, wantB, t(x), t(g), t(w))
    wantX, wantW, wantB = wantX.numpy(), wantW.numpy(), wantB.numpy()

    def close(got, wanted):
        # (rows at other addresses: the same lanes sum the same elements)
        assert_bit_equal(got, wanted)

    # windows in, windows out, in place
    room = thc.Tensor(kind).resize((rows, dim + 9)).fill(7)
    close(room.narrow(1, 3, dim).layer_norm(t(wide).narrow(1, 2, dim), t(w), t(b)).numpy(), want)
    held = room.numpy()
    assert np.all(held[:, :3] == 7) and np.all(held[:, 3 + dim:] == 7)
    place = t(wide)
    place.narrow(1, 2, dim).layer_norm(place.narrow(1, 2, dim), t(w), t(b))
    close(place.numpy()[:, 2:2 + dim], want)
    assert_bit_equal(place.numpy()[:, :2], wide[:, :2])
    # overlapping the input at another place
    both = t(np.concatenate([x.reshape(-1), np.zeros(dim, NP[kind])]))
    out = both.view_as_strided(dim, (rows, dim), (dim, 1))
    close(out.layer_norm(both.view_as_strided(0, (rows, dim), (dim, 1)), t(w), t(b)).numpy(), want)
    # transposed: columns of memory, strided weights
    cols = t(np.ascontiguousarray(x.T)).t()
    pairs = t(np.ascontiguousarray(np.stack([w, b], 1)))
    close(thc.Tensor(kind).layer_norm(cols, pairs.select(1, 0), pairs.select(1, 1)).numpy(), want)
    out = thc.Tensor(kind).resize((dim, rows)).t()
    close(out.layer_norm(t(x), t(w), t(b)).numpy(), want)
    # batches of rows; one row of one dim
    close(thc.Tensor(kind).layer_norm(t(x.reshape(3, 2, 2, dim)), t(w), t(b)).numpy().reshape(rows, dim), want)
    close(thc.Tensor(kind).layer_norm(t(x).select(0, 4), t(w), t(b)).numpy(), want[4])
    # gradients in the place of either input, of views, with strided sums in the gaps of one matrix
    for which in (0, 1):
        px, pg = t(wide), t(gwide)
        at = px.narrow(1, 2, dim) if which == 0 else pg.narrow(1, 3, dim)
        sums = thc.Tensor(kind).resize((dim, 2)).fill(3)
        at.layer_norm_grad(sums.select(1, 0), sums.select(1, 1), px.narrow(1, 2, dim), pg.narrow(1, 3, dim), t(w))
        close(at.numpy(), wantX)
        close(sums.numpy()[:, 0], wantW)
        close(sums.numpy()[:, 1], wantB)
    # a gradient that is one row for all (stride 0)
    line = t(g[:1].copy())
    spread = line.view_as_strided(0, (rows, dim), (0, 1))
    a, c = thc.Tensor(kind), thc.Tensor(kind)
    thc.Tensor(kind).layer_norm_grad(a, c, t(x), spread, t(w))
    a2, c2 = thc.Tensor(kind), thc.Tensor(kind)
    thc.Tensor(kind).layer_norm_grad(a2, c2, t(x), t(np.repeat(g[:1], rows, 0)), t(w))
    close(a.numpy(), a2.numpy())
    close(c.numpy(), c2.numpy())


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("dim", [5, 70, 1025])
def test_odd_values(thc, kind, dim):
    t = thc.Tensor.from_numpy
    x = np.ones((6, dim), NP[kind])
    x[1] = 0
    x[2, 0] = np.nan
    x[3, dim - 1] = np.inf
    x[4] = np.finfo(NP["half"]).max
    x[5] = np.where(np.arange(dim) % 2, -1, 1) * np.finfo(NP["half"]).max
    w = np.full(dim, 2, NP[kind])
    got = thc.Tensor(kind).layer_norm(t(x), t(w)).numpy()
    assert np.all(got[[0, 1, 4]] == 0) and np.all(np.isnan(got[2:4]))
    want = _norm(x[5:].astype(np.float64), 1e-5)[0] * 2
    assert np.all(np.abs(got[5:] - want) <= 1e-2)
    # rows of one value have no direction: their gradient is finite, with eps
    dx = thc.Tensor(kind).layer_norm_grad(None, None, t(x[:1]), t(w[None, :].copy())).numpy()
    assert np.all(dx == 0)
    # rows with a NaN leave the others alone; the sums over rows take it up
    gw = thc.Tensor(kind)
    dx = thc.Tensor(kind).layer_norm_grad(gw, None, t(x), t(np.ones((6, dim), NP[kind]))).numpy()
    assert np.all(np.isfinite(dx[[0, 1, 4, 5]])) and np.all(np.isnan(dx[2:4])) and np.all(np.isnan(gw.numpy()))


def test_many_rows(thc):
    """More rows than one launch has workgroups; sums of whole numbers are exact."""
    rows, dim = 70001, 24
    t = thc.Tensor.from_numpy
    x = np.where(np.arange(dim) % 2, -1.0, 1.0).astype(np.float32) * np.ones((rows, 1), np.float32)
    g = np.random.default_rng(0).integers(-3, 4, (rows, dim)).astype(np.float32)
    dw, db = thc.Tensor("float"), thc.Tensor("float")
    thc.Tensor("float").layer_norm_grad(dw, db, t(x), t(g), eps=0.0)
    assert np.array_equal(db.numpy(), g.sum(0, dtype=np.float64).astype(np.float32))
    assert np.array_equal(dw.numpy(), (g.astype(np.float64) * x).sum(0).astype(np.float32))


def test_refusals(thc):
    F = thc.Tensor
    x, w = F("float").resize((4, 6)).fill(1), F("float").resize((6,)).fill(1)
    for call, match in ((lambda: F("float").layer_norm(x, F("float").resize((5,)).fill(1)), "weights for rows of 6"),
                        (lambda: F("float").layer_norm(x, w, F("float").resize((7,)).fill(1)), "biases for rows of 6"),
                        (lambda: F("float").layer_norm(x, eps=-1.0), "eps is negative"),
                        (lambda: w.layer_norm(x, w), "may not be the weight"),
                        (lambda: F("float").layer_norm_grad(None, None, F("float"), F("float")), "input is empty"),
                        (lambda: F("float").layer_norm_grad(None, None, x, F("float").resize((6, 4)).fill(1)), "other sizes"),
                        (lambda: F("float").layer_norm_grad(F("float").resize((5,)).fill(1), None, x, x, accumulate=True), "to be added to for rows of 6"),
                        (lambda: F("float").layer_norm_grad(x, None, x, x), "may not be another operand"),
                        (lambda: F("float").layer_norm_grad(None, w, x, x, w), "may not be another operand")):
        with pytest.raises(thc.THCError, match=match):
            call()
    both = F("float").resize((10,)).fill(1)
    with pytest.raises(thc.THCError, match="weight and bias share memory"):
        F("float").layer_norm_grad(both.narrow(0, 0, 6), both.narrow(0, 4, 6), x, x)
    with pytest.raises(thc.THCError, match="one tensor"):
        both = F("float")
        F("float").layer_norm_grad(both, both, x, x)
    room = F("float").resize((30,)).fill(1)
    with pytest.raises(thc.THCError, match="weight and input share memory"):
        room.view_as_strided(0, (4, 6), (6, 1)).layer_norm_grad(room.narrow(0, 20, 6), None, x, x)
    with pytest.raises(ValueError):
        F("float").layer_norm(F("half"))
    assert F("float").layer_norm(F("float")).shape == ()


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("dim", [3, 64, 500, 513, 2048, 5000, 16384])
def test_gradients_of_few_rows(thc, kind, dim):
    """One workgroup's sums or several's: the weights' gradients of as many rows as either has, and a few more; added and written, one without the other."""
    rng = np.random.default_rng(dim)
    t = thc.Tensor.from_numpy
    for rows in (1, 2, 4, 5, 8, 9, 16, 17, 33, 128, 129):
        if rows * dim > 1 << 18:
            continue
        x, g, w = (rng.standard_normal(s).astype(NP[kind]) for s in ((rows, dim), (rows, dim), (dim,)))
        was = rng.standard_normal(dim).astype(NP[kind])
        X, G = x.astype(np.float64), g.astype(np.float64)
        m, v = X.mean(1, keepdims=True), X.var(1, keepdims=True)
        h = (X - m) / np.sqrt(v + 1e-5)
        both = thc.Tensor(kind), t(was.copy()), t(was.copy())
        both[0].layer_norm_grad(both[1], both[2], t(x), t(g), t(w), accumulate=True)
        one = thc.Tensor(kind), t(was.copy())
        one[0].layer_norm_grad(one[1], None, t(x), t(g), t(w))
        for got, terms, begin in ((both[1], G * h, was), (both[2], G, was), (one[1], G * h, 0 * was)):
            want = terms.sum(0) + begin.astype(np.float64)
            # a sum of `rows` terms in float, of which each has an h that is off by up to 8 roundings of itself and of the deviations' size, and the last rounding
            room = 2.0 ** -24 * ((rows + 16) * np.abs(terms).sum(0) + 16 * np.abs(G).sum(0) + np.abs(begin)) + 1.01 * UNIT[kind] * np.abs(want) + 2.0 ** -25
            assert np.all(np.abs(got.numpy().astype(np.float64) - want) <= room), (rows, np.max(np.abs(got.numpy() - want) / room))
