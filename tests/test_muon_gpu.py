"""Newton-Schulz orthogonalisation and the optimizer on it against float64: sizes around the products' tiles and blocks, tall and wide, batches,
matrices whose every element is known, lists, states, views."""
import numpy as np
import pytest

from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
NP = {"float": np.float32, "half": np.float16}
UNIT = {"float": 2.0 ** -24, "half": 2.0 ** -11}
TINY = {"float": 2.0 ** -149, "half": 2.0 ** -25}
A, B, C = 3.4445, -4.7750, 2.0315


def _steps(x, steps=5, eps=1e-7, noise=None):
    """The definition in float64. With `noise`, a generator, every operand of a product is off by up to 2^-22 of itself and of the usual size
    of its elements, and products are of floats: what the kernels' rounding may do, by the same steps."""
    x = x.astype(np.float64)
    x = x / (np.linalg.norm(x) + eps)

    def off(m):
        if noise is None:
            return m
        size = np.abs(m) + np.sqrt((m ** 2).mean())
        return (m + size * 2.0 ** -22 * noise.uniform(-1, 1, m.shape)).astype(np.float32)

    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.T
    for _ in range(steps):
        x = off(x)
        a = off(x @ x.T)
        b = off(np.float64(B) * a + np.float64(C) * (a @ a))
        x = np.float64(A) * x + b @ x
    return np.asarray(x.T if tall else x, np.float64)


def _check(got, source, kind, steps=5, seed=0):
    """got near the definition: 8 times what rounding did in the definition's steps, and the rounding to the type; no element off by more than that
    of the whole matrix, which an element left out would be."""
    want = _steps(source, steps)
    room = 8 * np.linalg.norm(_steps(source, steps, noise=np.random.default_rng(seed)) - want) + 2.0 ** -24 * np.linalg.norm(want)
    off = got.astype(np.float64) - want
    last = UNIT[kind] * np.abs(want) * 1.01 + TINY[kind]
    beyond = np.maximum(np.abs(off) - last, 0)
    assert np.linalg.norm(beyond) <= room, (np.linalg.norm(beyond) / np.linalg.norm(want), room / np.linalg.norm(want))
    # rounding spreads: an element has a few times its share of it
    share = 12 * room / np.sqrt(want.size) + 2.0 ** -20 * np.abs(want)
    assert np.all(beyond <= share), (float(np.max(beyond / share)), np.argwhere(beyond > share)[:3])


def _matrix(rng, rows, cols, kind, size=1.0):
    r = min(4, rows, cols)
    m = rng.standard_normal((rows, r)) * np.logspace(0, -1, r) @ rng.standard_normal((r, cols)) + 0.3 * rng.standard_normal((rows, cols))
    return (size * m).astype(NP[kind])


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 9), (9, 1), (2, 3), (5, 5), (31, 33), (32, 32), (64, 200), (65, 63), (127, 129), (128, 128), (129, 300),
                                       (300, 129), (257, 31), (400, 1000), (520, 520)])
def test_sizes(thc, kind, rows, cols):
    g = _matrix(np.random.default_rng(rows * 1000 + cols), rows, cols, kind)
    t = thc.Tensor.from_numpy
    got = thc.Tensor(kind).orthogonalize(t(g))
    assert thc.last_kernel() == "orthogonalize"
    _check(got.numpy(), g, kind)
    # the same bits in a second call and in place
    place = t(g)
    assert_bit_equal(place.orthogonalize(place).numpy(), got.numpy())


@pytest.mark.parametrize("steps", [1, 2, 3, 6, 9])
def test_steps(thc, steps):
    g = _matrix(np.random.default_rng(steps), 70, 150, "float")
    _check(thc.Tensor("float").orthogonalize(thc.Tensor.from_numpy(g), steps).numpy(), g, "float", steps)


def _scalar_steps(s, steps=5):
    for _ in range(steps):
        s = A * s + B * s ** 3 + C * s ** 5
    return s


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("rows,cols", [(7, 7), (33, 150), (150, 33), (260, 300), (300, 260)])
def test_one_element_a_row(thc, kind, rows, cols):
    """Matrices with one element in each row and column at most: the result has them at the same places, each by the polynomial of numbers, and zeros
    elsewhere, exactly. Every element of the products' operands is told from every other."""
    rng = np.random.default_rng(rows + cols)
    m = min(rows, cols)
    g = np.zeros((rows, cols), NP[kind])
    at = rng.permutation(rows)[:m], rng.permutation(cols)[:m]
    values = (rng.choice([-1, 1], m) * np.exp(rng.uniform(-3, 0, m))).astype(NP[kind])
    g[at] = values
    got = thc.Tensor(kind).orthogonalize(thc.Tensor.from_numpy(g)).numpy().astype(np.float64)
    want = _scalar_steps(values.astype(np.float64) / (np.linalg.norm(g.astype(np.float64)) + 1e-7))
    where = np.ones_like(got, bool)
    where[at] = False
    assert np.all(got[where] == 0)
    # an operand is off by 2^-22 of itself; a step makes at most 8 of that relative to the value, as s p'(s) / p(s) is between -0.85 and 1
    # up to s = 1.05, and p's terms add to at most 9 times p
    assert np.all(np.abs(got[at] - want) <= (5 * 10 * 2.0 ** -22 + UNIT[kind] * 1.01) * np.abs(want) * 1.5), np.max(np.abs(got[at] / want - 1))


@pytest.mark.parametrize("kind", ["float", "half"])
def test_singular_values(thc, kind):
    for rows, cols in ((90, 200), (200, 90), (256, 256)):
        g = _matrix(np.random.default_rng(rows), rows, cols, kind)
        got = thc.Tensor(kind).orthogonalize(thc.Tensor.from_numpy(g)).numpy().astype(np.float64)
        s = np.linalg.svd(got, compute_uv=False)
        first = np.linalg.svd(g.astype(np.float64), compute_uv=False) / np.linalg.norm(g.astype(np.float64))
        # a rounding of every element moves singular values by its norm at most
        assert np.all(np.abs(np.sort(s) - np.sort(_scalar_steps(first))) <= 2.0 * UNIT[kind] * np.sqrt(min(rows, cols)) * 1.3 + 1e-4)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("shape", [(3, 40, 70), (2, 3, 130, 20), (100, 17, 9), (1, 1, 5, 6)])
def test_batches(thc, kind, shape):
    rng = np.random.default_rng(len(shape))
    g = np.stack([_matrix(rng, shape[-2], shape[-1], kind, 10.0 ** rng.uniform(-2, 1)) for _ in range(int(np.prod(shape[:-2])))])
    t = thc.Tensor.from_numpy
    got = thc.Tensor(kind).orthogonalize(t(g.reshape(shape))).numpy().reshape(g.shape)
    for i in range(len(g)):
        assert_bit_equal(got[i], thc.Tensor(kind).orthogonalize(t(g[i])).numpy(), "matrix %d" % i)
    _check(got[-1], g[-1], kind)


@pytest.mark.parametrize("kind", ["float", "half"])
def test_views(thc, kind):
    rng = np.random.default_rng(8)
    wide = _matrix(rng, 60, 90, kind)
    t = thc.Tensor.from_numpy
    W = t(wide)
    inner = wide[3:53, 5:85].copy()
    want = thc.Tensor(kind).orthogonalize(t(inner)).numpy()
    view = W.narrow(0, 3, 50).narrow(1, 5, 80)
    assert_bit_equal(thc.Tensor(kind).orthogonalize(view).numpy(), want)
    room = thc.Tensor(kind).resize((55, 90)).fill(9)
    room.narrow(0, 2, 50).narrow(1, 4, 80).orthogonalize(view)
    held = room.numpy()
    assert_bit_equal(held[2:52, 4:84], want)
    held[2:52, 4:84] = 9
    assert np.all(held == 9)
    turned = thc.Tensor(kind).orthogonalize(view.t()).numpy()
    _check(turned, inner.T, kind)
    view.orthogonalize(view)
    held = W.numpy()
    assert_bit_equal(held[3:53, 5:85], want)
    held[3:53, 5:85] = inner
    assert_bit_equal(held, wide)
    flat = t(np.concatenate([inner.reshape(-1), np.zeros(80, NP[kind])]))
    assert_bit_equal(flat.view_as_strided(80, (50, 80), (80, 1)).orthogonalize(flat.view_as_strided(0, (50, 80), (80, 1))).numpy(), want)


def test_sizes_of_values(thc):
    """Norms beyond what squares of floats hold; zeros; what is not finite stays within its matrix."""
    t = thc.Tensor.from_numpy
    g = _matrix(np.random.default_rng(5), 40, 60, "float")
    for size in (1e-30, 1e-12, 1e15, 1e30):
        x = (g * np.float32(size)).astype(np.float32)
        got = thc.Tensor("float").orthogonalize(t(x), 5, 0.0).numpy()
        want = _steps(x, 5, 0.0)
        assert np.linalg.norm(got - want) <= 2e-5 * np.linalg.norm(want)
    batch = np.stack([g, 0 * g, g, g])
    batch[2, 3, 4] = np.nan
    batch[3, 0, 0] = np.inf
    got = thc.Tensor("float").orthogonalize(t(batch)).numpy()
    assert_bit_equal(got[0], thc.Tensor("float").orthogonalize(t(g)).numpy())
    assert np.all(got[1] == 0) and np.all(np.isnan(got[2])) and np.all(np.isnan(got[3]))
    # one element far above the others
    g = g * np.float32(1e-3)
    g[7, 9] = 50
    _check(thc.Tensor("float").orthogonalize(t(g)).numpy(), g, "float")


# ---------------------------------------------------------------------- the optimizer --
def _muon(p, g, m, scale, lr, beta, decay, nesterov, steps, eps, match):
    g = np.float32(scale) * g.astype(np.float64)
    m = np.float32(beta) * m + g
    u = (g + np.float32(beta) * m) if nesterov else m
    rows, cols = p.shape[-2:]
    rate = lr * (match * np.sqrt(max(rows, cols)) if match else np.sqrt(max(1, rows / cols)))
    shape = u.shape
    o = np.stack([_steps(x, steps, eps) for x in u.reshape((-1,) + shape[-2:])]).reshape(shape)
    return p * (1 - lr * decay) - rate * o, m, rate


@pytest.mark.parametrize("kind,master", [("float", False), ("half", False), ("half", True)])
@pytest.mark.parametrize("nesterov,match", [(True, 0.0), (False, 0.2)])
def test_step(thc, kind, master, nesterov, match):
    rng = np.random.default_rng(11)
    t = thc.Tensor.from_numpy
    shapes = [(5, 5), (70, 33), (33, 70), (3, 20, 150), (130, 260), (1, 8)] + [(9, 12)] * 50      # more than a launch takes
    params = [(0.1 * rng.standard_normal(s)).astype(np.float32) for s in shapes]
    source = params if kind == "float" or master else [p.astype(np.float16).astype(np.float32) for p in params]
    P = [t(p.astype(NP[kind])) for p in params]
    M = [t(p) for p in params] if master else None
    G = [thc.Tensor(kind) for _ in shapes]
    opt = thc.Muon(P, G, master=M, lr=0.03, beta=0.9, weight_decay=0.1, nesterov=nesterov, match_rms=match)
    m = [np.zeros(s) for s in shapes]
    p = [x.astype(np.float64) for x in source]
    for _ in range(3):
        g = [(8 * rng.standard_normal(s)).astype(NP[kind]) for s in shapes]
        opt.grads = [t(x) for x in g]
        opt.step(1 / 16)
        assert thc.last_kernel() == "muon"
        for i in range(len(shapes)):
            want, m[i], rate = _muon(p[i], g[i], m[i], 1 / 16, 0.03, 0.9, 0.1, nesterov, 5, 1e-7, match)
            # the momentum rounds once a step
            assert np.all(np.abs(opt.momentum[i].numpy() - m[i]) <= 2.0 ** -22 * (np.abs(m[i]) + 1))
            got = (M[i] if master else P[i]).numpy().astype(np.float64)
            # 1e-4 of the update's norm for its rounding (amplified up to 3.4445^5 in its smallest directions), and the parameter's own
            step = rate * np.sqrt(min(shapes[i][-2:])) * 1.3 * np.sqrt(np.prod(shapes[i][:-2]))
            unit = 2.0 ** -24 if master else UNIT[kind]
            assert np.linalg.norm(got - want) <= 2e-4 * step + 3 * unit * np.linalg.norm(want)
            if master:
                assert_bit_equal(P[i].numpy(), M[i].numpy().astype(np.float16))
            m[i] = opt.momentum[i].numpy().astype(np.float64)      # (go on from what is there)
            p[i] = got


def test_passes_and_pieces(thc):
    """A batch whose workspace is beyond one pass's is cut; the same bits come out."""
    rng = np.random.default_rng(2)
    one = _matrix(rng, 600, 600, "half")
    t = thc.Tensor.from_numpy
    want = thc.Tensor("half").orthogonalize(t(one)).numpy()
    many = thc.Tensor("half").resize((150, 600, 600))
    for i in range(150):
        many.select(0, i).copy(t(one))
    got = thc.Tensor("half").orthogonalize(many).numpy()
    for i in (0, 1, 74, 148, 149):
        assert_bit_equal(got[i], want)
    assert all(np.array_equal(got[0], x) for x in got)


@pytest.mark.parametrize("kind", ["float", "half"])
def test_a_matrix_does_not_depend_on_the_others(thc, kind):
    """Sizes of every way through the kernels, whose tiles and launches are chosen by all of a call's matrices: the bits of calls of their own."""
    rng = np.random.default_rng(6)
    shapes = [(600, 600), (65, 513), (128, 128), (30, 2000), (300, 1500), (40, 40), (1300, 260), (129, 129), (513, 65), (7, 3), (1024, 1100), (200, 3000)] * 2
    t = thc.Tensor.from_numpy
    params = [rng.standard_normal(s).astype(NP[kind]) for s in shapes]
    grads = [_matrix(rng, s[0], s[1], kind) for s in shapes]
    together = [t(p) for p in params]
    opt = thc.Muon(together, [t(g) for g in grads])
    opt.step(0.5)
    opt.step(0.5)
    for i, (p, g) in enumerate(zip(params, grads)):
        alone = t(p)
        one = thc.Muon([alone], [t(g)])
        one.step(0.5)
        one.step(0.5)
        assert_bit_equal(together[i].numpy(), alone.numpy(), "matrix %d" % i)
        assert_bit_equal(opt.momentum[i].numpy(), one.momentum[0].numpy())


def test_ends_of_the_floats(thc):
    """Elements so small or large that one float does not hold what they are multiplied by."""
    t = thc.Tensor.from_numpy
    for rows, cols in ((20, 30), (40, 300), (150, 140)):
        g = np.round(_matrix(np.random.default_rng(rows), rows, cols, "float") * 64).astype(np.float32)
        want = thc.Tensor("float").orthogonalize(t(g), 5, 0.0).numpy()
        for e in (-148, -130, 110, 118):      # (times a power of two: nothing rounds)
            got = thc.Tensor("float").orthogonalize(t(np.ldexp(g, e)), 5, 0.0).numpy()
            assert_bit_equal(got, want, "2^%d" % e)


def test_list_of_views_keeps_what_is_around(thc):
    rng = np.random.default_rng(3)
    t = thc.Tensor.from_numpy
    wide, g = rng.standard_normal((30, 50)).astype(np.float32), rng.standard_normal((20, 40)).astype(np.float32)
    W = t(wide)
    view = W.narrow(0, 4, 20).narrow(1, 3, 40)
    dense = t(wide[4:24, 3:43].copy())
    thc.Muon([view], [t(g)]).step()
    thc.Muon([dense], [t(g)]).step()
    held = W.numpy()
    assert_bit_equal(held[4:24, 3:43], dense.numpy())
    held[4:24, 3:43] = wide[4:24, 3:43]
    assert_bit_equal(held, wide)


def test_resumed_run(thc):
    rng = np.random.default_rng(4)
    t = thc.Tensor.from_numpy
    p, g = rng.standard_normal((40, 30)).astype(np.float32), rng.standard_normal((40, 30)).astype(np.float32)
    a = t(p)
    whole = thc.Muon([a], [t(g)])
    for _ in range(4):
        whole.step()
    b = t(p)
    first = thc.Muon([b], [t(g)])
    first.step()
    first.step()
    second = thc.Muon([b], [t(g)], momentum=[x.clone() for x in first.momentum])
    second.step()
    second.step()
    assert_bit_equal(b.numpy(), a.numpy())
    empty = thc.Muon([], [])
    empty.step()
    nothing = thc.Muon([thc.Tensor("float")], [thc.Tensor("float")])
    nothing.step()


def test_refusals(thc):
    F = thc.Tensor
    x = F("float").resize((4, 6)).fill(1)
    for call, match in ((lambda: F("float").orthogonalize(x.select(0, 0)), "two dims at least"), (lambda: F("float").orthogonalize(x, 0), "0 steps"),
                        (lambda: F("float").orthogonalize(x, 5, -1.0), "eps is negative"),
                        (lambda: thc.Muon([x.select(0, 0)], [x.select(0, 0)]).step(), "two dims at least"),
                        (lambda: thc.Muon([x], [x.t()]).step(), "other sizes"),
                        (lambda: thc.Muon([x], [x], beta=1.0).step(), "beta"),
                        (lambda: thc.Muon([x], [x], match_rms=-1.0).step(), "negative"),
                        (lambda: thc.Muon([x], [x], steps=0).step(), "steps"),
                        (lambda: thc.Muon([x.view_as_strided(0, (4, 6), (0, 1))], [x]).step(), "overlap")):
        with pytest.raises(thc.THCError, match=match):
            call()
    with pytest.raises(ValueError):
        thc.Muon([x], [F("half")])
    with pytest.raises(ValueError, match="float parameters have no mean"):
        thc.Muon([x], [x])._hold("mean", [x])
    assert np.all(x.numpy() == 1)
    assert F("float").orthogonalize(F("float")).shape == ()


def _chained(x, lengths, noise=None, eps=1e-7):
    """The definition in float64 with one X X' for several steps: A' = P A P, X'' = P' P X. `noise` as in `_steps`."""
    x = x.astype(np.float64)
    x = x / (np.linalg.norm(x) + eps)

    def off(m):
        if noise is None:
            return m
        size = np.abs(m) + np.sqrt((m ** 2).mean())
        return (m + size * 2.0 ** -22 * noise.uniform(-1, 1, m.shape)).astype(np.float32)

    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.T
    one = np.eye(len(x))
    for length in lengths:
        x = off(x)
        a, q = off(x @ x.T), None
        for k in range(length):
            p = off(A * one + np.float64(B) * a + np.float64(C) * (a @ a))
            q = p if q is None else off(p @ q)
            if k + 1 < length:
                a = off(off(p @ a) @ p)
        x = q @ x
    return np.asarray(x.T if tall else x, np.float64)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("rows,cols,steps", [(129, 258, 5), (257, 129, 5), (258, 129, 4), (140, 1201, 1), (1201, 140, 2), (140, 1201, 3), (200, 3001, 5),
                                             (513, 1030, 6), (130, 600, 7), (20, 500, 1), (500, 20, 2), (100, 300, 3), (129, 70, 4), (70, 129, 7)])
def test_steps_that_share_a_product(thc, kind, rows, cols, steps):
    """Matrices at least twice as long as high, and those of up to 128 rows: several steps with one X X'. With singular values from 1 to 1e-4 too."""
    odd = steps % 2
    lengths = [2] * (steps // 2) + [1] * odd if kind == "float" or steps == 1 else [3] * odd + [2] * ((steps - 3 * odd) // 2)
    rng = np.random.default_rng(rows + cols + steps)
    m = min(rows, cols)
    u, v = np.linalg.qr(rng.standard_normal((rows, m)))[0], np.linalg.qr(rng.standard_normal((cols, m)))[0]
    for g in (_matrix(rng, rows, cols, kind), ((u * np.logspace(0, -4, m)) @ v.T * 0.5).astype(NP[kind])):
        want = _steps(g, steps)
        assert np.linalg.norm(_chained(g, lengths) - want) <= 2.0 ** -40 * np.linalg.norm(want)
        got = thc.Tensor(kind).orthogonalize(thc.Tensor.from_numpy(g), steps).numpy().astype(np.float64)
        # eight times what rounding did in these steps, in either order, and the rounding to the type
        room = 8 * max(np.linalg.norm(f(g, *how, noise=np.random.default_rng(1)) - want) for f, how in ((_chained, (lengths,)), (_steps, (steps,))))
        beyond = np.maximum(np.abs(got - want) - UNIT[kind] * np.abs(want) * 1.01 - TINY[kind], 0)
        assert np.linalg.norm(beyond) <= room + 2.0 ** -24 * np.linalg.norm(want), np.linalg.norm(beyond) / room


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("rows,cols", [(70, 300), (300, 70), (140, 700), (700, 140), (260, 2000)])
def test_one_element_a_row_of_long_matrices(thc, kind, rows, cols):
    rng = np.random.default_rng(rows + cols)
    m = min(rows, cols)
    g = np.zeros((rows, cols), NP[kind])
    at = rng.permutation(rows)[:m], rng.permutation(cols)[:m]
    values = (rng.choice([-1, 1], m) * np.exp(rng.uniform(-3, 0, m))).astype(NP[kind])
    g[at] = values
    got = thc.Tensor(kind).orthogonalize(thc.Tensor.from_numpy(g)).numpy().astype(np.float64)
    want = _scalar_steps(values.astype(np.float64) / (np.linalg.norm(g.astype(np.float64)) + 1e-7))
    where = np.ones_like(got, bool)
    where[at] = False
    assert np.all(got[where] == 0)
    # 10 roundings a step relative to the value, as where steps go one by one, and those of the shared products: five of an operand for each of three
    # steps more, which a following step makes at most 2.8 of (a^2 of A's relative error against the slope of its square root's)
    assert np.all(np.abs(got[at] - want) <= ((5 * 10 + 3 * 5 * 2.8) * 2.0 ** -22 + UNIT[kind] * 1.01) * np.abs(want) * 1.5), np.max(np.abs(got[at] / want - 1))


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("shape", [(4, 40, 300), (4, 1400, 30), (4, 130, 270), (4, 150, 160)])
def test_not_finite_matrices_of_a_batch(thc, kind, shape):
    rng = np.random.default_rng(sum(shape))
    g = np.stack([_matrix(rng, shape[1], shape[2], kind) for _ in range(4)])
    g[0, -1, -1] = np.nan
    g[1, 0, -1] = np.inf
    g[2] = 0
    t = thc.Tensor.from_numpy
    got = thc.Tensor(kind).orthogonalize(t(g)).numpy()
    assert np.all(np.isnan(got[:2])) and np.all(got[2] == 0)
    assert_bit_equal(got[3], thc.Tensor(kind).orthogonalize(t(g[3])).numpy())


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("rows,cols", [(60, 700), (700, 60), (100, 1900)])
def test_strips_of_other_sizes(thc, kind, rows, cols):
    """Matrices of up to 128 rows go in strips of 128 columns, each first over its own norm: strips of zeros, of tiny and of large elements."""
    rng = np.random.default_rng(rows)
    g = _matrix(rng, min(rows, cols), max(rows, cols), kind).astype(np.float64)
    g[:, :128] *= 2.0 ** -9
    g[:, 128:256] = 0
    g[:, 256:384] *= 2.0 ** 5
    g[:, 640:] *= 2.0 ** -14
    g = np.ascontiguousarray(g if rows < cols else g.T).astype(NP[kind])
    _check(thc.Tensor(kind).orthogonalize(thc.Tensor.from_numpy(g)).numpy(), g, kind)
    if kind == "float":      # far beyond what is left of the result at all
        g.reshape(rows, cols)[(slice(None), slice(640, None)) if rows < cols else slice(640, None)] *= np.float32(2.0 ** -110)
        _check(thc.Tensor(kind).orthogonalize(thc.Tensor.from_numpy(g)).numpy(), g, kind)


@pytest.mark.parametrize("count,rows,cols", [(260, 600, 600), (1150, 200, 400), (1500, 100, 1000), (4000, 30, 3000)])
def test_batches_beyond_a_pass(thc, count, rows, cols):
    """Workspaces of more than 2 GiB in all, of each kind of matrices: the bits of one alone, for each."""
    one = _matrix(np.random.default_rng(rows), rows, cols, "half")
    t = thc.Tensor.from_numpy
    want = thc.Tensor("half").orthogonalize(t(one)).numpy()
    source, many = t(one), thc.Tensor("half").resize((count, rows, cols))
    for i in range(count):
        many.select(0, i).copy(source)
    many.orthogonalize(many)
    got = many.numpy()
    assert_bit_equal(got[0], want)
    assert_bit_equal(got[-1], want)
    assert all(np.array_equal(got[0], x) for x in got)
