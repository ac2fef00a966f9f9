"""AdamW over lists of tensors: bit for bit against the same operations in numpy, and against the formulas in float64."""
import numpy as np
import pytest

from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
NP = {"float": np.float32, "half": np.float16}
HYPER = dict(lr=2e-3, beta1=0.9, beta2=0.97, eps=1e-7, weight_decay=0.05)


def _f(x):
    return np.float32(x)


def _numpy_step(p, g, m, v, step, scale, h=HYPER):
    """The step in float32, one rounding an operation."""
    with np.errstate(all="ignore"):
        g = g.astype(np.float32) * _f(scale)
        m = m * _f(h["beta1"]) + g * _f(1 - h["beta1"])
        v = v * _f(h["beta2"]) + (g * g) * _f(1 - h["beta2"])
        root = np.sqrt(v) * _f(1 / np.sqrt(1 - h["beta2"] ** step)) + _f(h["eps"])
        return p * _f(1 - h["lr"] * h["weight_decay"]) - (m / root) * _f(h["lr"] / (1 - h["beta1"] ** step)), m, v


def _blocks(x):
    return np.concatenate([x, np.zeros(-x.size % 256, x.dtype)]).reshape(-1, 256)


def _numpy_codes(m, v):
    """8-bit states of float32 moments: codes of their sizes, and the blocks' largest magnitudes."""
    n, shape = m.size, m.shape
    bm, bv = _blocks(m.reshape(-1)), _blocks(v.reshape(-1))
    tm, tv = np.abs(bm).max(1), bv.max(1)
    im, iv = [np.where(t > 0, _f(1) / np.where(t > 0, t, 1), _f(0)).astype(np.float32)[:, None] for t in (tm, tv)]
    cm = np.rint(np.sqrt(np.abs(bm) * im) * _f(127)) * np.sign(bm)
    share = bv * iv
    cv = np.rint(np.sqrt(np.sqrt(share)) * _f(255))
    cv = np.where(share > 0, np.maximum(cv, 1), cv)
    return (cm.reshape(-1)[:n].reshape(shape).astype(np.int8), tm, cv.reshape(-1)[:n].reshape(shape).astype(np.uint8), tv)


def _numpy_values(cm, tm, cv, tv):
    n, shape = cm.size, cm.shape
    t = cm.reshape(-1).astype(np.float32) * _f(1 / 127)
    m = (t * np.abs(t)) * np.repeat(tm, 256)[:n]
    t = cv.reshape(-1).astype(np.float32) * _f(1 / 255)
    t = t * t
    return m.reshape(shape), ((t * t) * np.repeat(tv, 256)[:n]).reshape(shape)


SHAPES = {"one": [(1,)], "ragged": [(255,), (256,), (257,), (3, 5), (1,), (1023,), (7, 11, 13), (4096,), (4097,)],
          "many": [(1 + 37 * i % 600,) for i in range(230)], "large": [(1000, 1003), (5,)]}


def _problem(rng, shapes, kind, grad_mass=1.0):
    p = [(0.1 * rng.standard_normal(s)).astype(NP[kind]) for s in shapes]
    g = [(grad_mass * rng.standard_normal(s) * 10.0 ** rng.uniform(-3, 0)).astype(NP[kind]) for s in shapes]
    return p, g


def _put(thc, arrays):
    return [thc.Tensor.from_numpy(a) for a in arrays]


@pytest.mark.parametrize("shapes", sorted(SHAPES))
@pytest.mark.parametrize("kind,master", [("float", False), ("half", False), ("half", True)])
def test_steps(thc, shapes, kind, master):
    rng = np.random.default_rng(len(shapes))
    p, g = _problem(rng, SHAPES[shapes], kind)
    copies = [a.astype(np.float32) + _f(1e-5) for a in p] if master else None
    dp, dg, dm = _put(thc, p), _put(thc, g), _put(thc, copies) if master else None
    opt = thc.AdamW(dp, dg, master=dm, **HYPER)
    m, v = [np.zeros(a.shape, np.float32) for a in p], [np.zeros(a.shape, np.float32) for a in p]
    for step in range(1, 4):
        opt.step(0.5)
        assert thc.last_kernel() == "adamw"
        for i in range(len(p)):
            q, m[i], v[i] = _numpy_step(copies[i] if master else p[i].astype(np.float32), g[i], m[i], v[i], step, 0.5)
            if master:
                copies[i] = q
            p[i] = q.astype(NP[kind])
    for i in range(len(p)):
        assert_bit_equal(dp[i].numpy(), p[i], "parameter %d" % i)
        assert_bit_equal(opt.mean[i].numpy(), m[i], "mean %d" % i)
        assert_bit_equal(opt.square[i].numpy(), v[i], "square %d" % i)
        if master:
            assert_bit_equal(dm[i].numpy(), copies[i], "copy %d" % i)


@pytest.mark.parametrize("shapes", sorted(SHAPES))
@pytest.mark.parametrize("kind,master", [("float", False), ("half", False), ("half", True)])
def test_steps_with_8_bit_states(thc, shapes, kind, master):
    rng = np.random.default_rng(len(shapes) + 7)
    p, g = _problem(rng, SHAPES[shapes], kind)
    copies = [a.astype(np.float32) for a in p] if master else None
    dp, dg, dm = _put(thc, p), _put(thc, g), _put(thc, copies) if master else None
    opt = thc.AdamW(dp, dg, master=dm, bits=8, **HYPER)
    states = [_numpy_codes(np.zeros(a.shape, np.float32), np.zeros(a.shape, np.float32)) for a in p]
    for step in range(1, 4):
        opt.step()
        assert thc.last_kernel() == "adamw8"
        for i in range(len(p)):
            q, m, v = _numpy_step(copies[i] if master else p[i].astype(np.float32), g[i], *_numpy_values(*states[i]), step, 1.0)
            states[i] = _numpy_codes(m, v)
            if master:
                copies[i] = q
            p[i] = q.astype(NP[kind])
    mean, square = opt.moments()
    for i in range(len(p)):
        assert_bit_equal(dp[i].numpy(), p[i], "parameter %d" % i)
        for got, want in zip((opt.mean, opt.mean_scale, opt.square, opt.square_scale), states[i]):
            assert np.array_equal(got[i].numpy(), want), i
        m, v = _numpy_values(*states[i])
        assert_bit_equal(mean[i].numpy(), m)
        assert_bit_equal(square[i].numpy(), v)


@pytest.mark.parametrize("step", [1, 2, 1000, 10 ** 7])
def test_one_step_against_the_formulas_in_float64(thc, step):
    rng = np.random.default_rng(step)
    p, g, m = (rng.standard_normal(3001).astype(np.float32) for _ in range(3))
    v = (rng.standard_normal(3001) ** 2).astype(np.float32)
    t = [thc.Tensor.from_numpy(a) for a in (p, g, m, v)]
    thc.AdamW([t[0]], [t[1]], mean=[t[2]], square=[t[3]], step=step - 1, **HYPER).step(0.25)
    h = HYPER
    g64, eps = g.astype(np.float64) * 0.25, 2.0 ** -24
    m1 = h["beta1"] * m + (1 - h["beta1"]) * g64
    v1 = h["beta2"] * v + (1 - h["beta2"]) * g64 ** 2
    update = h["lr"] * m1 / (1 - h["beta1"] ** step) / (np.sqrt(v1 / (1 - h["beta2"] ** step)) + h["eps"])
    want = p * (1 - h["lr"] * h["weight_decay"]) - update
    # each operand is rounded, each operation too: three for the moments, eleven on the way to the update
    part = h["beta1"] * np.abs(m) + (1 - h["beta1"]) * np.abs(g64)
    assert np.all(np.abs(t[2].numpy() - m1) <= 4 * eps * part)
    assert np.all(np.abs(t[3].numpy() - v1) <= 6 * eps * v1)
    lost = 4 * eps * part / np.maximum(np.abs(m1), 1e-30) + 12 * eps
    assert np.all(np.abs(t[0].numpy() - want) <= np.abs(update) * lost + 4 * eps * (np.abs(p) + np.abs(update)))


def test_8_bit_states_are_near_what_they_stand_for(thc):
    """Values come back within half a code's step: 1/127 of the root of their share of the largest, 1/255 of the fourth root, and a rounding."""
    rng = np.random.default_rng(3)
    g = (rng.standard_normal(5000) * 10.0 ** rng.uniform(-4, 0, 5000)).astype(np.float32)
    p = thc.Tensor.from_numpy(np.zeros(5000, np.float32))
    opt = thc.AdamW([p], [thc.Tensor.from_numpy(g)], bits=8, **HYPER)
    opt.step()
    mean, square = [x[0].numpy().astype(np.float64) for x in opt.moments()]
    m, v = 0.1 * g.astype(np.float64), 0.03 * g.astype(np.float64) ** 2
    for got, want, codes, power in ((mean, m, 127, 2), (square, v, 255, 4)):
        top = np.repeat(np.abs(_blocks(want)).max(1), 256)[:5000]
        off = np.abs((np.abs(got) / top) ** (1 / power) - (np.abs(want) / top) ** (1 / power))
        held = np.maximum((np.abs(want) / top) ** (1 / power), 1 / codes if power == 4 else 0)      # a square's code is 1 at least
        off = np.minimum(off, np.abs((np.abs(got) / top) ** (1 / power) - held))
        assert np.all(off <= 0.5 / codes + 1e-5)
        assert np.all((got == 0) | (np.sign(got) == np.sign(want)))
    assert np.all(square[v > 1e-30] > 0)


def test_states_in_8_bits_train_like_those_in_32(thc):
    """A least-squares problem: both come down to the same loss within a few percent of where it began."""
    rng = np.random.default_rng(4)
    target = rng.standard_normal(2000).astype(np.float32) * 10.0 ** rng.uniform(-2, 0, 2000).astype(np.float32)
    loss = {}
    for bits in (8, 32):
        p, g, t = thc.Tensor.from_numpy(np.zeros(2000, np.float32)), thc.Tensor("float").resize((2000,)), thc.Tensor.from_numpy(target)
        opt = thc.AdamW([p], [g], lr=0.02, weight_decay=0.0, beta2=0.99, bits=bits)
        for _ in range(300):
            g.csub(p, 1, t)
            opt.step()
        loss[bits] = float(np.mean((p.numpy() - target) ** 2) / np.mean(target ** 2))
    assert loss[32] < 1e-2 and loss[8] < 3e-2, loss


@pytest.mark.parametrize("bits", [8, 32])
def test_strided_tensors(thc, bits):
    rng = np.random.default_rng(5)
    p, g = rng.standard_normal((40, 30)).astype(np.float32), rng.standard_normal((30, 40)).astype(np.float32)
    room = np.full((45, 33), 5, np.float32)
    room[2:42, 1:31] = p
    base, turned = thc.Tensor.from_numpy(room), thc.Tensor.from_numpy(g)
    plain, grad = thc.Tensor.from_numpy(p), thc.Tensor.from_numpy(np.ascontiguousarray(g.T))
    one = thc.AdamW([base.narrow(0, 2, 40).narrow(1, 1, 30)], [turned.t()], bits=bits, **HYPER)
    other = thc.AdamW([plain], [grad], bits=bits, **HYPER)
    # states that are views: of every second column of something wider
    one.mean = [thc.Tensor(one.mean[0].kind).resize((40, 60)).zero().view_as_strided(0, (40, 30), (60, 2))]
    one = thc.AdamW(one.params, one.grads, bits=bits, mean=one.mean, **HYPER)
    for _ in range(2):
        one.step()
        other.step()
    room[2:42, 1:31] = plain.numpy()
    assert_bit_equal(base.numpy(), room)
    assert np.array_equal(one.mean[0].numpy(), other.mean[0].numpy())


def test_offsets_off_the_16_byte_grid(thc):
    rng = np.random.default_rng(6)
    for kind, bits in (("float", 32), ("half", 32), ("float", 8), ("half", 8)):
        flat = [rng.standard_normal(5000).astype(NP[kind]) for _ in range(2)]
        big = [thc.Tensor.from_numpy(a) for a in flat]
        for at, n in ((1, 1000), (1003, 257), (1261, 3), (1267, 2049)):
            parts = [b.narrow(0, at, n) for b in big]
            plain = [thc.Tensor.from_numpy(a[at:at + n]) for a in flat]
            states = [thc.Tensor(k).resize((n + 3,)).zero().narrow(0, 3, n) for k in (("char", "byte") if bits == 8 else ("float", "float"))]
            thc.AdamW([parts[0]], [parts[1]], mean=[states[0]], square=[states[1]], bits=bits, **HYPER).step()
            thc.AdamW([plain[0]], [plain[1]], bits=bits, **HYPER).step()
            flat[0][at:at + n] = plain[0].numpy()
        assert_bit_equal(big[0].numpy(), flat[0])
        assert_bit_equal(big[1].numpy(), flat[1])


def test_values_that_are_not_finite_stay_where_they_are(thc):
    g = np.ones(1000, np.float32)
    g[10], g[300], g[600] = np.nan, np.inf, 0
    for bits, poisoned in ((32, [10, 300]), (8, None)):
        p = thc.Tensor.from_numpy(np.ones(1000, np.float32))
        opt = thc.AdamW([p], [thc.Tensor.from_numpy(g)], bits=bits, **HYPER)
        opt.step()
        got = p.numpy()
        assert sorted(np.flatnonzero(~np.isfinite(got))) == [10, 300]
        opt.grads[0].fill(1)
        opt.step()
        bad = np.flatnonzero(~np.isfinite(p.numpy()))
        if bits == 32:
            assert sorted(bad) == poisoned
        else:         # the blocks that held them, no others
            assert set(bad) <= set(range(512)) and {10, 300} <= set(bad)
    # zero gradients on zero states move nothing but by the decay
    p = thc.Tensor.from_numpy(np.ones(700, np.float32))
    opt = thc.AdamW([p], [thc.Tensor.from_numpy(np.zeros(700, np.float32))], bits=8, **HYPER)
    opt.step()
    assert np.all(p.numpy() == _f(1) * _f(1 - HYPER["lr"] * HYPER["weight_decay"]))


def test_refusals(thc):
    def new(kind="float", shape=(4, 3)):
        return thc.Tensor(kind).resize(shape).zero()

    with pytest.raises(thc.THCError, match="other sizes than its parameter"):
        thc.AdamW([new()], [new(shape=(3, 4))]).step()
    with pytest.raises(thc.THCError, match="1 scales for the 2 blocks"):
        thc.AdamW([new(shape=(300,))], [new(shape=(300,))], bits=8, mean_scale=[new(shape=(1,))]).step()
    with pytest.raises(thc.THCError, match="beta2"):
        thc.AdamW([new()], [new()], beta2=1.0).step()
    with pytest.raises(thc.THCError, match="beta1"):
        thc.AdamW([new()], [new()], beta1=-0.1).step()
    with pytest.raises(thc.THCError, match="eps"):
        thc.AdamW([new()], [new()], eps=-1e-8).step()
    with pytest.raises(thc.THCError, match="counted from 1"):
        thc.AdamW([new()], [new()], step=-1).step()
    with pytest.raises(thc.THCError, match="overlap"):
        p = new().view_as_strided(0, (4, 3), (0, 1))
        thc.AdamW([p], [new()]).step()
    with pytest.raises(thc.THCError, match="scales of tensor 1's states overlap"):
        thc.AdamW([new(shape=(300,))], [new(shape=(300,))], bits=8, mean_scale=[new(shape=(1,)).view_as_strided(0, (2,), (0,))]).step()
    for bad in (dict(params=[new("half"), new()], grads=[new(), new()]), dict(params=[new()], grads=[]), dict(params=[new()], grads=[new("half")]),
                dict(params=[new()], grads=[new()], master=[new()]), dict(params=[new()], grads=[new()], bits=16)):
        with pytest.raises(ValueError):
            thc.AdamW(**bad)
    thc.AdamW([], []).step()         # nothing to do
    thc.AdamW([thc.Tensor("float")], [thc.Tensor("float")], bits=8).step()


def test_moments_in_windows_of_one_storage(thc):
    """Outputs that share a storage, which grows for the second one."""
    rng = np.random.default_rng(8)
    p, g = _problem(rng, [(300,), (7, 100)], "float")
    opt = thc.AdamW(_put(thc, p), _put(thc, g), bits=8, **HYPER)
    opt.step()
    want = [[t.numpy() for t in l] for l in opt.moments()]
    room = thc.Tensor("float").resize((350,)).zero()
    mean, square = opt.moments([room.narrow(0, 0, 300), thc.Tensor("float")], [thc.Tensor("float"), room.narrow(0, 300, 50)])
    for a, b in zip(mean + square, want[0] + want[1]):
        assert_bit_equal(a.numpy(), b)
    with pytest.raises(thc.THCError, match="two moments share memory"):
        opt.moments([room, thc.Tensor("float")], [room, thc.Tensor("float")])
    with pytest.raises(thc.THCError, match="lies on its scales"):
        opt.moments([opt.mean_scale[0], thc.Tensor("float")], [thc.Tensor("float"), thc.Tensor("float")])
