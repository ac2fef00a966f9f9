"""The operators of a decoder together: a small model's forward and backward pass and its two optimizers' steps against float64, to the last bit
again on other streams, and replayed from a graph."""
import ctypes as C
import threading

import numpy as np
import pytest

from tests.test_muon_gpu import _steps
from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
EPS = 1e-5


class _Model(object):
    """Rows of a table by token, normalised, turned by their positions in heads, normalised again; the loss is the sum of what comes out times
    given numbers. Muon steps the table, AdamW the norms' weights."""

    def __init__(self, thc, seed=0, vocab=40, heads=3, dim=16, tokens=70, kind="float"):
        rng = np.random.default_rng(seed)
        self.thc, self.kind = thc, kind
        self.real = np.float16 if kind == "half" else np.float32
        self.heads, self.dim, self.width, self.count = heads, dim, heads * dim, tokens
        self.first = [rng.standard_normal((vocab, self.width)), 1 + 0.2 * rng.standard_normal(self.width), 0.1 * rng.standard_normal(self.width),
                      1 + 0.2 * rng.standard_normal(dim)]
        self.first = [x.astype(self.real) for x in self.first]
        t = thc.Tensor.from_numpy
        self.table, self.w1, self.b1, self.w2 = (t(x) for x in self.first)
        self.ids, self.at = rng.integers(1, vocab + 1, tokens), rng.integers(0, 100000, tokens)
        self.tokens, self.positions = t(self.ids), t(self.at)
        self.frequencies = thc.Tensor("double").rotary_frequencies(dim - 4, 500.0)
        self.wanted = rng.standard_normal((tokens, heads, dim)).astype(self.real)
        self.g = t(self.wanted)
        self.x, self.n, self.r, self.y, self.dr, self.dn, self.dx = (thc.Tensor(kind) for _ in range(7))
        self.grads = [thc.Tensor(kind).resize(p.shape).zero() for p in (self.table, self.w1, self.b1, self.w2)]
        self.muon = thc.Muon([self.table], [self.grads[0]], lr=0.05, weight_decay=0.1)
        self.adam = thc.AdamW([self.w1, self.b1, self.w2], self.grads[1:], lr=0.01)

    def as_heads(self, t):
        return t.view_as_strided(t.offset, (self.count, self.heads, self.dim), (self.width, self.dim, 1))

    def as_rows(self, t):
        return t.view_as_strided(t.offset, (self.count, self.width), (self.width, 1))

    def gradients(self):
        self.x.embedding(self.table, self.tokens, 0.5)
        self.n.layer_norm(self.x, self.w1, self.b1, EPS)
        self.r.rotary(self.as_heads(self.n), self.positions, self.frequencies)
        self.y.layer_norm(self.r, self.w2, None, EPS)
        self.dr.layer_norm_grad(self.grads[3], None, self.r, self.g, self.w2, EPS)
        self.dn.rotary(self.dr, self.positions, self.frequencies, inverse=True)
        self.dx.layer_norm_grad(self.grads[1], self.grads[2], self.x, self.as_rows(self.dn), self.w1, EPS)
        self.grads[0].embedding_grad(self.tokens, self.dx, 0.5)
        return [self.y] + self.grads

    def step(self):
        self.gradients()
        self.muon.step()
        self.adam.step()
        return [self.table, self.w1, self.b1, self.w2, self.y, self.muon.momentum[0]]


def _norm(x):
    away = x - x.mean(-1, keepdims=True)
    r = 1 / np.sqrt((away ** 2).mean(-1, keepdims=True) + EPS)
    return away * r, r


def _norm_back(x, gw):
    h, r = _norm(x)
    return r * (gw - gw.mean(-1, keepdims=True) - h * (gw * h).mean(-1, keepdims=True))


def _turn(x, angle):
    n = angle.shape[-1]
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = x[..., :n], x[..., n:2 * n]
    return np.concatenate([a * c - b * s, a * s + b * c, x[..., 2 * n:]], -1)


def _formula(model, params):
    """(output, gradients) in float64."""
    table, w1, b1, w2 = params
    angle = np.outer(model.at, 500.0 ** (-np.arange(0, model.dim - 4, 2) / (model.dim - 4)))
    x = 0.5 * table[model.ids - 1]
    h1, _ = _norm(x)
    r = _turn((h1 * w1 + b1).reshape(model.count, model.heads, model.dim), angle)
    h2, _ = _norm(r)
    g = model.wanted.astype(np.float64)
    dr = _norm_back(r, g * w2)
    dn = _turn(dr, -angle).reshape(model.count, model.width)
    dx = _norm_back(x, dn * w1)
    dt = np.zeros_like(table)
    np.add.at(dt, model.ids - 1, 0.5 * dx)
    return h2 * w2, [dt, (dn * h1).sum(0), dn.sum(0), (g * h2).sum((0, 1))]


def test_gradients(thc):
    model = _Model(thc)
    params = [x.astype(np.float64) for x in model.first]
    y, grads = _formula(model, params)
    got = [t.numpy().astype(np.float64) for t in model.gradients()]
    # five operators of at most a hundred roundings each, of values of a few units over deviations of 0.5 at least
    for a, b in zip(got, [y] + grads):
        assert np.linalg.norm(a - b) <= 2000 * F32 * np.linalg.norm(b)
    # and the formulas by differences of the loss along random directions
    rng = np.random.default_rng(1)
    for k, grad in enumerate(grads):
        d = rng.standard_normal(grad.shape)
        ends = [_formula(model, [p + s * 1e-5 * d if i == k else p for i, p in enumerate(params)])[0] for s in (1, -1)]
        slope = float(((ends[0] - ends[1]) * model.wanted).sum()) / 2e-5
        assert abs(slope - float((grad * d).sum())) <= 1e-5 * float(np.abs(grad * d).sum())


def test_steps(thc):
    model = _Model(thc)
    p = [x.astype(np.float64) for x in model.first]
    momentum = np.zeros_like(p[0])
    m, v = [np.zeros_like(x) for x in p[1:]], [np.zeros_like(x) for x in p[1:]]
    for k in range(1, 4):
        grads = _formula(model, p)[1]
        momentum = np.float32(0.95) * momentum + grads[0]
        p[0] = p[0] * (1 - 0.05 * 0.1) - 0.05 * _steps(grads[0] + np.float32(0.95) * momentum)
        for i in range(3):
            m[i] = 0.9 * m[i] + 0.1 * grads[1 + i]
            v[i] = 0.999 * v[i] + 0.001 * grads[1 + i] ** 2
            p[1 + i] = p[1 + i] * (1 - 0.01 * 0.01) - 0.01 * (m[i] / (1 - 0.9 ** k)) / (np.sqrt(v[i] / (1 - 0.999 ** k)) + 1e-8)
        got = model.step()
        # a step moves by 0.05 of a matrix of about 6 in norm and 0.01 an element; gradients are 2000 roundings off, which Newton-Schulz steps take up to
        # 485 times as far in directions that are hardly there
        assert np.linalg.norm(got[0].numpy() - p[0]) <= k * (0.05 * 485 * 2000 * F32 * 6 + 4 * F32 * np.linalg.norm(p[0]))
        for i in range(3):
            assert np.linalg.norm(got[1 + i].numpy() - p[1 + i]) <= 1e-3 * k * np.linalg.norm(p[1 + i]) * 0.01 + 4 * F32 * k * np.linalg.norm(p[1 + i])


def _hip():
    hip = C.CDLL("libamdhip64.so")
    P = C.c_void_p
    for name, args in (("hipStreamCreate", [C.POINTER(P)]), ("hipStreamSynchronize", [P]), ("hipStreamBeginCapture", [P, C.c_int]),
                       ("hipStreamEndCapture", [P, C.POINTER(P)]), ("hipGraphInstantiate", [C.POINTER(P), P, P, P, C.c_size_t]), ("hipGraphLaunch", [P, P]),
                       ("hipGraphExecDestroy", [P]), ("hipGraphDestroy", [P])):
        getattr(hip, name).argtypes = args
    return hip


@pytest.mark.parametrize("kind", ["float", "half"])
def test_steps_on_streams_of_their_own(thc, kind):
    hip = _hip()
    sizes = dict(vocab=700, heads=5, dim=70, tokens=900, kind=kind)

    def run(model):
        for _ in range(3):
            out = model.step()
        return out

    want = [[x.numpy() for x in run(_Model(thc, seed, **sizes))] for seed in (1, 2)]
    again = [x.numpy() for x in run(_Model(thc, 1, **sizes))]
    for a, b in zip(again, want[0]):
        assert_bit_equal(a, b)
    models = [_Model(thc, seed, **sizes) for seed in (1, 2)]      # made for the default stream, used on others
    thc.synchronize()
    got, errors = [None, None], []

    def worker(i):
        stream = C.c_void_p()
        try:
            assert hip.hipStreamCreate(C.byref(stream)) == 0
            thc.lib().THCState_setCurrentStream(thc.state(), stream)
            out = run(models[i])
            assert hip.hipStreamSynchronize(stream) == 0
            got[i] = [x.numpy() for x in out]
            del out
        except Exception as e:
            errors.append(e)
        finally:
            thc.lib().THCState_setCurrentStream(thc.state(), None)

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in range(2):
        for k, (a, b) in enumerate(zip(got[i], want[i])):
            assert_bit_equal(a, b, "model %d, output %d" % (i, k))


def test_replays_from_a_graph(thc):
    """Norms and turns that take no memory are captured; replays follow what their operands hold. What takes memory refuses."""
    hip = _hip()
    rng = np.random.default_rng(3)
    rows, heads, dim = 50, 4, 40
    t = thc.Tensor.from_numpy
    first = [rng.standard_normal((rows, heads * dim)).astype(np.float32) for _ in range(4)]
    x, w, b, g = t(first[0]), t(first[1][0]), t(first[2][0]), t(first[3])
    at, f = t(rng.integers(0, 5000, rows)), thc.Tensor("double").rotary_frequencies(dim)
    y, r, dx = (thc.Tensor("float").resize((rows, heads * dim)) for _ in range(3))
    turned = r.view_as_strided(0, (rows, heads, dim), (heads * dim, dim, 1))
    source = y.view_as_strided(0, (rows, heads, dim), (heads * dim, dim, 1))

    def work():
        y.layer_norm(x, w, b)
        turned.rotary(source, at, f)
        dx.layer_norm_grad(None, None, x, r, w)

    square, small = thc.Tensor("float").resize((20, 30)).fill(1), thc.Tensor("float").resize((20, 30)).fill(1)
    sums = thc.Tensor("float").resize((heads * dim,))
    muon = thc.Muon([square], [small])
    refused = (lambda: thc.Tensor("float").layer_norm(x.t()), lambda: dx.layer_norm_grad(sums, None, x, r, w), lambda: small.orthogonalize(square),
               lambda: muon.step(), lambda: r.layer_norm(x, x.select(1, 0).view_as_strided(0, (heads * dim,), (2,))),
               lambda: r.view_as_strided(0, (heads, dim, rows), (dim, 1, heads * dim)).t(0, 2).t(1, 2).rotary(source.t(0, 1).t(0, 1), at, f.view_as_strided(0, (10,), (2,))))
    work()
    thc.synchronize()
    stream, graph, program = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    thc.lib().THCState_setCurrentStream(thc.state(), stream)
    try:
        assert hip.hipStreamBeginCapture(stream, 2) == 0      # (relaxed: other threads and streams go on)
        try:
            work()
            for call in refused:
                with pytest.raises(thc.THCError, match="cannot be captured"):
                    call()
        finally:
            assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(program), graph, None, None, 0) == 0
        for k in range(4):
            x.copy(t((first[0] * (k + 1) + k).astype(np.float32)))
            at.copy(t(rng.integers(0, 5000, rows)))
            for out in (y, r, dx):
                out.fill(-7)
            assert hip.hipStreamSynchronize(stream) == 0
            assert hip.hipGraphLaunch(program, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            got = [o.numpy() for o in (y, r, dx)]
            for out in (y, r, dx):
                out.fill(-7)
            work()
            assert hip.hipStreamSynchronize(stream) == 0
            for a, o in zip(got, (y, r, dx)):
                assert_bit_equal(a, o.numpy(), "replay %d" % k)
    finally:
        thc.lib().THCState_setCurrentStream(thc.state(), None)
        thc.synchronize()
        if program:
            hip.hipGraphExecDestroy(program)
        if graph:
            hip.hipGraphDestroy(graph)      # (the stream stays: the allocator waits for it before it hands out again what was used on it)
