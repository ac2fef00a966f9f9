"""Embedding lookup and its gradient against float64, at the sizes where rows end inside a pack, tokens fill one group or cross
many, and tables are seen through views."""
import numpy as np
import pytest

from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
NP = {"float": np.float32, "half": np.float16}


def _tensor(thc, a, kind=None):
    return thc.Tensor.from_numpy(a, kind)


def _table(rng, vocab, dim, kind):
    return rng.standard_normal((vocab, dim)).astype(NP[kind])


def _lookup(table, tokens, f):
    """One rounding of the product, NaN rows for tokens outside."""
    inside = (tokens >= 1) & (tokens <= table.shape[0])
    rows = table[np.where(inside, tokens - 1, 0)].astype(np.float32) * np.float32(f)
    rows = np.where(inside[..., None], rows, np.float32(np.nan))
    return rows.astype(table.dtype)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("dim", [1, 3, 4, 7, 8, 9, 63, 64, 513, 2048])
@pytest.mark.parametrize("count", [1, 2, 65, 1000])
def test_lookup(thc, kind, dim, count):
    rng = np.random.default_rng(dim * 1000 + count)
    table = _table(rng, 77, dim, kind)
    tokens = rng.integers(1, 78, count)
    got = thc.Tensor(kind).embedding(_tensor(thc, table), _tensor(thc, tokens), 1.7)
    assert thc.last_kernel() == "embedding"
    assert_bit_equal(got.numpy(), _lookup(table, tokens, 1.7))


@pytest.mark.parametrize("kind", ["float", "half"])
def test_lookup_views(thc, kind):
    rng = np.random.default_rng(5)
    wide = _table(rng, 40, 50, kind)
    tokens = rng.integers(1, 41, (6, 7))
    w, t = _tensor(thc, wide), _tensor(thc, tokens)
    # a window of the table's columns, a transposed table, transposed tokens
    assert_bit_equal(thc.Tensor(kind).embedding(w.narrow(1, 3, 41), t, 1.0).numpy(), _lookup(wide[:, 3:44], tokens, 1))
    short = np.minimum(tokens, 50)
    assert_bit_equal(thc.Tensor(kind).embedding(w.t(), _tensor(thc, short), 2.0).numpy(), _lookup(np.ascontiguousarray(wide.T), short, 2))
    got = thc.Tensor(kind).embedding(w, t.t(), 0.5)
    assert got.shape == (7, 6, 50)
    assert_bit_equal(got.numpy(), _lookup(wide, tokens.T, 0.5))
    # an output that is a window of something larger keeps what is around it
    room = thc.Tensor(kind).resize((42, 60)).fill(9)
    room.narrow(1, 4, 50).embedding(w, _tensor(thc, tokens.reshape(-1)), 1.0)
    want = np.full((42, 60), 9, NP[kind])
    want[:, 4:54] = _lookup(wide, tokens.reshape(-1), 1)
    assert_bit_equal(room.numpy(), want)
    # and one that lies on the table's own storage
    both = thc.Tensor.from_numpy(np.concatenate([wide, wide]))
    both.narrow(0, 20, 42).embedding(both.narrow(0, 0, 40), _tensor(thc, tokens.reshape(-1)), 1.0)
    assert_bit_equal(both.numpy()[20:62], _lookup(wide, tokens.reshape(-1), 1))


@pytest.mark.parametrize("kind", ["float", "half"])
def test_lookup_outside_and_in_pieces(thc, kind):
    rng = np.random.default_rng(6)
    table = _table(rng, 9, 33, kind)
    tokens = np.array([1, 0, 9, 10, -1, 5, 2 ** 40, -2 ** 62, 3])
    for items in (1 << 30, 20, 1):      # as much as one launch takes
        thc.set_tuning("embedding.items", items)
        try:
            got = thc.Tensor(kind).embedding(_tensor(thc, table), _tensor(thc, tokens), 3.0).numpy()
        finally:
            thc.set_tuning("embedding.items", 1 << 30)
        want = _lookup(table, tokens, 3.0)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])


def _sums(shape, tokens, out, f, padding, start=None):
    """float64 sums, and the magnitude and number of what went into each."""
    vocab, dim = shape
    flat, rows = tokens.reshape(-1), out.reshape(-1, dim).astype(np.float64)
    used = (flat >= 1) & (flat <= vocab) & (flat != padding)
    total, mass, count = np.zeros(shape), np.zeros(shape), np.zeros(vocab)
    np.add.at(total, flat[used] - 1, rows[used])
    np.add.at(mass, flat[used] - 1, np.abs(rows[used]))
    np.add.at(count, flat[used] - 1, 1)
    total, mass = total * np.float32(f), mass * abs(np.float32(f))
    if start is not None:
        total, mass = total + start, mass + np.abs(start)
    return total, mass, count


def _near(got, want, mass, count, kind):
    """Sums of n floats in any order are off by n 2^-24 of their mass at most; the product and the added start round once each, a half
    result once more."""
    bound = (count[:, None] + 2) * 2.0 ** -24 * mass
    if kind == "half":
        bound = bound + 2.0 ** -11 * np.abs(want) * (1 + 2.0 ** -10) + 2.0 ** -25
    off = np.abs(got.astype(np.float64) - want)
    assert np.all(off <= bound), (float(np.max(off - bound)), np.argwhere(off > bound)[:3])


def _tokens(rng, how, vocab, count):
    if how == "one":
        return np.full(count, 1 + vocab // 2)
    if how == "two":
        return np.where(rng.random(count) < 0.9, 1, vocab)
    if how == "each":
        return rng.permutation(np.arange(count) % vocab) + 1
    return np.minimum(vocab, np.exp(rng.random(count) * np.log(vocab + 1)).astype(np.int64))


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("how", ["text", "one", "two", "each"])
@pytest.mark.parametrize("vocab,dim,count", [(1, 1, 1), (1, 8, 300), (7, 3, 1), (7, 5, 64), (300, 4, 129), (300, 17, 1000), (257, 64, 2000),
                                             (1000, 130, 700), (5003, 513, 515), (255, 1025, 333)])
@pytest.mark.parametrize("add", [False, True])
def test_gradient(thc, kind, how, vocab, dim, count, add):
    rng = np.random.default_rng(vocab + dim + count)
    tokens = _tokens(rng, how, vocab, count)
    out = rng.standard_normal((count, dim)).astype(NP[kind])
    start = _table(rng, vocab, dim, kind)
    grad = _tensor(thc, start)
    grad.embedding_grad(_tensor(thc, tokens), _tensor(thc, out), 0.75, accumulate=add)
    assert thc.last_kernel() == "embedding-grad"
    want, mass, n = _sums((vocab, dim), tokens, out, 0.75, 0, start.astype(np.float64) if add else None)
    got = grad.numpy()
    _near(got, want, mass, n, kind)
    if add:       # rows without a token keep their bits
        assert_bit_equal(got[n == 0], start[n == 0])
    else:
        assert not got[n == 0].any()
    again = _tensor(thc, start)
    again.embedding_grad(_tensor(thc, tokens), _tensor(thc, out), 0.75, accumulate=add)
    assert_bit_equal(again.numpy(), got)
    thc.set_tuning("embedding.few", 0)       # as many positions are summed
    try:
        again = _tensor(thc, start)
        again.embedding_grad(_tensor(thc, tokens), _tensor(thc, out), 0.75, accumulate=add)
    finally:
        thc.set_tuning("embedding.few", 3 << 20)
    _near(again.numpy(), want, mass, n, kind)


@pytest.fixture
def split(thc):
    """Positions are split between their owners first, as those of many tokens are."""
    thc.set_tuning("embedding.split", 0)
    thc.set_tuning("embedding.few", 0)
    yield
    thc.set_tuning("embedding.split", 40000)
    thc.set_tuning("embedding.few", 3 << 20)


@pytest.mark.parametrize("how", ["text", "one", "two", "each"])
@pytest.mark.parametrize("vocab,dim,count", [(1, 1, 1), (2, 3, 4096), (7, 5, 64), (300, 17, 1000), (5003, 64, 4097), (255, 9, 8191),
                                             (131073, 4, 12289), (262144, 3, 9000), (524288, 2, 20000), (524289, 2, 5000), (300, 5, 70000)])
def test_gradient_of_split_positions(thc, split, how, vocab, dim, count):
    rng = np.random.default_rng(vocab + count)
    tokens = _tokens(rng, how, vocab, count)
    tokens[rng.random(count) < 0.02] = 0
    out = rng.standard_normal((count, dim)).astype(np.float32)
    start = _table(rng, vocab, dim, "float")
    for add in (False, True):
        grad = _tensor(thc, start)
        grad.embedding_grad(_tensor(thc, tokens), _tensor(thc, out), 0.5, padding=vocab // 2, accumulate=add)
        want, mass, n = _sums((vocab, dim), tokens, out, 0.5, vocab // 2, start.astype(np.float64) if add else None)
        _near(grad.numpy(), want, mass, n, "float")


WAYS = {"positions": {"embedding.few": 3 << 20, "embedding.own": 0}, "owners": {"embedding.few": 0, "embedding.own": 1 << 40},
        "three": {"embedding.few": 0, "embedding.own": 0}, "split": {"embedding.few": 0, "embedding.own": 0, "embedding.split": 0}}


@pytest.fixture(params=sorted(WAYS))
def way(thc, request):
    """A launch of positions, a launch of owners, three launches, and those after a split: where the sizes allow it."""
    for key, value in WAYS[request.param].items():
        thc.set_tuning(key, value)
    yield request.param
    for key, value in (("embedding.few", 3 << 20), ("embedding.own", 4 << 20), ("embedding.split", 40000)):
        thc.set_tuning(key, value)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("how", ["text", "one", "two", "each"])
@pytest.mark.parametrize("vocab,dim,count", [(1, 1, 2), (2, 3, 4096), (3, 9, 513), (255, 31, 511), (513, 33, 1025), (1000, 7, 4095), (5003, 8, 2049),
                                             (300, 513, 900), (100000, 16, 3000), (262144, 4, 1500), (40, 1030, 4000), (262145, 4, 100)])
def test_gradient_in_every_way(thc, way, kind, how, vocab, dim, count):
    rng = np.random.default_rng(vocab + dim + count)
    tokens = _tokens(rng, how, vocab, count)
    tokens[rng.random(count) < 0.02] = vocab + 1
    padding = 1 if vocab > 2 else 0
    out = rng.standard_normal((count, dim + 3)).astype(NP[kind])
    start = _table(rng, vocab, dim + 5, kind)
    for add in (False, True):
        # windows of something wider: what is around the gradient stays
        room = _tensor(thc, start)
        room.narrow(1, 2, dim).embedding_grad(_tensor(thc, tokens), _tensor(thc, out).narrow(1, 1, dim), 1.25, padding=padding, accumulate=add)
        got = room.numpy()
        want, mass, n = _sums((vocab, dim), tokens, np.ascontiguousarray(out[:, 1:dim + 1]), 1.25, padding,
                              start[:, 2:dim + 2].astype(np.float64) if add else None)
        _near(got[:, 2:dim + 2], want, mass, n, kind)
        keeps = np.ascontiguousarray(start) if add else np.where((np.arange(dim + 5) < 2) | (np.arange(dim + 5) >= dim + 2), start, 0).astype(NP[kind])
        assert_bit_equal(got[n == 0], keeps[n == 0])
        assert_bit_equal(got[:, :2], start[:, :2])
        assert_bit_equal(got[:, dim + 2:], start[:, dim + 2:])
        again = _tensor(thc, start)
        again.narrow(1, 2, dim).embedding_grad(_tensor(thc, tokens), _tensor(thc, out).narrow(1, 1, dim), 1.25, padding=padding, accumulate=add)
        assert_bit_equal(again.numpy(), got)


@pytest.mark.parametrize("vocab,count", [(262143, 5000), (300001, 4099), (1 << 20, 1000)])
def test_gradient_of_a_large_table(thc, vocab, count):
    rng = np.random.default_rng(vocab)
    tokens = np.concatenate([_tokens(rng, "text", vocab, count), [1, vocab, vocab, vocab - 1]])
    out = rng.standard_normal((count + 4, 3)).astype(np.float32)
    grad = _tensor(thc, np.ones((vocab, 3), np.float32))
    grad.embedding_grad(_tensor(thc, tokens), _tensor(thc, out))
    want, mass, n = _sums((vocab, 3), tokens, out, 1, 0)
    _near(grad.numpy(), want, mass, n, "float")


@pytest.mark.parametrize("count", [40000, 70001])
def test_gradient_of_many_tokens(thc, count):
    rng = np.random.default_rng(count)
    tokens = _tokens(rng, "text", 2000, count)
    out = rng.standard_normal((count, 40)).astype(np.float16)
    grad = _tensor(thc, np.ones((2000, 40), np.float16))
    grad.embedding_grad(_tensor(thc, tokens), _tensor(thc, out), 0.01, padding=2)
    want, mass, n = _sums((2000, 40), tokens, out, 0.01, 2)
    _near(grad.numpy(), want, mass, n, "half")


@pytest.mark.parametrize("how", ["one", "two"])
def test_gradient_of_one_common_token(thc, how):
    """Its positions are more than a workgroup keeps between its sweeps, its run crosses hundreds of chunks."""
    rng = np.random.default_rng(13)
    tokens = _tokens(rng, how, 3000, 30011)
    out = rng.standard_normal((30011, 9)).astype(np.float32)
    grad = _tensor(thc, np.ones((3000, 9), np.float32))
    grad.embedding_grad(_tensor(thc, tokens), _tensor(thc, out))
    want, mass, n = _sums((3000, 9), tokens, out, 1, 0)
    _near(grad.numpy(), want, mass, n, "float")


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("add", [False, True])
def test_gradient_leaves_out_padding_and_tokens_outside(thc, kind, add):
    rng = np.random.default_rng(8)
    tokens = rng.integers(-2, 14, (9, 30))
    tokens[0, :3] = [2 ** 40, -2 ** 60, 12]
    out = rng.standard_normal((9, 30, 21)).astype(NP[kind])
    out[tokens == 4] = np.nan
    out[tokens > 11] = np.inf
    start = _table(rng, 11, 21, kind)
    grad = _tensor(thc, start)
    grad.embedding_grad(_tensor(thc, tokens), _tensor(thc, out), 2.0, padding=4, accumulate=add)
    clean = np.where(np.isfinite(out), out, 0)
    want, mass, n = _sums((11, 21), tokens, clean, 2.0, 4, start.astype(np.float64) if add else None)
    _near(grad.numpy(), want, mass, n, kind)
    # nothing but padding
    grad.embedding_grad(_tensor(thc, np.full(50, 4)), _tensor(thc, np.full((50, 21), np.nan, NP[kind])), 1.0, padding=4, accumulate=add)
    if not add:
        assert not grad.numpy().any()


def test_gradient_views(thc):
    rng = np.random.default_rng(9)
    tokens = rng.integers(1, 13, (8, 10))
    wide = rng.standard_normal((8, 10, 30)).astype(np.float32)
    o, t = _tensor(thc, wide), _tensor(thc, tokens)
    for view, plain, toks, handle in ((o.narrow(2, 5, 19), wide[:, :, 5:24], tokens, t), (o.t(0, 1).narrow(2, 0, 19), wide.transpose(1, 0, 2)[:, :, :19], tokens.T, t.t()),
                                      (o.narrow(1, 2, 7).narrow(2, 1, 19), wide[:, 2:9, 1:20], tokens[:, 2:9], t.narrow(1, 2, 7))):
        room = thc.Tensor.from_numpy(np.full((14, 25), 7, np.float32))
        room.narrow(0, 1, 12).narrow(1, 2, 19).embedding_grad(handle, view, 1.0)
        want, mass, n = _sums((12, 19), np.ascontiguousarray(toks), np.ascontiguousarray(plain), 1.0, 0)
        got = room.numpy()
        _near(got[1:13, 2:21], want, mass, n, "float")
        around = got.copy()
        around[1:13, 2:21] = 7
        assert np.all(around == 7)
        # a transposed table's gradient
        turned = thc.Tensor.from_numpy(np.ones((19, 12), np.float32))
        turned.t().embedding_grad(handle, view, 1.0, accumulate=True)
        _near(turned.numpy().T, want + 1, mass + 1, n, "float")


def test_gradient_is_that_of_the_lookup(thc):
    """<dY, lookup(W + h D) - lookup(W - h D)> / 2h = <dW, D>: the lookup is linear, so the difference is exact but for rounding."""
    rng = np.random.default_rng(10)
    table, move = _table(rng, 50, 12, "float"), _table(rng, 50, 12, "float")
    tokens, out = rng.integers(1, 51, 200), rng.standard_normal((200, 12)).astype(np.float32)
    t = _tensor(thc, tokens)
    ends = [thc.Tensor("float").embedding(_tensor(thc, (table + s * move).astype(np.float32)), t, 1.5).numpy().astype(np.float64) for s in (1, -1)]
    differ = np.sum(out * (ends[0] - ends[1])) / 2
    grad = _tensor(thc, table)
    grad.embedding_grad(t, _tensor(thc, out), 1.5)
    along = np.sum(grad.numpy().astype(np.float64) * move)
    # 2400 products of about 1, each of a value rounded a few times
    assert abs(differ - along) <= 2400 * 8 * 2.0 ** -24


def test_refusals(thc):
    w, t, y = thc.Tensor("float").resize((5, 4)).zero(), thc.Tensor.from_numpy(np.array([1, 2])), thc.Tensor("float").resize((2, 4)).zero()
    with pytest.raises(thc.THCError, match="two dims"):
        thc.Tensor("float").embedding(thc.Tensor("float").resize((5,)), t)
    with pytest.raises(thc.THCError, match="may not be the table"):
        w.embedding(w, t)
    with pytest.raises(thc.THCError, match="two dims"):
        thc.Tensor("float").resize((5,)).embedding_grad(t, y)
    with pytest.raises(thc.THCError, match="8 elements of the output's gradient for 3 tokens of 4"):
        w.embedding_grad(thc.Tensor.from_numpy(np.array([1, 2, 3])), y)
    with pytest.raises(thc.THCError, match="padding token is outside"):
        w.embedding_grad(t, y, padding=6)
    with pytest.raises(thc.THCError, match="overlap"):
        w.view_as_strided(0, (5, 4), (0, 1)).embedding_grad(t, y)
    half = thc.Tensor("half").resize((2, 4)).zero()
    for call in (lambda: thc.Tensor("half").embedding(w, t), lambda: thc.Tensor("float").embedding(w, y), lambda: w.embedding_grad(t, half),
                 lambda: w.embedding_grad(y, y)):
        with pytest.raises(ValueError):
            call()
    # no tokens: an empty output, a gradient of zeros
    assert thc.Tensor("float").embedding(w, thc.Tensor("long")).shape == ()
    w.fill(3).embedding_grad(thc.Tensor("long"), thc.Tensor("float"), accumulate=True)
    assert np.all(w.numpy() == 3)
    w.embedding_grad(thc.Tensor("long"), thc.Tensor("float"))
    assert not w.numpy().any()
