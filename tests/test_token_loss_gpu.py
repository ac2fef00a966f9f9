"""Token log-probabilities and the policy loss with its gradient against float64, at row lengths around every kernel's edges, with
masked rows and logits that are not finite."""
import numpy as np
import pytest

from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
NP = {"float": np.float32, "half": np.float16}
EPS = 2.0 ** -24
LENGTHS = [1, 2, 3, 5, 7, 8, 9, 15, 16, 17, 63, 65, 255, 257, 511, 513, 1000, 1025, 2047, 2049, 4097, 8191, 8200, 16385, 32000, 33001]
LONG = [50001, 65537, 70003, 131071, 131080, 150001, 262144]


def _logits(rng, rows, vocab, kind, spread=3.0):
    return (spread * rng.standard_normal((rows, vocab))).astype(NP[kind])


def _log_prob(x, tokens):
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    lse = m[:, 0] + np.log(np.exp(x - m).sum(1))
    return x[np.arange(len(x)), tokens - 1] - lse


def _lp_bound(x, tokens, want):
    """x - max rounds once, so does its product with log2(e); exp2 and its sums (a lane adds vocab / 64 terms at most, then a tree), the
    logarithm, the last two subtractions round; terms far below the maximum weigh their distance's rounding little: 3 stands for it."""
    span = (x.max(1) - x[np.arange(len(x)), tokens - 1]).astype(np.float64)
    return EPS * (x.shape[1] / 64 + 24 + 3 + 4 * span + 4 * np.abs(want))


@pytest.fixture(params=["split", "whole"])
def rows_are(thc, request):
    """Few long rows are split between workgroups, or not, as many are not."""
    thc.set_tuning("loss.split", 100 if request.param == "split" else 1 << 30)
    yield request.param
    thc.set_tuning("loss.split", 100)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", [40001, 81913, 120000, 160011, 262145])
def test_log_prob_of_long_rows(thc, rows_are, kind, vocab):
    rng = np.random.default_rng(vocab)
    for rows in (2, 70):
        x, tokens = _logits(rng, rows, vocab, kind), rng.integers(1, vocab + 1, rows)
        want = _log_prob(x, tokens)
        off = np.abs(thc.Tensor("float").token_log_prob(thc.Tensor.from_numpy(x), thc.Tensor.from_numpy(tokens)).numpy() - want)
        assert np.all(off <= _lp_bound(x, tokens, want)), (rows, off.max())


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", LENGTHS + LONG)
def test_log_prob(thc, kind, vocab):
    rng = np.random.default_rng(vocab)
    for rows in (1, 3, 300) if vocab < 3000 else (1, 3):
        x, tokens = _logits(rng, rows, vocab, kind), rng.integers(1, vocab + 1, rows)
        got = thc.Tensor("float").token_log_prob(thc.Tensor.from_numpy(x), thc.Tensor.from_numpy(tokens))
        assert thc.last_kernel() == "token-logprob"
        want = _log_prob(x, tokens)
        off = np.abs(got.numpy() - want)
        assert np.all(off <= _lp_bound(x, tokens, want)), (rows, off.max())


def _policy(x, tokens, old, advantage, reference, weight, low, high, kl, scale):
    """Losses, log-probabilities and gradient in float64, and the slope of each loss in its log-probability."""
    rows, vocab = x.shape
    lp = _log_prob(x, tokens)
    r = np.exp(lp - old)
    free, held = r * advantage, np.clip(r, np.float32(1 - low), np.float32(1 + high)) * advantage
    loss, slope = -np.minimum(free, held), np.where(free <= held, -free, 0.0)
    if reference is not None:
        e = np.exp(reference - lp)
        loss, slope = loss + kl * (e - (reference - lp) - 1), slope + kl * (1 - e)
    p = np.exp(x.astype(np.float64) - x.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    hot = np.zeros(x.shape)
    hot[np.arange(rows), tokens - 1] = 1
    return weight * loss, lp, (scale * weight * slope)[:, None] * (hot - p), slope, p


def _case(rng, rows, vocab, kind, reference, masked):
    x, tokens = _logits(rng, rows, vocab, kind), rng.integers(1, vocab + 1, rows)
    lp = _log_prob(x, tokens)
    # ratios inside, below and above the clip (0.8 to 1.2 or 1.25), none near its edges
    old = (lp - rng.choice([-0.5, -0.1, 0.05, 0.4], rows)).astype(np.float32)
    advantage = rng.standard_normal(rows).astype(np.float32)
    ref = (lp + 0.5 * rng.standard_normal(rows)).astype(np.float32) if reference else None
    weight = rng.random(rows).astype(np.float32) + np.float32(0.1)
    if masked:
        weight[rng.random(rows) < 0.3] = 0
    return x, tokens, old, advantage, ref, weight


def _bounds(x, tokens, old, advantage, ref, weight, kl, scale, want, kind):
    loss, lp, grad, slope, p = want
    dlp = _lp_bound(x, tokens, lp)
    r, e = np.exp(lp - old), np.exp(ref - lp) if ref is not None else np.zeros(len(x))
    # a ratio is off by its exponent's error; a few roundings of each term follow
    near = np.abs(lp) + np.abs(old) + (np.abs(ref) if ref is not None else 0)
    d = dlp + 2 * EPS * near + 4 * EPS
    b_loss = weight * ((np.abs(advantage) * r + kl * (e + 1)) * (d + 6 * EPS) + kl * EPS * 4 * (e + near + 1))
    b_slope = (np.abs(advantage) * r + kl * e) * (d + 6 * EPS) + kl * EPS * 4
    away = x.max(1, keepdims=True).astype(np.float64) - x
    b_grad = abs(scale) * weight[:, None] * (b_slope[:, None] + np.abs(slope)[:, None] * p * (dlp[:, None] + EPS * (8 + 4 * away)) + np.abs(slope)[:, None] * 4 * EPS)
    if kind == "half":
        b_grad = b_grad + 2.0 ** -11 * np.abs(grad) * (1 + 2.0 ** -10) + 2.0 ** -25
    return b_loss, dlp, b_grad


def _run(thc, case, low=0.2, high=0.25, kl=0.1, scale=1.0, grad=True, into=None):
    x, tokens, old, advantage, ref, weight = case
    t = thc.Tensor.from_numpy
    logits = t(x)
    kind = logits.kind
    g = thc.Tensor(kind) if grad and into is None else logits if into == "logits" else into
    loss, lp = thc.Tensor("float"), thc.Tensor("float")
    loss.policy_loss(lp, g, logits, t(tokens), t(old), t(advantage), t(ref) if ref is not None else None,
                     t(weight) if weight is not None else None, low, high, kl, scale)
    assert thc.last_kernel() == "policy-loss"
    return loss.numpy(), lp.numpy(), g.numpy() if g is not None else None


def _check(thc, rng, rows, vocab, kind, reference, masked, scale=8.0):
    case = _case(rng, rows, vocab, kind, reference, masked)
    x, tokens, old, advantage, ref, weight = case
    want = _policy(x, tokens, old.astype(np.float64), advantage.astype(np.float64), ref.astype(np.float64) if reference else None,
                   weight.astype(np.float64), 0.2, 0.25, np.float32(0.1), scale)
    b_loss, b_lp, b_grad = _bounds(x, tokens, old, advantage, ref, weight, 0.1, scale, want, kind)
    loss, lp, grad = _run(thc, case, scale=scale)
    kept = weight != 0
    assert np.all(np.abs(loss - want[0]) <= b_loss), np.max(np.abs(loss - want[0]) - b_loss)
    assert np.all(np.abs(lp - want[1])[kept] <= b_lp[kept])
    off = np.abs(grad.astype(np.float64) - want[2])
    assert np.all(off <= b_grad), (np.max(off - b_grad), np.argwhere(off > b_grad)[:4])
    assert not loss[~kept].any() and not lp[~kept].any() and not grad[~kept].any()
    return case, (loss, lp, grad)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", LENGTHS)
@pytest.mark.parametrize("reference", [False, True])
def test_policy_loss(thc, kind, vocab, reference):
    rng = np.random.default_rng(vocab + reference)
    for rows in (1, 7, 200) if vocab < 600 else (1, 7):
        case, first = _check(thc, rng, rows, vocab, kind, reference, masked=rows > 1)
        for a, b in zip(_run(thc, case, scale=8.0), first):
            assert_bit_equal(a, b)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", LONG + [81850, 102400, 204700, 210001])
def test_policy_loss_of_long_rows(thc, rows_are, kind, vocab):
    rng = np.random.default_rng(vocab)
    _check(thc, rng, 3, vocab, kind, True, masked=False, scale=512.0)
    _check(thc, rng, 11, vocab, kind, False, masked=True, scale=512.0)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("rows,vocab", [(600, 4001), (1100, 2000), (300, 16390)])
def test_policy_loss_of_many_rows(thc, kind, rows, vocab):
    _check(thc, np.random.default_rng(rows), rows, vocab, kind, True, masked=True)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", [5, 1000, 1001, 33001, 140001, 210001])
def test_gradient_in_the_logits_place(thc, rows_are, kind, vocab):
    rng = np.random.default_rng(vocab)
    case = _case(rng, 40 if vocab < 2000 else 4, vocab, kind, True, True)
    apart, place = _run(thc, case, scale=8.0), _run(thc, case, scale=8.0, into="logits")
    for a, b in zip(apart, place):
        assert_bit_equal(b, a)
    loss, lp, none = _run(thc, case, grad=False)
    assert none is None
    # losses alone may be summed by another kernel
    assert np.all(np.abs(loss - apart[0]) <= 1e-5 * (1 + np.abs(apart[0]))) and np.all(np.abs(lp - apart[1]) <= 1e-5 * (1 + np.abs(apart[1])))


@pytest.mark.parametrize("kind", ["float", "half"])
def test_views(thc, kind):
    """Sequences whose last position is left out, a window of the vocabulary, a transposed batch, outputs that are views."""
    rng = np.random.default_rng(2)
    wide = _logits(rng, 6 * 9, 120, kind).reshape(6, 9, 120)
    tokens = rng.integers(1, 101, (6, 9))
    d, t = thc.Tensor.from_numpy(wide), thc.Tensor.from_numpy(tokens)
    for view, plain, toks, tview in ((d.narrow(1, 0, 8).narrow(2, 7, 101), wide[:, :8, 7:108], tokens[:, :8], t.narrow(1, 0, 8)),
                                     (d.t(0, 1), wide.transpose(1, 0, 2), tokens.T, t.t()),
                                     (d.t(1, 2).narrow(1, 0, 110).t(1, 2), wide[:, :, :110], tokens, t),
                                     (d.t(0, 2).t(0, 2).select(0, 3), wide[3], tokens[3], t.select(0, 3))):
        x = np.ascontiguousarray(plain).reshape(-1, plain.shape[-1])
        flat = np.ascontiguousarray(toks).reshape(-1)
        want = _log_prob(x, flat)
        got = thc.Tensor("float").token_log_prob(view, tview)
        assert got.shape == toks.shape
        assert np.all(np.abs(got.numpy().reshape(-1) - want) <= _lp_bound(x, flat, want))
        old, advantage = (want - 0.05).astype(np.float32), rng.standard_normal(want.size).astype(np.float32)
        room = thc.Tensor(kind).resize((int(np.prod(toks.shape)), x.shape[1] + 5)).fill(3)
        out = room.narrow(1, 2, x.shape[1]) if toks.ndim == 1 else None
        g = thc.Tensor(kind) if out is None else out
        loss, lp = thc.Tensor("float").resize(toks.shape[::-1]).t() if toks.ndim == 2 else thc.Tensor("float"), thc.Tensor("float")
        shaped = [thc.Tensor.from_numpy(a.reshape(toks.shape)) for a in (old, advantage)]
        loss.policy_loss(lp, g, view, tview, *shaped, None, None, 0.2, 0.25, 0.0, 16.0)
        assert loss.shape == toks.shape and g.shape == plain.shape
        weight = np.full(want.size, 1.0 / want.size)
        ref = _policy(x, flat, old.astype(np.float64), advantage.astype(np.float64), None, weight, 0.2, 0.25, 0, 16.0)
        b_loss, _, b_grad = _bounds(x, flat, old, advantage, None, weight, 0, 16.0, ref, kind)
        assert np.all(np.abs(loss.numpy().reshape(-1) - ref[0]) <= b_loss + EPS * np.abs(ref[0]))
        assert np.all(np.abs(g.numpy().reshape(x.shape) - ref[2]) <= b_grad + EPS * np.abs(ref[2]))
        if out is not None:
            assert np.all(room.numpy()[:, :2] == 3) and np.all(room.numpy()[:, 2 + x.shape[1]:] == 3)


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", [6, 1000, 9001, 140001])
def test_rows_that_hold_nothing_to_learn_from(thc, rows_are, kind, vocab):
    """Masked logits (-inf and the type's lowest value), rows of weight 0 that hold anything, a token that the mask has taken away."""
    rng = np.random.default_rng(vocab)
    x, tokens, old, advantage, ref, weight = _case(rng, 8, vocab, kind, True, False)
    cut = vocab // 2
    tokens[:] = rng.integers(1, cut + 1, 8)
    x[0, cut:] = -np.inf
    x[1, cut:] = np.finfo(NP[kind]).min
    x[2], weight[2], old[2], ref[2] = np.nan, 0, np.nan, np.inf
    x[3], weight[3], advantage[3] = -np.inf, 0, np.nan
    tokens[4], weight[4] = 0, 0
    tokens[5], weight[5] = vocab + 1, 0
    lp = _log_prob(x[[0, 1, 6, 7]].astype(np.float64), tokens[[0, 1, 6, 7]])
    old[[0, 1, 6, 7]] = (lp - 0.05).astype(np.float32)
    loss, got, grad = _run(thc, (x, tokens, old, advantage, ref, weight), scale=4.0)
    rows = [0, 1, 6, 7]
    with np.errstate(all="ignore"):
        want = _policy(x[rows].astype(np.float64), tokens[rows], old[rows].astype(np.float64), advantage[rows].astype(np.float64),
                       ref[rows].astype(np.float64), weight[rows].astype(np.float64), 0.2, 0.25, np.float32(0.1), 4.0)
        finite = np.where(x[rows] > -1e4, x[rows], x[rows].max(1, keepdims=True) - 100)
        b_loss, b_lp, b_grad = _bounds(finite, tokens[rows], old[rows], advantage[rows], ref[rows], weight[rows], 0.1, 4.0, want, kind)
    assert np.all(np.abs(got[rows] - want[1]) <= b_lp) and np.all(np.abs(loss[rows] - want[0]) <= b_loss)
    assert np.all(np.abs(grad[rows] - want[2]) <= b_grad)
    assert not grad[:2, cut:].any()
    for r in (2, 3, 4, 5):
        assert loss[r] == 0 and got[r] == 0 and not grad[r].any()
    # with a weight, what cannot be computed says so
    weight[:] = 1
    loss, got, grad = _run(thc, (x, tokens, old, advantage, ref, weight))
    for r in (2, 3, 4, 5):
        assert np.isnan(loss[r]) and np.isnan(got[r])
    # a token whose logit is -inf: probability 0, no gradient through the ratio
    x[6, tokens[6] - 1] = -np.inf
    loss, got, grad = _run(thc, (x, tokens, old, np.abs(advantage), ref, weight), kl=0.0)
    assert got[6] == -np.inf and loss[6] == 0 and not grad[6].any()


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", [3, 700, 5000, 90001])
def test_rows_of_one_extreme_value(thc, rows_are, kind, vocab):
    """A mask of the type's lowest value over all of a row leaves every token as likely, whatever the value; so does its highest."""
    low, high = np.finfo(NP[kind]).min, np.finfo(NP[kind]).max
    x = np.stack([np.full(vocab, v, NP[kind]) for v in (low, high, low / 2, NP[kind](1))])
    x[2, 1] = low            # one that is lower still has no chance
    tokens = np.array([1, vocab, 1, 2])
    got = thc.Tensor("float").token_log_prob(thc.Tensor.from_numpy(x), thc.Tensor.from_numpy(tokens)).numpy()
    want = -np.log([vocab, vocab, vocab - 1, vocab])
    assert np.all(np.abs(got - want) <= EPS * (vocab / 64 + 40 + 4 * np.abs(want)))
    old, advantage = want.astype(np.float32), -np.ones(4, np.float32)
    loss, lp, grad = _run(thc, (x, tokens, old, advantage, None, np.ones(4, np.float32)))
    share = np.full((4, vocab), 1.0 / vocab)
    share[2] = 1.0 / (vocab - 1)
    share[2, 1] = 0
    hot = np.zeros((4, vocab))
    hot[np.arange(4), tokens - 1] = 1
    # the ratios are 1 but for roundings, so are the slopes
    bound = (EPS * (vocab / 32 + 200)) + (2.0 ** -11 * np.abs(hot - share) + 2.0 ** -25 if kind == "half" else 0)
    assert np.all(np.abs(loss - 1) <= EPS * (vocab / 64 + 100)) and np.all(np.abs(grad - (hot - share)) <= bound)


def test_more_rows_than_a_grid_has_across(thc):
    """2^21 rows and some, of three logits."""
    rng = np.random.default_rng(3)
    rows = (1 << 21) + 1000
    case = _case(rng, rows, 3, "half", False, True)
    x, tokens, old, advantage, _, weight = case
    want = _policy(x, tokens, old.astype(np.float64), advantage.astype(np.float64), None, weight.astype(np.float64), 0.2, 0.25, 0, 1.0)
    b_loss, b_lp, b_grad = _bounds(x, tokens, old, advantage, None, weight, 0, 1.0, want, "half")
    loss, lp, grad = _run(thc, case)
    assert np.all(np.abs(loss - want[0]) <= b_loss) and np.all(np.abs(grad - want[2]) <= b_grad)
    got = thc.Tensor("float").token_log_prob(thc.Tensor.from_numpy(x), thc.Tensor.from_numpy(tokens)).numpy()
    assert np.all(np.abs(got - want[1]) <= b_lp) and np.all(np.abs(lp - want[1])[weight != 0] <= b_lp[weight != 0])


def test_gradient_against_differences(thc):
    """Central differences of the losses themselves, at logits that move one at a time by 2^-6: they are off by h^2/6 times the third
    derivative (some units here) and by the losses' own rounding over h."""
    rng = np.random.default_rng(11)
    case = _case(rng, 5, 9, "float", True, False)
    x = case[0]
    h = 2.0 ** -6
    _, _, grad = _run(thc, case)
    for j in range(9):
        ends = []
        for s in (h, -h):
            y = x.copy()
            y[:, j] += np.float32(s)
            ends.append(_run(thc, (y,) + case[1:], grad=False)[0].astype(np.float64))
        difference = (ends[0] - ends[1]) / (2 * h)
        steep = (np.abs(case[3]) * 1.7 + 0.2) * case[5]
        assert np.all(np.abs(difference - grad[:, j]) <= steep * (h * h * 4 + 64 * EPS / h)), (j, difference - grad[:, j])


def test_outputs_on_an_inputs_storage(thc):
    rng = np.random.default_rng(12)
    x, tokens, old, advantage, ref, weight = _case(rng, 30, 50, "float", True, False)
    want = _run(thc, (x, tokens, old, advantage, ref, weight))
    t = thc.Tensor.from_numpy
    together = t(np.stack([old, advantage, ref, weight]))
    o, a, r, w = (together.select(0, i) for i in range(4))
    lp, g = thc.Tensor("float"), thc.Tensor("float")
    a.policy_loss(w, g, t(x), t(tokens), o, a, r, w, 0.2, 0.25, 0.1, 1.0)      # losses over the advantages, log-probabilities over the weights
    got = together.numpy()
    assert_bit_equal(got[1], want[0])
    assert_bit_equal(got[3], want[1])
    assert_bit_equal(g.numpy(), want[2])
    assert_bit_equal(got[0], old)
    # a gradient that lies on the logits, but not as they lie
    big = t(np.concatenate([x, np.zeros_like(x)]))
    shifted = big.narrow(0, 10, 30)
    thc.Tensor("float").policy_loss(lp, shifted, big.narrow(0, 0, 30), t(tokens), t(old), t(advantage), t(ref), t(weight), 0.2, 0.25, 0.1, 1.0)
    assert_bit_equal(shifted.numpy(), want[2])


def test_outputs_that_make_a_shared_storage_grow(thc):
    """Losses, log-probabilities and gradient are windows behind the inputs, and grow: everything moves with the storage."""
    rng = np.random.default_rng(13)
    x, tokens, old, advantage, ref, weight = _case(rng, 30, 50, "float", True, False)
    want = _run(thc, (x, tokens, old, advantage, ref, weight))
    t = thc.Tensor.from_numpy
    end = 1500 + 120
    room = t(np.concatenate([x.reshape(-1), old, advantage, ref, weight, np.zeros(61, np.float32)]))
    logits = room.view_as_strided(0, (30, 50), (50, 1))
    o, a, r, w = (room.narrow(0, 1500 + 30 * i, 30) for i in range(4))
    lp, loss, g = (room.narrow(0, end + 30 * i, 1) for i in range(3))
    loss.policy_loss(lp, g, logits, t(tokens), o, a, r, w, 0.2, 0.25, 0.1, 1.0)
    for got, wanted in ((loss, want[0]), (lp, want[1]), (g, want[2]), (logits, x), (o, old), (a, advantage), (r, ref), (w, weight)):
        assert_bit_equal(got.numpy(), wanted)
    with pytest.raises(thc.THCError, match="may not be the logits"):
        same = t(x)
        thc.Tensor("float").policy_loss(same, None, same, t(tokens), t(old), t(advantage))
    with pytest.raises(thc.THCError, match="losses may not be"):
        lp = thc.Tensor("float")
        lp.policy_loss(lp, None, t(x), t(tokens), t(old), t(advantage))


def test_refusals(thc):
    t = thc.Tensor.from_numpy
    x, tokens, per = t(np.zeros((4, 6), np.float32)), t(np.ones(4, np.int64)), t(np.zeros(4, np.float32))
    short = t(np.zeros(3, np.float32))
    f = lambda: thc.Tensor("float")   # noqa: E731
    with pytest.raises(thc.THCError, match="logits are empty"):
        f().token_log_prob(f(), tokens)
    with pytest.raises(thc.THCError, match="3 tokens for 4 rows"):
        f().token_log_prob(x, t(np.ones(3, np.int64)))
    with pytest.raises(thc.THCError, match="3 old log-probabilities"):
        f().policy_loss(f(), f(), x, tokens, short, per)
    with pytest.raises(thc.THCError, match="3 advantages"):
        f().policy_loss(f(), f(), x, tokens, per, short)
    with pytest.raises(thc.THCError, match="3 reference log-probabilities"):
        f().policy_loss(f(), f(), x, tokens, per, per, reference=short)
    with pytest.raises(thc.THCError, match="3 weights"):
        f().policy_loss(f(), f(), x, tokens, per, per, weight=short)
    for low, high in ((-0.1, 0.2), (1.5, 0.2), (0.2, -0.2), (float("nan"), 0.2)):
        with pytest.raises(thc.THCError, match="clipped"):
            f().policy_loss(f(), f(), x, tokens, per, per, clip_low=low, clip_high=high)
    half, longs = thc.Tensor("half"), thc.Tensor("long")
    for call in (lambda: half.token_log_prob(x, tokens), lambda: f().token_log_prob(x, per), lambda: half.policy_loss(f(), f(), x, tokens, per, per),
                 lambda: f().policy_loss(f(), half, x, tokens, per, per), lambda: f().policy_loss(longs, f(), x, tokens, per, per),
                 lambda: f().policy_loss(f(), f(), x, tokens, per, half), lambda: f().policy_loss(f(), f(), x, per, per, per)):
        with pytest.raises(ValueError):
            call()
