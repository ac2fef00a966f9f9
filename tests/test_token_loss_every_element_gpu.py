"""Every element of a row counts once: rows whose sums are whole numbers, rows with one logit far above the others, and bounds of the
gradient in proportion to each element. Any pack or edge that is left out, taken twice or written over is seen, at every length; that
the checks see it is tested on the oracle, which needs no GPU.

Roundings. EPS is half a place. A lane adds at most `chain` packs into its sum, each after a factor, behind the pack's own tree of 3 and
before 10 steps of joining lanes and waves, of 3 roundings each: no kernel has more than 25 packs of a row in a lane but those that read the rest
of a row again, in 1024 lanes, and the log-probabilities of rows below 256 packs or of 4800 rows, in 64. A term's exponent is a distance
below the maximum, off by 3 roundings of itself, and exp2 by 2."""
import numpy as np
import pytest

EPS = 2.0 ** -24
NP = {"float": np.float32, "half": np.float16}
gpu = pytest.mark.gpu
# around the ends of what a lane, a wave and a workgroup hold (packs of 4 floats or 8 halves), on both sides of the split of long rows
LENGTHS = [1, 2, 7, 8, 9, 31, 64, 255, 257, 511, 513, 1023, 1025, 2049, 4095, 4097, 8191, 8193, 16385, 24571, 32769, 40961, 51197, 65537, 81913,
           102391, 102401, 131073, 204793, 204805, 262143]


def chain(vocab, kind, rows, graded):
    packs = vocab * NP[kind]().itemsize // 16 + 8
    lanes = 1024 if graded else 64 if rows >= 4800 or packs < 256 else 128
    return packs / lanes + 25


@pytest.fixture(params=["split", "whole"])
def rows_are(thc, request):
    thc.set_tuning("loss.split", 100 if request.param == "split" else 1 << 30)
    yield request.param
    thc.set_tuning("loss.split", 100)


def _run(thc, x, tokens, old, advantage, ref=None, weight=None, scale=1.0, kl=0.0, shift=0, place=False):
    """Loss, log-probability and gradient; `shift`: the rows are a window that begins so many elements into wider ones."""
    t = thc.Tensor.from_numpy
    rows, vocab = x.shape
    if shift:
        logits = t(np.concatenate([np.full((rows, shift), 9, x.dtype), x], 1)).narrow(1, shift, vocab)
        room = thc.Tensor(logits.kind).resize((rows, vocab + shift)).fill(3)
        g = room.narrow(1, shift, vocab)
    else:
        logits = t(x)
        g = room = logits if place else thc.Tensor(logits.kind)
    loss, lp = thc.Tensor("float"), thc.Tensor("float")
    loss.policy_loss(lp, g, logits, t(tokens), t(old), t(advantage), t(ref) if ref is not None else None, t(weight) if weight is not None else None,
                     0.2, 0.25, kl, scale)
    if shift:
        assert np.all(room.narrow(1, 0, shift).numpy() == 3)
    return loss.numpy(), lp.numpy(), g.numpy()


# ---------------------------------------------------------------- equal logits --
def equal_case(rng, rows, vocab):
    """Logits of 0: a row's sum is its length exactly, all probabilities are alike."""
    tokens = rng.integers(1, vocab + 1, rows)
    tokens[0], tokens[-1] = 1, vocab
    old = np.full(rows, -np.log(vocab) - 0.05, np.float32)
    advantage = rng.choice([-1.0, -0.5, 0.5, 1.0], rows).astype(np.float32)
    return tokens, old, advantage


def off_log_prob(vocab):
    """log2 of the sum is off by a place, the factor ln 2 by a quarter of one, their product by half."""
    place = 2.0 ** np.floor(np.log2(max(1.0, np.log2(vocab)))) * 2 * EPS
    return np.log(2) * place + 1.5 * EPS * np.log(vocab)


def check_equal(lp, grad, tokens, advantage, scale, kind):
    rows, vocab = grad.shape
    assert np.all(np.abs(lp + np.log(vocab)) <= off_log_prob(vocab)), np.max(np.abs(lp + np.log(vocab)))
    g, i = grad.astype(np.float64), np.arange(rows)
    hot = g[i, tokens - 1]
    slope = -advantage.astype(np.float64) * np.exp(0.05) * scale / rows
    if vocab > 1:
        # the slope itself: the ratio's exponent is off by the log-probability and the roundings of two numbers of its size
        near = off_log_prob(vocab) + EPS * (8 * np.log(vocab) + 16)
        half = 2.0 ** -11 if kind == "half" else 0
        assert np.all(np.abs(hot - slope * (1 - 1 / vocab)) <= np.abs(slope) * (near + half)), np.abs(hot / slope - 1).max()
        g[i, tokens - 1] = np.nan
        others = -g * vocab / slope[:, None]
        if kind == "float":      # beside it, all others: c times 1, a quotient, two products
            others *= (slope * (1 - 1 / vocab) / hot)[:, None]
            near = 8 * EPS
        else:
            near += half + 2.0 ** -25 * vocab / np.abs(slope).min()
        assert np.nanmax(np.abs(others - 1)) <= near, np.nanmax(np.abs(others - 1))
    else:
        assert np.all(np.abs(g) <= np.abs(slope)[:, None] * 4 * EPS)


def _equal_oracle(tokens, advantage, vocab, scale, kind, count=None, lost=()):
    """The row's sum as `count` (the length where it is right), gradients of the elements `lost` not written."""
    rows = len(tokens)
    count = vocab if count is None else count
    slope = (-advantage.astype(np.float64) * np.exp(0.05) * scale / rows).astype(np.float32)
    g = np.repeat((-slope / np.float32(count))[:, None], vocab, 1)
    g[np.arange(rows), tokens - 1] += slope
    g[:, list(lost)] = 0
    return np.full(rows, np.float32(-np.log(count))), g.astype(NP[kind])


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", [513, 33001, 131073, 262143])
def test_the_checks_see_what_is_left_out(kind, vocab):
    rng = np.random.default_rng(vocab)
    tokens, _, advantage = equal_case(rng, 3, vocab)
    scale = 1024.0
    check_equal(*_equal_oracle(tokens, advantage, vocab, scale, kind), tokens, advantage, scale, kind)
    pack = 16 // NP[kind]().itemsize
    at = vocab // 2
    for wrong in (dict(count=vocab - 1), dict(count=vocab + 1), dict(count=vocab - pack), dict(count=vocab + pack), dict(lost=[at]),
                  dict(lost=[0]), dict(lost=[vocab - 1]), dict(lost=range(at, at + pack))):
        with pytest.raises(AssertionError):
            check_equal(*_equal_oracle(tokens, advantage, vocab, scale, kind, **wrong), tokens, advantage, scale, kind)


@gpu
@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", LENGTHS)
def test_equal_logits(thc, rows_are, kind, vocab):
    rng = np.random.default_rng(vocab)
    for rows, shift, place in ((3, 0, False), (3, 0, True), (5, 1, False), (2, 3, False), (2, 7, False)):
        tokens, old, advantage = equal_case(rng, rows, vocab)
        x = np.zeros((rows, vocab), NP[kind])
        scale = 1024.0
        _, lp, grad = _run(thc, x, tokens, old, advantage, scale=scale, shift=shift, place=place)
        check_equal(lp, grad, tokens, advantage, scale, kind)
        alone = thc.Tensor("float").token_log_prob(thc.Tensor.from_numpy(x), thc.Tensor.from_numpy(tokens)).numpy()
        assert np.all(np.abs(alone + np.log(vocab)) <= off_log_prob(vocab))


@gpu
@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("rows,vocab", [(5000, 301), (4900, 2049), (2500, 2051), (1300, 4099), (650, 8201), (300, 16389), (140, 40961), (129, 131073)])
def test_equal_logits_of_many_rows(thc, kind, rows, vocab):
    """As many rows as change the waves of each."""
    rng = np.random.default_rng(rows)
    tokens, old, advantage = equal_case(rng, rows, vocab)
    x, scale = np.zeros((rows, vocab), NP[kind]), 1024.0 * rows / 3
    _, lp, grad = _run(thc, x, tokens, old, advantage, scale=scale)
    check_equal(lp, grad, tokens, advantage, scale, kind)
    alone = thc.Tensor("float").token_log_prob(thc.Tensor.from_numpy(x), thc.Tensor.from_numpy(tokens)).numpy()
    assert np.all(np.abs(alone + np.log(vocab)) <= off_log_prob(vocab))


# -------------------------------------------------------------- one far above --
def spikes(vocab, kind):
    """The ends of a row and of what its lanes, waves, workgroups and parts hold, and their neighbours."""
    pack = 16 // NP[kind]().itemsize
    ends = [0, vocab]
    ends += [64 * waves * packs * pack for waves in (1, 2, 4, 8, 16) for packs in (1, 2, 4, 8, 12, 16, 21, 25)]
    ends += [vocab * part // 64 for part in range(0, 64, 7)]
    near = {e + d for e in ends for d in (-pack - 1, -pack, -1, 0, 1, pack - 1, pack)}
    near = sorted(p for p in near if 0 <= p < vocab)
    return near if len(near) <= 120 else near[:8] + sorted(np.random.default_rng(vocab).choice(near[8:-8], 104, replace=False).tolist()) + near[-8:]


@gpu
@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", [1025, 8193, 32769, 51197, 81913, 102401, 131073, 204805, 262143])
def test_one_logit_far_above_the_others(thc, rows_are, kind, vocab):
    """It has all the probability, 200 above the rest: a maximum that misses it overflows, a sum that misses it is off by everything."""
    at = np.array(spikes(vocab, kind))
    rows = len(at)
    x = np.zeros((rows, vocab), NP[kind])
    x[np.arange(rows), at] = 200
    tokens = np.where(at + 1 < vocab, at + 2, at)           # a neighbour
    lp = thc.Tensor("float").token_log_prob(thc.Tensor.from_numpy(x), thc.Tensor.from_numpy(tokens)).numpy()
    assert np.all(np.abs(lp + 200) <= 200 * 6 * EPS)
    one = np.ones(rows, np.float32)
    for first in range(0, rows, 16):       # (few rows: they are split)
        i = slice(first, min(rows, first + 16))
        n = i.stop - first
        old = np.full(n, -200 - 0.05, np.float32)
        loss, lp, grad = _run(thc, x[i], tokens[i], old, -one[i], weight=one[i])
        # the ratio's exponent is the difference of two numbers of 200, each off by some roundings of that
        ratio, near = np.exp(-200 - old.astype(np.float64)), 200 * 8 * EPS
        assert np.all(np.abs(lp + 200) <= 200 * 6 * EPS) and np.all(np.abs(loss / ratio - 1) <= near)
        half = 2.0 ** -11 if kind == "half" else 0
        g, r = grad.astype(np.float64), np.arange(n)
        assert np.all(np.abs(g[r, tokens[i] - 1] / ratio - 1) <= near + half) and np.all(np.abs(g[r, at[i]] / -ratio - 1) <= near + half)
        g[r, tokens[i] - 1] = g[r, at[i]] = 0
        assert not g.any()
        # the token itself: it is certain, and nothing is to learn
        loss, lp, grad = _run(thc, x[i], at[i] + 1, np.full(n, -0.05, np.float32), one[i], weight=one[i])
        assert np.all(np.abs(lp) <= 200 * 2 * EPS) and np.all(np.abs(grad) <= 200 * 8 * EPS)


# ------------------------------------------------------------- bounds by element --
def oracle(x, tokens, old, advantage, ref, weight, kl, scale, without=()):
    """Loss, log-probability, gradient and what the bounds are made of, in float64; `without`: columns that a sum misses."""
    x = x.astype(np.float64)
    rows = np.arange(len(x))
    away = x.max(1, keepdims=True) - x
    e = np.exp(-away)
    counted = e.copy()
    counted[:, list(without)] = 0
    s = counted.sum(1)
    lp = -away[rows, tokens - 1] - np.log(s)
    p = e / s[:, None]
    r = np.exp(lp - old)
    free, held = r * advantage, np.clip(r, np.float32(0.8), np.float32(1.25)) * advantage
    loss, slope = -np.minimum(free, held), np.where(free <= held, -free, 0.0)
    k = np.exp(ref - lp)
    loss, slope = loss + kl * (k - (ref - lp) - 1), slope + kl * (1 - k)
    hot = np.zeros(x.shape)
    hot[rows, tokens - 1] = 1
    return weight * loss, lp, (scale * weight * slope)[:, None] * (hot - p), dict(away=away, p=p, r=r, k=k, slope=slope, hot=hot)


def check_bounds(got, want, x, tokens, old, advantage, ref, weight, kl, scale, kind, links):
    w_loss, w_lp, w_grad, u = want
    away, p, slope, k, r = u["away"], u["p"], u["slope"], u["k"], u["r"]
    span = away[np.arange(len(x)), tokens - 1]
    d_sum = EPS * (2 * links + 3 + 30 + 2 + 3 * (p * away).sum(1))
    d_lp = d_sum + EPS * (4 * span + 4 * np.abs(w_lp) + 4)
    near = np.abs(w_lp) + np.abs(old) + np.abs(ref)
    d = d_lp + EPS * (2 * near + 10)
    d_slope = (np.abs(advantage) * r + kl * k) * d + 4 * EPS * kl
    d_loss = weight * (d_slope + 4 * EPS * kl * (k + near + 1))
    d_grad = weight[:, None] * scale * (d_slope[:, None] * np.abs(u["hot"] - p) + np.abs(slope)[:, None] *
                                        (p * (d_sum[:, None] + EPS * (3 * away + 6)) + 4 * EPS * (u["hot"] + p))) + 1e-37
    if kind == "half":
        d_grad = d_grad + 2.0 ** -11 * np.abs(w_grad) * (1 + 2.0 ** -10) + 2.0 ** -25
    loss, lp, grad = got
    assert np.all(np.abs(lp - w_lp) <= d_lp), (np.abs(lp - w_lp) / d_lp).max()
    assert np.all(np.abs(loss - w_loss) <= d_loss), (np.abs(loss - w_loss) / d_loss).max()
    off = np.abs(grad.astype(np.float64) - w_grad)
    assert np.all(off <= d_grad), ((off / d_grad).max(), np.argwhere(off > d_grad)[:4])


def bounds_case(rng, rows, vocab, kind):
    x = (1.5 * rng.standard_normal((rows, vocab))).astype(NP[kind])
    tokens = rng.integers(1, vocab + 1, rows)
    tokens[0], tokens[-1] = vocab, 1
    z = x.astype(np.float64)
    lp = z[np.arange(rows), tokens - 1] - np.log(np.exp(z).sum(1))
    old = (lp - rng.choice([-0.5, -0.1, 0.05, 0.4], rows)).astype(np.float32)
    advantage = (rng.choice([-1, 1], rows) * rng.uniform(0.5, 2, rows)).astype(np.float32)
    ref = (lp + 0.5 * rng.standard_normal(rows)).astype(np.float32)
    return x, tokens, old, advantage, ref, (0.5 + rng.random(rows)).astype(np.float32)


def _wide(case):
    return tuple(a.astype(np.float64) for a in case[2:])


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", [1000, 33001, 131071])
def test_the_bounds_see_wrong_elements(kind, vocab):
    """Of the gradient rounded to its type, one element in its place: zero, its negative, off by a hundredth; and sums without a pack."""
    case = bounds_case(np.random.default_rng(vocab), 2, vocab, kind)
    kl, scale, links = np.float32(0.1), 4096.0, chain(vocab, kind, 2, True)
    want = oracle(case[0], case[1], *_wide(case), kl, scale)
    args = (want, case[0], case[1], *_wide(case), kl, scale, kind, links)
    right = (want[0], want[1], want[2].astype(NP[kind]))
    check_bounds(right, *args)
    # rows whose ratio is clipped learn from the KL term's small difference alone; the smallest halves are far apart
    size, learns = np.abs(want[2]), np.abs(want[3]["slope"]) > 0.1
    told = np.argwhere((size > (2.0 ** -22 if kind == "half" else 0)) & learns[:, None])
    assert len(told) > 0.9 * vocab * learns.sum() > 0
    for row, column in told[:: max(1, len(told) // 40)]:
        for wrong in (0, -want[2][row, column]) + ((1.01 * want[2][row, column],) if size[row, column] > 2.0 ** -15 else ()):
            grad = right[2].copy()
            grad[row, column] = wrong
            with pytest.raises(AssertionError):
                check_bounds((right[0], right[1], grad), *args)
    pack = 16 // NP[kind]().itemsize
    whole = want[3]["p"][0][: vocab // pack * pack].reshape(-1, pack).sum(1)
    # those that have more than 5e-5 of the row; equal logits tell of the others
    some = np.flatnonzero(whole > 5e-5)
    assert len(some) > 0.1 * len(whole)
    for j in some[:: max(1, len(some) // 40)]:
        less = oracle(case[0], case[1], *_wide(case), kl, scale, without=range(j * pack, j * pack + pack))
        with pytest.raises(AssertionError):
            check_bounds((less[0], less[1], less[2].astype(NP[kind])), *args)


@gpu
@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("vocab", LENGTHS)
def test_every_element_of_the_gradient(thc, rows_are, kind, vocab):
    rng = np.random.default_rng(vocab + 1)
    for rows, shift, place in ((3, 0, False), (3, 0, True), (2, 5, False)) + (((300, 0, False),) if vocab < 600 else ()):
        case = bounds_case(rng, rows, vocab, kind)
        x, tokens, old, advantage, ref, weight = case
        kl, scale = np.float32(0.1), float(2.0 ** min(13, 3 + np.floor(np.log2(vocab))))
        if kind == "half":
            scale = min(scale, 4096.0)      # (the token's own gradient stays below the type's largest)
        got = _run(thc, x, tokens, old, advantage, ref, weight, scale, kl, shift, place)
        check_bounds(got, oracle(x, tokens, *_wide(case), kl, scale), x, tokens, *_wide(case), kl, scale, kind, chain(vocab, kind, rows, True))
        alone = thc.Tensor("float").token_log_prob(thc.Tensor.from_numpy(x), thc.Tensor.from_numpy(tokens)).numpy()
        want = oracle(x, tokens, *_wide(case), kl, scale)
        u = want[3]
        span = u["away"][np.arange(rows), tokens - 1]
        bound = EPS * (2 * chain(vocab, kind, rows, False) + 35 + 3 * (u["p"] * u["away"]).sum(1) + 4 * span + 4 * np.abs(want[1]) + 4)
        assert np.all(np.abs(alone - want[1]) <= bound)
