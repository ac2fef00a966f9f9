"""The training operators on operands of more than 2^31 elements: what lies behind that is found where it should be."""
import numpy as np
import pytest

from tests.util import assert_bit_equal
from tests.test_token_loss_gpu import _log_prob, _lp_bound

pytestmark = pytest.mark.gpu
BIG = 2 ** 31


@pytest.fixture(autouse=True)
def room(thc):
    yield
    import gc
    gc.collect()


def _halves(rng, *size):
    return rng.standard_normal(size).astype(np.float16)


def test_lookup_out_of_and_into_more_than_2_31_elements(thc):
    rng = np.random.default_rng(1)
    dim = 4099
    rows = BIG // dim + 100
    ends = _halves(rng, 60, dim)
    table = thc.Tensor("half").resize((rows, dim)).zero()
    table.narrow(0, rows - 60, 60).copy_from(thc.Tensor.from_numpy(ends))
    tokens = np.full(rows, 1)
    tokens[-80:] = rng.integers(rows - 59, rows + 1, 80)
    got = thc.Tensor("half").embedding(table, thc.Tensor.from_numpy(tokens), 1.0)
    assert got.shape == (rows, dim)
    assert_bit_equal(got.narrow(0, rows - 80, 80).numpy(), ends[tokens[-80:] - 1 - (rows - 60)])
    assert_bit_equal(got.narrow(0, 0, 3).numpy(), np.zeros((3, dim), np.float16))


@pytest.mark.parametrize("few", [True, False])
def test_gradient_of_more_than_2_31_elements(thc, few):
    rng = np.random.default_rng(2)
    dim = 4099
    rows = BIG // dim + 100
    count = 300 if few else 3000
    tokens = np.concatenate([rng.permutation(50)[:40] + 1, rng.permutation(60) + rows - 59, np.full(count - 100, rows)])
    out = _halves(rng, count, dim)
    grad = thc.Tensor("half").resize((rows, dim)).fill(3)
    grad.embedding_grad(thc.Tensor.from_numpy(tokens), thc.Tensor.from_numpy(out), 1.0)
    for first, n in ((0, 50), (rows // 2, 20), (rows - 70, 70)):
        got = grad.narrow(0, first, n).numpy().astype(np.float64)
        for i in range(n):
            mine = out[tokens == first + i + 1].astype(np.float64)
            # each addition rounds in float, the sum to half
            bound = np.abs(mine).sum(0) * max(0, len(mine) - 1) * 2.0 ** -24 + np.abs(mine.sum(0)) * 2.0 ** -11 + 2.0 ** -25
            assert np.all(np.abs(got[i] - mine.sum(0)) <= bound)


def test_output_gradient_of_more_than_2_31_elements(thc):
    rng = np.random.default_rng(3)
    dim = 4096
    count = BIG // dim + 500
    ends = _halves(rng, 400, dim)
    out = thc.Tensor("half").resize((count, dim)).zero()
    out.narrow(0, count - 400, 400).copy_from(thc.Tensor.from_numpy(ends))
    tokens = rng.integers(1, 21, count)
    tokens[-400:] = rng.permutation(np.arange(400)) + 21
    grad = thc.Tensor("half").resize((420, dim))
    grad.embedding_grad(thc.Tensor.from_numpy(tokens), out, 1.0)
    assert_bit_equal(grad.narrow(0, 0, 20).numpy(), np.zeros((20, dim), np.float16))
    want = np.empty_like(ends)
    want[tokens[-400:] - 21] = ends
    assert_bit_equal(grad.narrow(0, 20, 400).numpy(), want)


@pytest.mark.parametrize("kind,dim", [("half", 1024), ("half", 1032), ("float", 512)])
def test_gradient_of_a_table_beyond_128_mib(thc, kind, dim):
    rng = np.random.default_rng(6)
    rows, count = 70001, 5000
    dtype = np.float16 if kind == "half" else np.float32
    tokens = rng.permutation(rows)[:count] + 1
    out = rng.standard_normal((count, dim)).astype(dtype)
    grad = thc.Tensor(kind).resize((rows, dim)).fill(7)
    grad.embedding_grad(thc.Tensor.from_numpy(tokens), thc.Tensor.from_numpy(out), 1.0)
    want = np.zeros((rows, dim), dtype)
    want[tokens - 1] = out
    assert_bit_equal(grad.numpy(), want)


@pytest.mark.parametrize("vocab", [262144, 32001])
def test_losses_of_more_than_2_31_logits(thc, vocab):
    rng = np.random.default_rng(4)
    rows = BIG // vocab + 70
    ends = (3 * rng.standard_normal((60, vocab))).astype(np.float16)
    tokens = rng.integers(1, vocab + 1, rows)
    weight = np.zeros(rows, np.float32)
    weight[-60:] = 0.5
    logits = thc.Tensor("half").resize((rows, vocab)).zero()
    logits.narrow(0, rows - 60, 60).copy_from(thc.Tensor.from_numpy(ends))
    ids = thc.Tensor.from_numpy(tokens)
    want = _log_prob(ends, tokens[-60:])
    bound = _lp_bound(ends, tokens[-60:], want)
    lp = thc.Tensor("float").token_log_prob(logits, ids).numpy()
    assert np.all(np.abs(lp[-60:] - want) <= bound)
    flat = -np.log(vocab)
    assert np.all(np.abs(lp[:-60] - flat) <= _lp_bound(np.zeros((1, vocab), np.float16), np.array([1]), np.array([flat])))
    # the gradient, in the logits' place, is that of the last rows alone in a tensor of their own
    old = thc.Tensor.from_numpy(want.astype(np.float32))
    far = thc.Tensor("float").resize((rows,)).zero()
    far.narrow(0, rows - 60, 60).copy_from(old)
    ones = np.ones(rows, np.float32)
    loss, new = thc.Tensor("float"), thc.Tensor("float")
    loss.policy_loss(new, logits, logits, ids, far, thc.Tensor.from_numpy(ones), weight=thc.Tensor.from_numpy(weight))
    x = ends.astype(np.float64)
    p = np.exp(x - x.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    p[np.arange(60), tokens[-60:] - 1] -= 1
    got = logits.narrow(0, rows - 60, 60).numpy().astype(np.float64)
    # the slope is -r A w, r = 1 to the log-probability's bound; p to the same; the result rounds to half
    assert np.all(np.abs(got - 0.5 * p) <= 0.5 * np.abs(p) * (4 * bound[:, None] + 2.0 ** -10) + 2.0 ** -24)
    assert_bit_equal(logits.narrow(0, 0, 4).numpy(), np.zeros((4, vocab), np.float16))
    assert_bit_equal(logits.narrow(0, rows - 64, 4).numpy(), np.zeros((4, vocab), np.float16))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_of_more_than_2_31_elements(thc, bits):
    rng = np.random.default_rng(5)
    n = BIG + 256 * 1000 + 77
    tail = 256 * 5 + 77
    p, g = _halves(rng, tail), _halves(rng, tail)
    param, grad = [thc.Tensor("half").resize((n,)).fill(1) for _ in range(2)]
    for whole, end in ((param, p), (grad, g)):
        whole.narrow(0, n - tail, tail).copy_from(thc.Tensor.from_numpy(end))
    own, ownGrad = thc.Tensor.from_numpy(p), thc.Tensor.from_numpy(g)
    first, firstGrad = [thc.Tensor("half").resize((512,)).fill(1) for _ in range(2)]
    for a, b in ((param, grad), (own, ownGrad), (first, firstGrad)):
        steps = thc.AdamW([a], [b], bits=bits, lr=1e-2)
        steps.step()
        steps.step()
    assert_bit_equal(param.narrow(0, n - tail, tail).numpy(), own.numpy())
    for at in (0, BIG // 2 - 200, BIG - 200):
        assert_bit_equal(param.narrow(0, at, 512).numpy(), first.numpy())
