"""Outputs of the policy loss on one storage: side by side and in each other's gaps they are what they are apart, on one another they
are refused."""
import numpy as np
import pytest

from tests.test_token_loss_gpu import _case, _run
from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu


def _call(thc, case, loss, lp, g, logits=None):
    x, tokens, old, advantage, ref, weight = case
    t = thc.Tensor.from_numpy
    loss.policy_loss(lp, g, logits if logits is not None else t(x), t(tokens), t(old), t(advantage), t(ref), t(weight), 0.2, 0.25, 0.1, 1.0)


@pytest.mark.parametrize("rows,vocab", [(30, 50), (3, 50001)])
def test_outputs_in_each_others_gaps(thc, rows, vocab):
    case = _case(np.random.default_rng(vocab), rows, vocab, "float", True, False)
    want = _run(thc, case)
    # losses and log-probabilities as the two columns behind the gradient's rows, then in a gap between two of those rows
    room = thc.Tensor("float").resize((rows, vocab + 64)).fill(7)
    for loss, lp in ((room.select(1, vocab), room.select(1, vocab + 1)), (room.select(0, 0).narrow(0, vocab, rows), room.select(0, 1).narrow(0, vocab, rows))):
        _call(thc, case, loss, lp, room.narrow(1, 0, vocab))
        for got, wanted in zip((loss, lp, room.narrow(1, 0, vocab)), want):
            assert_bit_equal(got.numpy(), wanted)
        assert np.all(room.narrow(1, vocab + rows, 64 - rows).numpy() == 7)
        room.fill(7)
    # one behind the other, and each other's odd elements
    both = thc.Tensor("float").resize((2 * rows,)).fill(7)
    for loss, lp in ((both.narrow(0, rows, rows), both.narrow(0, 0, rows)), (both.view_as_strided(0, (rows,), (2,)), both.view_as_strided(1, (rows,), (2,)))):
        _call(thc, case, loss, lp, thc.Tensor("float"))
        assert_bit_equal(loss.numpy(), want[0])
        assert_bit_equal(lp.numpy(), want[1])


def test_outputs_on_one_another_are_refused(thc):
    case = _case(np.random.default_rng(1), 30, 50, "float", True, False)
    room = thc.Tensor("float").resize((1600,)).fill(7)
    grad = room.view_as_strided(0, (30, 50), (50, 1))
    apart = room.narrow(0, 1540, 30)
    for loss, lp, g, match in ((room.narrow(0, 1500, 30), room.narrow(0, 1529, 30), grad, "losses and the log-probabilities share"),
                               (room.narrow(0, 0, 30), apart, grad, "losses and the gradient share"),
                               (apart, room.narrow(0, 1490, 30), grad, "log-probabilities and the gradient share")):
        with pytest.raises(thc.THCError, match=match):
            _call(thc, case, loss, lp, g)
    # the gradient in the logits' place, the losses there, too
    logits = thc.Tensor.from_numpy(case[0])
    with pytest.raises(thc.THCError, match="losses and the gradient share"):
        _call(thc, case, logits.select(0, 0).narrow(0, 0, 30), apart, logits, logits)
    assert np.all(room.numpy() == 7)
    # an output that a call makes grow is looked at as it grows to be
    small = room.narrow(0, 1540, 1)
    with pytest.raises(thc.THCError, match="losses and the log-probabilities share"):
        _call(thc, case, small, room.narrow(0, 1550, 30), grad)
