"""The operators of a training step together: the example's policy learns its rule, and steps on streams of their own give the bits of
steps on the default one."""
import ctypes as C
import importlib.util
import os
import threading

import numpy as np
import pytest

from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("bigram_policy", os.path.join(ROOT, "examples", "bigram_policy.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("kind", ["float", "half"])
@pytest.mark.parametrize("bits", [32, 8])
def test_the_example_learns(thc, kind, bits):
    rewards = _example().train(vocab=64, batch=4096, rounds=12, kind=kind, bits=bits)
    assert rewards[0] < 0.05 and rewards[-1] > 0.4, rewards
    assert rewards == _example().train(vocab=64, batch=4096, rounds=12, kind=kind, bits=bits)      # to the last bit


class _Chain(object):
    """Lookup, log-probabilities, loss, gradient and step of one set of operands, of sizes that take workspaces."""

    def __init__(self, thc, seed, kind, vocab=9000, dim=70, count=5000, classes=90001):
        rng = np.random.default_rng(seed)
        real = np.float16 if kind == "half" else np.float32
        self.thc, self.kind = thc, kind
        t = thc.Tensor.from_numpy
        self.table, self.tokens = t((0.1 * rng.standard_normal((vocab, dim))).astype(real)), t(rng.integers(1, vocab + 1, count))
        self.logits, self.chosen = t(rng.standard_normal((5, classes)).astype(real)), t(rng.integers(1, classes + 1, 5))
        self.old = t(np.full(5, -11.5, np.float32))
        self.advantage = t(rng.standard_normal(5).astype(np.float32))
        self.grad = thc.Tensor(kind).resize((vocab, dim))
        # a strided parameter: it goes through a copy
        self.room = t(np.zeros((vocab, dim + 3), real))
        self.view = self.room.narrow(1, 1, dim).copy(self.table)
        self.optimizer = thc.AdamW([self.table, self.view], [self.grad, self.grad], bits=8)

    def run(self, turns=4):
        thc = self.thc
        rows, loss, lp, gl = (thc.Tensor(k) for k in (self.kind, "float", "float", self.kind))
        for _ in range(turns):
            rows.embedding(self.table, self.tokens, 3.0)
            self.grad.embedding_grad(self.tokens, rows, 0.5)
            self.optimizer.step(2.0)
            lp.token_log_prob(self.logits, self.chosen)
            loss.policy_loss(lp, gl, self.logits, self.chosen, self.old, self.advantage, grad_scale=64.0)
        return [rows, loss, lp, gl, self.table, self.room, self.grad]


@pytest.mark.parametrize("kind", ["float", "half"])
def test_steps_on_streams_of_their_own(thc, kind):
    hip = C.CDLL("libamdhip64.so")
    hip.hipStreamCreate.argtypes = [C.POINTER(C.c_void_p)]
    hip.hipStreamDestroy.argtypes = [C.c_void_p]
    hip.hipStreamSynchronize.argtypes = [C.c_void_p]
    want = [[x.numpy() for x in _Chain(thc, seed, kind).run()] for seed in (1, 2)]
    chains = [_Chain(thc, seed, kind) for seed in (1, 2)]      # made for the default stream, used on others
    thc.synchronize()
    got, errors = [None, None], []

    def worker(i):
        stream = C.c_void_p()
        try:
            assert hip.hipStreamCreate(C.byref(stream)) == 0
            thc.lib().THCState_setCurrentStream(thc.state(), stream)
            out = chains[i].run()
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
            assert_bit_equal(a, b, "chain %d, output %d" % (i, k))
