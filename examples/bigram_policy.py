#!/usr/bin/env python3
"""A whole training step of a small language model out of the library's own operators: a bigram policy.

The logits of the next token are the last token's row of a table, times a factor. Each round samples continuations from the current
policy, rewards those that follow a hidden rule (the next token is the last one times 3 plus 1, modulo the vocabulary), and makes some steps of the clipped
policy loss with a KL term that keeps the policy near where it began:

    embedding -> policyLoss (losses, log-probabilities, gradient of the logits) -> embeddingGrad -> AdamW

    python examples/bigram_policy.py [--vocab 256] [--batch 4096] [--rounds 20] [--type float] [--bits 32]

prints the mean reward and the divergence from the first policy of every round.
"""
import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import cutorch_amd as thc  # noqa: E402

FACTOR = 4.0          # of the table's rows: their values stay small
LOSS_SCALE = 1024.0   # half gradients keep their small values


class Policy(object):
    """The table, in float or half with float copies, and what a step needs besides."""

    def __init__(self, vocab, kind, bits, rng):
        first = (0.02 * rng.standard_normal((vocab, vocab))).astype(np.float32)
        self.kind, self.vocab = kind, vocab
        self.master = thc.Tensor.from_numpy(first)
        self.table = thc.Tensor(kind).resize((vocab, vocab)).copy_from(self.master) if kind == "half" else self.master
        self.start = self.table.clone()
        self.grad = thc.Tensor(kind).resize((vocab, vocab)).zero()
        self.optimizer = thc.AdamW([self.table], [self.grad], master=[self.master] if kind == "half" else None, lr=0.02, beta2=0.99,
                                   weight_decay=0.0, bits=bits)
        self.logits, self.grad_logits = thc.Tensor(kind), thc.Tensor(kind)
        self.loss, self.log_prob = thc.Tensor("float"), thc.Tensor("float")

    def scores(self, tokens, table=None):
        return self.logits.embedding(table or self.table, tokens, FACTOR)

    def step(self, tokens, chosen, old, advantage, reference, weight):
        """One update; returns the loss."""
        self.scores(tokens)
        self.loss.policy_loss(self.log_prob, self.grad_logits, self.logits, chosen, old, advantage, reference, weight, kl=0.01,
                              grad_scale=LOSS_SCALE)
        self.grad.embedding_grad(tokens, self.grad_logits, FACTOR)
        self.optimizer.step(1.0 / LOSS_SCALE)
        return self.loss.sumall()


def train(vocab=256, batch=4096, rounds=20, kind="float", bits=32, seed=0, say=lambda *a: None):
    """The mean reward of every round."""
    rng = np.random.default_rng(seed)
    policy = Policy(vocab, kind, bits, rng)
    rewards = []
    for r in range(rounds):
        last = rng.integers(1, vocab + 1, batch)
        tokens = thc.Tensor.from_numpy(last)
        # the largest of logits plus Gumbel noise is a sample from their softmax
        noise = thc.Tensor.from_numpy(rng.gumbel(size=(batch, vocab)).astype(np.float16 if kind == "half" else np.float32))
        noisy, chosen = thc.Tensor(kind), thc.Tensor("long")
        noisy.cadd(policy.scores(tokens), 1, noise)
        thc.Tensor(kind).max(chosen, noisy, 1)
        chosen = chosen.view_as_strided(0, (batch,), (1,))
        picked = chosen.numpy()
        reward = ((picked - 1) == (3 * (last - 1) + 1) % vocab).astype(np.float32)
        reference = thc.Tensor("float").token_log_prob(policy.scores(tokens, policy.start), chosen)
        old = thc.Tensor("float").token_log_prob(policy.scores(tokens), chosen)
        # samples that get what is usual teach nothing; a tenth of the batch is kept out
        advantage = (reward - reward.mean()) / (reward.std() + 1e-6)
        kept = (rng.random(batch) < 0.9).astype(np.float32)
        weight = thc.Tensor.from_numpy(kept / max(1.0, kept.sum()))
        advantage = thc.Tensor.from_numpy(advantage.astype(np.float32))
        losses = [policy.step(tokens, chosen, old, advantage, reference, weight) for _ in range(4)]
        away = float(np.mean(old.numpy() - reference.numpy()))
        rewards.append(float(reward.mean()))
        say("round %2d  reward %.3f  losses %s  away from the start %.3f" % (r + 1, rewards[-1], " ".join("%7.4f" % x for x in losses), away))
    return rewards


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--vocab", type=int, default=256)
    ap.add_argument("--batch", type=int, default=4096)
    ap.add_argument("--rounds", type=int, default=20)
    ap.add_argument("--type", choices=("float", "half"), default="float")
    ap.add_argument("--bits", type=int, choices=(8, 32), default=32)
    a = ap.parse_args()
    train(a.vocab, a.batch, a.rounds, a.type, a.bits, say=print)


if __name__ == "__main__":
    main()
