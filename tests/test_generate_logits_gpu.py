"""The logits that generation chooses from keep 32 bits."""

import dataclasses

import numpy as np
import pytest
import torch

from quail_b200.api import B200Executor
from quail_b200.generate import Generator
from quail_b200.model import TINY

pytestmark = pytest.mark.gpu


def prompts(seed, lengths):
    rng = np.random.default_rng(seed)
    return [rng.integers(16, 500, n).tolist() for n in lengths]


@pytest.mark.parametrize("vocab", [512, 4096])
def test_logits_keep_32_bits(vocab):
    """The tied head in f32: products of bf16 numbers, summed in steps of 16 that
    truncate 17 terms at 2^-25 of the largest (2^-20.8 of the sum of magnitudes a
    step)."""
    ex = B200Executor(torch, dataclasses.replace(TINY, vocab=vocab), 64, seed=3)
    gen = Generator(ex)
    rows = prompts(1, [3, 20, 70])
    keys = gen._reserve(rows, 1, 1)
    normed = gen._prefill(rows, keys)
    gen._release(keys)
    got = gen.logits(normed)
    assert got.dtype == torch.float32
    x, w = normed.double(), ex.weights.embed.double()
    bound = ex.cfg.hidden / 16 * 2 ** -20.8 * (x.abs() @ w.abs().t())
    assert bool(((got.double() - x @ w.t()).abs() <= bound).all())
    # a token's score is its log-probability under them: the selection's own bound
    # (2^-19 and 2^-22 of the magnitudes) and twice the logits'
    out = ex.generate(rows, 1)
    exact = torch.log_softmax(x @ w.t(), -1)
    for i, o in enumerate(out):
        at = float(exact[i, o.tokens[0][0]])
        assert abs(o.scores[0] - at) <= 2 ** -19 + 2 ** -22 * (abs(at) + 32) + 2 * float(
            bound[i].max())
