"""Generation end to end on the GPU: the tokens and scores of B200Executor.
generate against the prefill's own logits for the same tokens.

The prefill computes a token's attention in another kernel (bf16 weights in
its second product, another order of sums), and each layer re-quantises to
e4m3, so log-probabilities agree to the differences that two correct
roundings show on a two-layer model: at most 0.2 (0.16 was measured between
this library and fp32-BLAS semantics for the difference of two logits). The
8-bit cache adds its own rounding of K and V (2^-4 relative at most, 2^-5.5
rms): 0.5.
"""

import dataclasses

import numpy as np
import pytest
import torch

from quail_b200 import _native as nat
from quail_b200.api import B200Executor
from quail_b200.model import TINY

pytestmark = pytest.mark.gpu

TOL = {"bf16": 0.2, "fp8": 0.5}


@pytest.fixture(scope="module", params=["fp32", "ue8m0"])
def executor(request):
    return B200Executor(torch, dataclasses.replace(TINY, vocab=512), 400, seed=3,
                        scales=request.param)


def prompts(seed, lengths):
    rng = np.random.default_rng(seed)
    return [rng.integers(16, 500, n).tolist() for n in lengths]


def log_probs(ex, rows):
    """log-softmax (64 bits) of the next token after each row, by prefill."""
    from quail_b200.generate import Generator
    gen = Generator(ex)
    keys = gen._reserve(rows, 1, 1)
    try:
        return torch.log_softmax(gen.logits(gen._prefill(rows, keys)).double(), -1).cpu()
    finally:
        gen._release(keys)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_greedy_follows_the_prefill(executor, kv):
    rows = prompts(1, [1, 2, 15, 16, 17, 40, 131])
    free = executor.arena.free_pages
    out = executor.generate(rows, 20, kv=kv)
    assert executor.arena.free_pages == free
    assert nat.kernel_status(0) == 0
    total = [0.0] * len(rows)
    for t in range(20):
        lp = log_probs(executor, [r + o.tokens[0][:t] for r, o in zip(rows, out)])
        for i, o in enumerate(out):
            assert len(o.tokens) == 1 and len(o.tokens[0]) == 20
            token = o.tokens[0][t]
            total[i] += float(lp[i, token])
            assert float(lp[i].max() - lp[i, token]) <= TOL[kv], (i, t)
    for i, o in enumerate(out):
        assert abs(o.scores[0] - total[i]) <= 20 * TOL[kv] / 4, i


@pytest.mark.parametrize("kv,beams", [("bf16", 4), ("fp8", 3), ("bf16", 8)])
def test_beam_scores_are_their_tokens(executor, kv, beams):
    rows = prompts(2, [5, 33, 64, 100])
    steps = 18
    out = executor.generate(rows, steps, beams=beams, kv=kv)
    assert nat.kernel_status(0) == 0
    for o in out:
        assert len({tuple(t) for t in o.tokens}) == beams          # beams differ
        assert o.scores == sorted(o.scores, reverse=True)
    flat = [(r, t) for r, o in zip(rows, out) for t in o.tokens]
    total = np.zeros(len(flat))
    for t in range(steps):
        lp = log_probs(executor, [r + tokens[:t] for r, tokens in flat])
        total += [float(lp[i, tokens[t]]) for i, (_, tokens) in enumerate(flat)]
    scores = np.array([s for o in out for s in o.scores])
    # the differences of single steps are independent in sign: a quarter of
    # their bound a step
    assert np.abs(scores - total).max() <= steps * TOL[kv] / 4
    greedy = executor.generate(rows, steps, kv=kv)
    for o, g in zip(out, greedy):
        assert o.scores[0] >= g.scores[0] - steps * TOL[kv] / 4


def test_more_beams_than_one_step_of_plain_search(executor):
    """Three steps of beam search by hand over the prefill's log-probabilities
    give the same best score."""
    rows, beams = prompts(5, [30, 47]), 5
    out = executor.generate(rows, 3, beams=beams)
    for row, o in zip(rows, out):
        held = [((), 0.0)]
        for _ in range(3):
            lp = log_probs(executor, [row + list(t) for t, _ in held])
            every = [(t + (v,), s + float(lp[i, v])) for i, (t, s) in enumerate(held)
                     for v in range(lp.shape[1])]
            held = sorted(every, key=lambda e: -e[1])[:beams]
        assert abs(held[0][1] - o.scores[0]) <= 3 * TOL["bf16"] / 2


def test_ending_token(executor):
    rows = prompts(3, [20, 21])
    plain = executor.generate(rows, 12)
    eos = plain[0].tokens[0][4]
    out = executor.generate(rows, 40, eos=eos)
    first = plain[0].tokens[0].index(eos)
    assert out[0].tokens[0] == plain[0].tokens[0][:first + 1]
    assert eos not in out[1].tokens[0][:-1]
    wide = executor.generate(rows, 12, beams=4, eos=eos)
    for o in wide:
        for tokens in o.tokens:
            assert eos not in tokens[:-1]


def test_refusals(executor):
    with pytest.raises(ValueError, match="empty prompt"):
        executor.generate([[1], []], 4)
    with pytest.raises(ValueError, match="beams"):
        executor.generate([[1]], 4, beams=33)
    with pytest.raises(ValueError, match="rotary"):
        executor.generate([[1]], TINY.max_pos)
    with pytest.raises(ValueError, match="kv"):
        executor.generate([[1]], 4, kv="int4")
    free = executor.arena.free_pages
    with pytest.raises(RuntimeError, match="short of pages"):
        executor.generate(prompts(4, [100] * 100), 100, beams=8)
    assert executor.arena.free_pages == free
    assert executor.generate([], 4) == []
