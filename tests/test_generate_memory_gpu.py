"""What generation takes and leaves on the GPU: the arena's pages, the 8-bit
cache's memory and the executor's own lifetime."""

import dataclasses
import gc
import weakref

import numpy as np
import pytest
import torch

from quail_b200 import _native as nat
from quail_b200.api import B200Executor
from quail_b200.generate import Generator
from quail_b200.model import TINY

pytestmark = pytest.mark.gpu

CFG = dataclasses.replace(TINY, vocab=512)


def prompts(seed, lengths):
    rng = np.random.default_rng(seed)
    return [rng.integers(16, 500, n).tolist() for n in lengths]


def test_an_8_bit_cache_holds_twice_the_tokens():
    """Rows whose bf16 pages would take one and a half times the arena."""
    ex = B200Executor(torch, CFG, 60, seed=3)
    rows = prompts(2, [64] * 15)          # 15 x 6 pages
    with pytest.raises(RuntimeError, match="short of pages"):
        ex.generate(rows, 20)
    wide = B200Executor(torch, CFG, 400, weights=ex.weights)
    want = wide.generate(rows, 20, kv="fp8")
    got = ex.generate(rows, 20, kv="fp8")
    assert ex.arena.free_pages == 60 and nat.kernel_status(0) == 0
    # (chunks of other sizes: the same kernels on the same rows)
    for a, b in zip(got, want):
        assert a.tokens == b.tokens and a.scores == b.scores


@pytest.mark.parametrize("beams", [1, 3])
def test_8_bit_generation_needs_no_second_arena(beams):
    """Beside the arena: the codes' scale bytes (1 / head_dim of its bytes), the
    workspace, and the passes' own tensors, a few MB at these sizes."""
    ex = B200Executor(torch, CFG, 16384, seed=3)
    arena = ex.arena.pools.numel() * 2
    rows = prompts(3, [40, 7, 90])
    ex.generate(rows, 4, beams=beams)                 # the passes' tensors, cached
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ex.generate(rows, 20, beams=beams, kv="fp8")
    peak = torch.cuda.max_memory_allocated() - before
    assert peak <= arena / CFG.head_dim + (16 << 20), (peak, arena)
    # and nothing of it stays (but the stream's own workspaces)
    assert torch.cuda.memory_allocated() - before <= 4 << 20


@pytest.mark.parametrize("lengths,beams", [([64], 1), ([50, 64], 1), ([30], 2)])
def test_8_bit_generation_in_an_arena_of_its_bf16_pages(lengths, beams):
    """Few rows, whose bf16 pages are all the arena has: those that the arena
    cannot hold in 8 bits beside a prompt's bf16 pages run all the same."""
    rows = prompts(9, lengths)
    pages = sum(n // 16 + beams * (-(-(n + 20) // 16) - n // 16) for n in lengths)
    ex = B200Executor(torch, CFG, pages, seed=3)
    wide = B200Executor(torch, CFG, 400, weights=ex.weights)
    got = ex.generate(rows, 20, beams=beams, kv="fp8")
    want = wide.generate(rows, 20, beams=beams, kv="fp8")
    assert [(o.tokens, o.scores) for o in got] == [(o.tokens, o.scores) for o in want]
    assert ex.arena.free_pages == pages and nat.kernel_status(0) == 0


def test_a_generator_serves_calls_of_either_place():
    """One generator, its cache in the arena, beside it, and in it again; a
    refusal between them."""
    ex = B200Executor(torch, CFG, 12, seed=3)
    gen = Generator(ex, "fp8")
    small, large = prompts(10, [16, 20, 9]), prompts(11, [150])
    want = gen.generate(small, 6)
    first = gen.generate(large, 20)
    with pytest.raises(RuntimeError, match="short of pages"):
        gen.generate(large * 2, 20)
    assert gen.quant is None and ex.arena.free_pages == 12
    assert [o.tokens for o in gen.generate(small, 6)] == [o.tokens for o in want]
    assert gen.generate(large, 20)[0].tokens == first[0].tokens


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_an_executor_ends_with_its_last_reference(kv):
    gc.collect()
    gc.disable()
    try:
        ex = B200Executor(torch, CFG, 64, seed=3)
        ex.generate(prompts(4, [20, 5]), 4, kv=kv)
        gone = weakref.ref(ex)
        del ex
        assert gone() is None
    finally:
        gc.enable()


def retained(ex, n, tokens, alias="doc"):
    for i in range(n):
        assert ex.arena.alloc((alias, i), tokens) is not None
        ex.arena.retain((alias, i), tokens)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_retained_keys_give_way(kv):
    """Keys kept for a later operator are evicted, as few as needed, where the
    arena is short; pinned ones are not."""
    ex = B200Executor(torch, CFG, 60, seed=3)
    rows = prompts(5, [64, 64])           # 6 pages each in bf16
    want = ex.generate(rows, 20, kv=kv)
    retained(ex, 15, 62)                  # 4 pages each: the arena is full
    assert ex.arena.free_pages == 0
    got = ex.generate(rows, 20, kv=kv)
    assert [o.tokens for o in got] == [o.tokens for o in want]
    # bf16: 12 pages; 8 bit: 6, and 4 for a prompt on its way through
    assert len(ex.arena.retained_keys()) == 12 and ex.arena.free_pages == 12
    for key in ex.arena.retained_keys():
        ex.arena.pin(key)
    held = ex.arena.free_pages
    with pytest.raises(RuntimeError, match="short of pages"):
        ex.generate(rows * 4, 20, kv=kv)
    assert ex.arena.free_pages == held
    ex.arena.reset()


def test_nothing_is_evicted_for_rows_that_never_fit():
    ex = B200Executor(torch, CFG, 60, seed=3)
    retained(ex, 5, 62)
    for key in [("doc", 0), ("doc", 1)]:
        ex.arena.pin(key)
    with pytest.raises(RuntimeError, match="short of pages"):
        ex.generate(prompts(6, [64] * 9), 20)        # 54 pages of at most 52
    assert len(ex.arena.retained_keys()) == 3
    ex.arena.reset()


def test_generation_after_a_filter_that_retains():
    """Through the executor's own calls: a filter keeps its survivors' KV in a
    nearly full arena, generation takes their pages."""
    ex = B200Executor(torch, CFG, 48, seed=3)
    docs = prompts(7, [60] * 10)          # 4 pages each
    result = ex.filter(docs, [[7]], keys=[("t", i) for i in range(10)], retain_survivors=True,
                       budget=128)
    kept = len(ex.arena.retained_keys())
    assert kept == int(result.bits.sum()) and ex.arena.free_pages == 48 - 4 * kept
    out = ex.generate(prompts(8, [64] * 7), 20)      # 42 pages
    assert len(out) == 7
    assert len(ex.arena.retained_keys()) <= 1
    ex.arena.reset()
