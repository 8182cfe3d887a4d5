"""KVArena.evictable_pages: what evicting every retained key would free."""

import numpy as np
import pytest

from quail_b200.arena import KVArena


@pytest.mark.parametrize("seed", range(20))
def test_evictable_pages_are_what_eviction_frees(seed):
    rng = np.random.default_rng(seed)
    arena = KVArena(1, 200, 16, 1, 64, device=None)
    keys = []
    for i in range(int(rng.integers(1, 30))):
        borrow = None
        tokens = int(rng.integers(1, 100))
        if keys and rng.random() < 0.4:
            parent = keys[int(rng.integers(len(keys)))]
            shared = arena.tokens(parent) // 16 * 16
            if shared and shared <= tokens:
                borrow = (parent, shared)
        if arena.alloc(("d", i), tokens, borrow=borrow) is not None:
            keys.append(("d", i))
    for key in keys:
        if rng.random() < 0.6:
            arena.retain(key, arena.tokens(key))
            if rng.random() < 0.2:
                arena.hold(key, 1)
    expected, free = arena.evictable_pages(), arena.free_pages
    arena.evict_retained(arena.n_pages)
    assert arena.free_pages - free == expected
    assert arena.evictable_pages() == 0
