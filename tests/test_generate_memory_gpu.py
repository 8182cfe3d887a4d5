"""What generation takes and leaves on the GPU."""

import dataclasses
import gc
import weakref

import numpy as np
import pytest
import torch

from quail_b200.api import B200Executor
from quail_b200.model import TINY

pytestmark = pytest.mark.gpu

CFG = dataclasses.replace(TINY, vocab=512)


def prompts(seed, lengths):
    rng = np.random.default_rng(seed)
    return [rng.integers(16, 500, n).tolist() for n in lengths]


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
