"""Generation on one GPU: the example that runs its operators together.

``python -m quail_b200.generate_bench [--rows 64] [--prompt 300] [--new 32]
[--beams 1] [--kv bf16|fp8] [--scales fp32|ue8m0]`` continues seeded random
prompts on the random-init Qwen3-4B FP8 model (B200Executor.generate) and
prints one JSON line: the seconds of a whole call, and per step of new tokens
(from the times of this call and of one that generates a single token).
"""

import argparse
import json
import time

import numpy as np


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--rows", type=int, default=64)
    p.add_argument("--prompt", type=int, default=300)
    p.add_argument("--new", type=int, default=32)
    p.add_argument("--beams", type=int, default=1)
    p.add_argument("--kv", choices=["bf16", "fp8"], default="bf16")
    p.add_argument("--scales", choices=["fp32", "ue8m0"], default="ue8m0")
    args = p.parse_args(argv)
    import torch

    from quail_b200 import _native as nat
    from quail_b200.api import B200Executor
    from quail_b200.model import QWEN3_4B as cfg

    tokens = args.prompt + args.new
    pages = args.rows * (-(-tokens // 16) + (args.beams - 1) * (-(-args.new // 16) + 1)) + 16
    ex = B200Executor(torch, cfg, pages, scales=args.scales)
    rng = np.random.default_rng(0)
    prompts = rng.integers(1000, 150000, (args.rows, args.prompt)).tolist()

    def seconds(new):
        torch.cuda.synchronize()
        t = time.perf_counter()
        out = ex.generate(prompts, new, beams=args.beams, kv=args.kv)
        return time.perf_counter() - t, out
    seconds(2)                     # warm-up: allocator, kernels' first launches
    first, _ = seconds(1)
    total, out = seconds(args.new)
    assert len(out) == args.rows and len(out[0].tokens) == args.beams
    step = (total - first) / max(args.new - 1, 1)
    print(json.dumps(dict(
        model=cfg.name, data="synthetic", rows=args.rows, prompt=args.prompt, new=args.new,
        beams=args.beams, kv=args.kv, scales=args.scales, s=total, prefill_s=first,
        ms_per_step=1e3 * step, tokens_per_s=args.rows / step, status=nat.kernel_status())))


if __name__ == "__main__":
    main()
