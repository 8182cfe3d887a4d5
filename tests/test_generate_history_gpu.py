"""Every attention call of a generation against 64-bit attention over a history
that is kept on the host: each beam's keys and values as its prompt's prefill and
its own steps produced them, following its parents.

So a wrong count of keys, a page that does not follow its beam, or a started page
copied in part shows in the call that reads it, within that call's own bounds
(those of tests/test_decode_gpu.py). A history that lacks one key must be told
apart at every length.
"""

import dataclasses

import numpy as np
import pytest
import torch

from quail_b200 import _native as nat
from quail_b200 import decode, generate
from quail_b200.api import B200Executor
from quail_b200.model import TINY
from tests.test_decode_gpu import Case, e4m3_value, e8m0_value, quantise64

pytestmark = pytest.mark.gpu


class History:
    def __init__(self, monkeypatch, ex, beams):
        self.ex, self.beams = ex, beams
        self.prompts, self.held, self.rows = [], None, None
        self.calls = self.steps = 0
        self.forward = generate.Generator._forward
        self.reorder, self.attention = decode.beam_reorder, decode.decode_attention
        monkeypatch.setattr(generate.Generator, "_forward",
                            lambda gen, *a: self.on_forward(gen, *a))
        monkeypatch.setattr(decode, "beam_reorder", self.on_reorder)
        monkeypatch.setattr(decode, "decode_attention", self.on_attention)

    def on_forward(self, gen, prompts, keys):
        """The prompts' keys and values, from the pages of their prefill."""
        result = self.forward(gen, prompts, keys)
        for key, prompt in zip(keys, prompts):
            at = torch.from_numpy(self.ex.arena.capacity_rows(key)[:len(prompt)]).cuda()
            layers = [[x[at].cpu().double() for x in self.ex.arena.layer_kv(layer)]
                      for layer in range(self.ex.cfg.n_layers)]
            if gen.kv == "fp8":
                layers = [[quantise64(x)[0] for x in kv] for kv in layers]
            self.prompts.append(layers)
        return result

    def on_reorder(self, pools, parents, used, table, **kw):
        if self.held is None:
            self.held = [p for p in self.prompts for _ in range(self.beams)]
        came = parents.cpu() + torch.arange(parents.shape[0])[:, None] * self.beams
        self.held = [[list(kv) for kv in self.held[int(i)]] for i in came.reshape(-1)]
        result = self.reorder(pools, parents, used, table, **kw)
        self.rows = result[1]
        self.steps += 1
        return result

    def on_attention(self, q, kv, table, used, *, softmax_scale, **kw):
        layer = self.calls % self.ex.cfg.n_layers
        self.calls += 1
        out = torch.empty_like(q)
        self.attention(q, kv, table, used, softmax_scale=softmax_scale, out=out, **kw)
        if len(kv) == 4:   # what the step wrote for its own token
            new = [e4m3_value(c.view(torch.uint8)[self.rows].view(torch.float8_e4m3fn))
                   * e8m0_value(s[self.rows])[..., None]
                   for c, s in ((kv.k, kv.k_scale), (kv.v, kv.v_scale))]
        else:
            new = [x[self.rows].cpu().double() for x in kv]
        for r, held in enumerate(self.held):
            held[layer] = [torch.cat([h, x[r:r + 1]]) for h, x in zip(held[layer], new)]
        case = Case.__new__(Case)
        case.kv, case.q, case.d, case.n_kv = kv, q, q.shape[2], self.ex.cfg.n_kv
        case.lengths = [held[layer][0].shape[0] for held in self.held]
        case.values = lambda r: [x.permute(1, 0, 2) for x in self.held[r][layer]]
        assert used.tolist() == case.lengths
        case.check(out, scale=softmax_scale)
        if self.steps % 6 == 0:   # one key less is seen
            for drop in (0, -2):
                case.values = lambda r: [
                    torch.cat([x[:drop], x[drop + 1:]]).permute(1, 0, 2)
                    for x in self.held[r][layer]]
                for r in range(len(self.held)):
                    with pytest.raises(AssertionError):
                        case.check(out, scale=softmax_scale, rows=[r])


@pytest.mark.parametrize("kv,beams", [("bf16", 1), ("fp8", 1), ("bf16", 4), ("fp8", 3)])
def test_attention_reads_each_beams_own_history(monkeypatch, kv, beams):
    ex = B200Executor(torch, dataclasses.replace(TINY, vocab=512), 400, seed=3)
    rng = np.random.default_rng(6)
    rows = [rng.integers(16, 500, n).tolist() for n in (1, 2, 15, 16, 17, 40, 131)]
    history = History(monkeypatch, ex, beams)
    out = ex.generate(rows, 20, beams=beams, kv=kv)
    assert history.steps == 19 and history.calls == 19 * ex.cfg.n_layers
    assert len(out) == len(rows) and nat.kernel_status(0) == 0
