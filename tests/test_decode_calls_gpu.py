"""The generation operators' calls in captured graphs, on other streams, over
pages that rows share, and on pools past 2^32 bytes."""

import pytest
import torch

from quail_b200 import decode
from tests.test_decode_gpu import Case, check_select, dev, reorder_by_hand, status  # noqa: F401

pytestmark = pytest.mark.gpu


class Inputs:
    """Inputs of the cache's and the beams' calls, in buffers that stay."""

    def __init__(self, dev, groups=3, beams=4, page=16):  # noqa: F811
        rows, width = groups * beams, 4
        self.page = page
        self.k, self.v = (torch.empty(24, 2, 64, dtype=torch.bfloat16, device=dev)
                          for _ in range(2))
        self.dst = torch.empty(24, dtype=torch.int64, device=dev)
        self.kv = decode.QuantKV(1, 4, page, 2, 64).layer_kv(0)
        self.logits = torch.empty(rows, 5003, device=dev)
        self.scores = torch.empty(groups, beams, device=dev)
        self.finished = torch.empty(groups, beams, dtype=torch.bool, device=dev)
        n_pages = rows * width
        self.table = torch.randperm(n_pages, device=dev).to(torch.int32).view(rows, width)
        self.used = torch.empty(groups, dtype=torch.int32, device=dev)
        self.pool = torch.empty(2, 2, n_pages * page, 2, 64, dtype=torch.bfloat16, device=dev)

    def fill(self, seed):
        g = torch.Generator(device=self.k.device).manual_seed(seed)
        for x in (self.k, self.v, self.logits, self.scores, self.pool):
            x.copy_(torch.randn(x.shape, generator=g, device=x.device))
        self.dst.copy_(torch.randperm(64, generator=g, device=self.k.device)[:24])
        self.finished.copy_(torch.rand(self.finished.shape, generator=g,
                                       device=self.k.device) < 0.3)
        self.used.copy_(torch.randint(0, 3 * self.page, self.used.shape, generator=g,
                                      device=self.k.device))

    def run(self):
        decode.kv_quant_write(self.k, self.v, self.kv, self.dst)
        back = decode.kv_quant_read(self.kv, self.dst)
        chosen = decode.beam_select(self.logits, self.scores, finished=self.finished, pad=7)
        moved = decode.beam_reorder((self.pool,), chosen[1], self.used, self.table,
                                    page_tokens=self.page)
        return [*back, *chosen, *moved, self.pool]


def test_cache_and_beams_in_a_graph(dev):  # noqa: F811
    """A replay answers for what its input buffers hold then, twice over."""
    x = Inputs(dev)
    x.fill(0)
    x.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = x.run()
    for seed in (1, 2, 1):
        x.fill(seed)
        want = [t.clone() for t in x.run()]
        x.fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        check_select(out[2:5], x.logits, x.scores, x.finished, 7)
    assert status() == 0


def test_cache_and_beams_on_other_streams(dev):  # noqa: F811
    """Two streams at a time, each with its own inputs and workspace."""
    sides = [(torch.cuda.Stream(), Inputs(dev)) for _ in range(2)]
    want = []
    for i, (_, x) in enumerate(sides):
        x.fill(10 + i)
        want.append([t.clone() for t in x.run()])
        x.fill(10 + i)
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for stream, x in sides:
            with torch.cuda.stream(stream):
                got.append(x.run())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            # (the pool moves on from pass to pass)
            assert all(torch.equal(s, t) for s, t in zip(a[:-1], b[:-1]))
    assert status() == 0


@pytest.mark.parametrize("quant", [False, True])
def test_decode_attention_rows_that_share_pages(dev, quant):  # noqa: F811
    """Beams of a row: the same full pages in several tables, own last ones."""
    case = Case(dev, 32, 8, 128, [330, 331, 322, 335, 40, 33], quant=quant, seed=21)
    case.table[1:4, :20] = case.table[0, :20]
    case.table[5, :2] = case.table[4, :2]
    out, lse = decode.decode_attention(case.q, case.kv, case.table, case.used, with_lse=True)
    assert status() == 0
    case.check(out, lse)


@pytest.mark.parametrize("quant", [False, True])
def test_beam_reorder_past_32_bit_offsets(dev, quant):  # noqa: F811
    """Slabs of over 2^32 bytes, the pages that move at both ends."""
    page, n_kv, d = 64, 8, 128
    n_pages = 2 ** 32 // (page * n_kv * d * (1 if quant else 2)) + 8
    if quant:
        kv = decode.QuantKV(1, n_pages, page, n_kv, d)
        pools = kv.pools
    else:
        pools = (torch.empty(1, 2, n_pages * page, n_kv, d, dtype=torch.bfloat16, device=dev),)
    ids = [0, n_pages - 1, n_pages - 2, 1]      # the beams' started pages
    table = torch.tensor([[i] for i in ids], dtype=torch.int32)
    near = [torch.arange(p * page, (p + 1) * page) for p in ids]
    at = torch.cat(near).to(dev)
    g = torch.Generator(device=dev).manual_seed(5)
    small = []
    for pool in pools:
        raw = pool.view(torch.uint8)
        raw[:, :, at] = torch.randint(0, 100, (1, 2, len(at), *raw.shape[3:]), generator=g,
                                      device=dev, dtype=torch.uint8)
        small.append(raw[:, :, at].cpu())
    parents = torch.tensor([[1, 1, 3, 3]], dtype=torch.int32)
    used = [37]
    # by hand over the four pages alone
    held = [(s, s.clone()) for s in small]
    want, _ = reorder_by_hand(held, parents, used, torch.arange(4, dtype=torch.int32)[:, None],
                              page)
    got, rows = decode.beam_reorder(pools, parents.to(dev),
                                    torch.tensor(used, dtype=torch.int32, device=dev),
                                    table.to(dev), page_tokens=page)
    assert status() == 0
    assert got[:, 0].tolist() == [ids[i] for i in want[:, 0].tolist()]
    assert rows.tolist() == [i * page + 37 for i in got[:, 0].tolist()]
    for pool, (_, new) in zip(pools, held):
        assert torch.equal(pool.view(torch.uint8)[:, :, at].cpu(), new)
