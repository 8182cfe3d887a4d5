"""Decode attention on the GPU where keys are left out, against the formulas in
64 bits (the bounds are those of tests/test_decode_gpu.py).
"""

import math

import pytest
import torch

from quail_b200 import decode
from tests.test_decode_gpu import BAD_INDEX, Case, dev, status  # noqa: F401

pytestmark = pytest.mark.gpu


def behind_a_page(x, page, byte=None):
    """The pool behind one more page, whose rows hold NaN (or the byte)."""
    y = torch.empty(x.shape[0] + page, *x.shape[1:], dtype=x.dtype, device=x.device)
    y[page:] = x
    if byte is None:
        y[:page] = math.nan
    else:
        y.view(torch.uint8)[:page] = byte
    return y


@pytest.mark.parametrize("n_q,n_kv,d", [(4, 2, 128), (8, 1, 64), (32, 8, 128)])
@pytest.mark.parametrize("quant", [False, True])
def test_keys_of_bad_pages_are_left_out(dev, quant, n_q, n_kv, d):  # noqa: F811
    """Whatever the pool's first rows hold: here NaN, codes and scale bytes. A
    bad page at the start, in the middle, at the end; a row of bad pages only."""
    case = Case(dev, n_q, n_kv, d, [48, 300, 40, 33, 20, 64], quant=quant, seed=n_q + d)
    if quant:
        kv = decode.QuantLayer(
            *(behind_a_page(x.view(torch.uint8), 16, 0x7F).view(torch.float8_e4m3fn)
              for x in case.kv[:2]), *(behind_a_page(x, 16, 255) for x in case.kv[2:]))
    else:
        kv = tuple(behind_a_page(x, 16) for x in case.kv)
    table = case.table + 1
    bad = {0: [1], 1: [0, 7, 18], 2: [2], 3: [0, 1, 2]}
    for r, pages in bad.items():
        table[r, pages] = 10 ** 9 if r % 2 else -1
    out, lse = decode.decode_attention(case.q, kv, table, case.used, with_lse=True)
    assert status() == BAD_INDEX
    left = Case.__new__(Case)
    left.__dict__ = dict(case.__dict__)
    rows = [case.rows_of(r) for r in range(6)]
    for r, pages in bad.items():
        at = torch.arange(len(rows[r]), device=dev) // 16
        rows[r] = rows[r][~torch.isin(at, torch.tensor(pages, device=dev))]
    left.rows_of = lambda r: rows[r]
    left.lengths = [len(r) for r in rows]
    assert left.lengths[3] == 0
    left.check(out, lse)
