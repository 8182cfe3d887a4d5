"""Decode attention on the GPU where keys are left out or nearly cancel, against
the formulas in 64 bits (the bounds are those of tests/test_decode_gpu.py).

Where V's contributions cancel, the output is small beside sum w |v|, so its
rounding to bf16 hides nothing of the weights' own: a weight is off by
expm1(2 dx) against the normaliser, 2^-20 for the exponential and its rounding
for the second product, 2^-16 for a pair of bf16 or of f16 numbers (22 bits of
the latter, of which subnormals may drop some).
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


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("quant", [False, True])
def test_values_that_cancel(dev, quant, d):  # noqa: F811
    """Half of the keys weigh 1 and hold the value 1, the others weigh about 2/3
    and hold -3/2: the output is what the weights' rounding leaves."""
    n = 32
    case = Case(dev, 8, 1, d, [n], quant=quant, seed=3, spare=0)
    case.q[:] = 0
    case.q[:, :, 0] = 1.0
    odd = (torch.arange(n, device=dev) % 2).view(n, 1, 1)
    k = torch.zeros(n, 1, d, dtype=torch.bfloat16, device=dev)
    k[:, :, :1] = -odd.to(torch.bfloat16)
    v = torch.where(odd == 1, -1.5, 1.0).to(torch.bfloat16).expand(n, 1, d).contiguous()
    at = case.rows_of(0)
    if quant:
        decode.kv_quant_write(k, v, case.kv, at)
    else:
        case.kv[0][at], case.kv[1][at] = k, v
    for step in range(24):
        scale = math.log(1.5) + (step - 12) * 2.0 ** -11
        out = decode.decode_attention(case.q, case.kv, case.table, case.used,
                                      softmax_scale=scale)
        b = math.exp(-scale)
        want, size = (1 - 1.5 * b) / (1 + b), (1 + 1.5 * b) / (1 + b)
        dx = d / 16 * 2 ** -20.8 * scale
        dw = math.expm1(2 * dx) + 2 ** -16 + 2 ** -20 + (n / 16 + 32) * 2 ** -21
        bound = dw * size + 2 ** -8 * (1 + dw) * abs(want)
        assert float((out.double() - want).abs().max()) <= bound, (step, want, out[0, 0, :2])
    assert status() == 0
