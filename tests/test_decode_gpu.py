"""The generation operators on the GPU against plain implementations in 64
bits: decode attention, the 8-bit KV cache, beam selection and reordering.

Bounds. u is the unit roundoff of the format a value is rounded to.
- Attention: x = q . k comes from D / 16 tensor-core steps, each of which
  truncates 17 terms at 2^-25 of the largest and rounds its sum toward zero:
  |dx| <= D / 16 * 2^-20.8 * X with X = max_i sum_d |q_d k_id| * scale (the
  model pinned in tests/test_oracle_model.py). A weight e^x is then off by
  expm1(2 dx) against the normaliser, by its rounding for the second product
  (2^-11 in f16, 2^-16 as a bf16 pair) and by 2^-20 for the exponential; the
  sums over n keys add (n / 16 + 32) 2^-21 of sum w |v|. The output is rounded
  to bf16 (u = 2^-8).
- The log-sum-exp: dx, the sum's (n / 16 + 32) 2^-23 and 2^-22 |lse|.
- The cache: codes and scale bytes are defined exactly, so equality.
- Beams: lse from fp32 terms, each within 2^-21, summed in chunks:
  2^-19 + 2^-23 |lse|; a score adds two roundings of its own size.
"""

import math

import numpy as np
import pytest
import torch

from quail_b200 import _native as nat
from quail_b200 import decode
from quail_b200.engine import QuantRows

pytestmark = pytest.mark.gpu

BAD_INDEX = 1 << 9


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda")


def status():
    return nat.kernel_status(torch.cuda.current_device())


def e4m3_value(codes):
    return codes.contiguous().view(torch.uint8).cpu().view(torch.float8_e4m3fn).double()


def e8m0_value(byte):
    b = byte.cpu().to(torch.int64)
    x = torch.ldexp(torch.ones(b.shape, dtype=torch.float64), b - 127)
    x[b == 255] = math.nan
    return x


def quantise64(x):
    """(value, scale byte) by the definition, in 64 bits, over the last axis."""
    x = x.double().cpu().numpy()
    amax = np.abs(x).max(-1)
    with np.errstate(all="ignore"):
        m, e = np.frexp(np.maximum(amax, 1e-10) / 448.0)
        e = np.where(m == 0.5, e - 1, e)
        byte = np.where(np.isfinite(amax), e + 127, 255).astype(np.int64)
        unit = np.ldexp(1.0, np.where(np.isfinite(amax), e, 0))[..., None]
        y = x / unit
        _, ey = np.frexp(np.maximum(np.abs(y), 2.0 ** -6))
        step = np.ldexp(1.0, ey - 1 - 3)
        y = np.round(y / step) * step * unit       # numpy rounds halves to even
        y[~np.isfinite(amax)] = math.nan
    return torch.from_numpy(y), torch.from_numpy(byte)


# ---- the 8-bit cache -------------------------------------------------------------


@pytest.mark.parametrize("rows,n_kv,d", [(1, 8, 128), (64, 8, 128), (131, 2, 64), (37, 3, 64),
                                         (9, 1, 128), (5, 5, 128), (300, 1, 64)])
def test_kv_quant_round_trip(dev, rows, n_kv, d):
    g = torch.Generator(device=dev).manual_seed(rows * d + n_kv)
    k = torch.randn(rows, n_kv, d, generator=g, device=dev)
    k *= torch.exp(8 * torch.randn(rows, n_kv, 1, generator=g, device=dev))
    v = torch.randn(rows, n_kv, d, generator=g, device=dev)
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    kv = decode.QuantKV(2, 2 * (rows // 16 + 1), 16, n_kv, d)
    kv.codes.view(torch.uint8).fill_(0x7F)
    kv.scales.fill_(77)
    layer = kv.layer_kv(1)
    dst = torch.randperm(layer.k.shape[0], generator=g, device=dev)[:rows]
    decode.kv_quant_write(k, v, layer, dst)
    got_k, got_v = decode.kv_quant_read(layer, dst)
    assert status() == 0
    for x, codes, scale, got in ((k, layer.k, layer.k_scale, got_k),
                                 (v, layer.v, layer.v_scale, got_v)):
        want, byte = quantise64(x)
        assert torch.equal(scale[dst].cpu().long(), byte)
        held = e4m3_value(codes.view(torch.uint8)[dst].view(torch.float8_e4m3fn))
        assert torch.equal(held * e8m0_value(scale[dst])[..., None], want)
        assert torch.equal(got.cpu().double(), want)
    # nothing else was written
    others = torch.ones(layer.k.shape[0], dtype=torch.bool, device=dev)
    others[dst] = False
    assert bool((layer.k.view(torch.uint8)[others] == 0x7F).all())
    assert bool((layer.v_scale[others] == 77).all())
    assert bool((kv.scales[0] == 77).all())


def test_kv_quant_special_values(dev):
    """Zeros, values far below the scale floor, bf16's largest, infinities and
    NaN; a head that is not finite poisons itself and no other."""
    n_kv, d = 2, 64
    rows = 9
    k = torch.zeros(rows, n_kv, d, dtype=torch.bfloat16)
    k[1] = 1e-30
    k[2, 0, 3] = -1e-12
    k[3, 1, :] = 448.0
    k[4, 0, :] = 449.0          # bf16 450: one step over 448
    k[5, 0, 7] = math.inf
    k[5, 1, 7] = 5.0
    k[6, 1, 0] = math.nan
    k[6, 0, 0] = -3.0
    k[7, 0, 0] = 1.5 * 2.0 ** 127
    k[7, 0, 1] = 2.0 ** 120
    k[8, :, :] = torch.arange(d) * 2.0 ** -12 - 0.001
    v = k.flip(0)
    kv = decode.QuantKV(1, 2, 16, n_kv, d).layer_kv(0)
    dst = torch.arange(rows, device=dev) + 3
    decode.kv_quant_write(k.to(dev), v.to(dev), kv, dst)
    got = decode.kv_quant_read(kv, dst)
    assert status() == 0
    for x, y in zip((k, v), got):
        want, _ = quantise64(x)
        assert torch.equal(torch.isnan(want), torch.isnan(y.cpu()))
        fine = ~torch.isnan(want)
        assert torch.equal(y.cpu().double()[fine], want[fine])
    assert int(kv.k_scale[dst[5], 0]) == 255 and int(kv.k_scale[dst[5], 1]) != 255


def test_kv_quant_sources_strides_and_skips(dev):
    """k and v as slices of a projection, chosen source rows, negative
    destinations on both ways."""
    n_kv, d, rows = 2, 128, 50
    g = torch.Generator(device=dev).manual_seed(4)
    qkv = torch.randn(rows, (4 + 2 * 2) * d, generator=g, device=dev).to(torch.bfloat16)
    k = qkv[:, 4 * d:6 * d].view(rows, n_kv, d)
    v = qkv[:, 6 * d:].view(rows, n_kv, d)
    kv = decode.QuantKV(1, 8, 16, n_kv, d).layer_kv(0)
    kv.k_scale.fill_(1)
    src = torch.randperm(rows, generator=g, device=dev)[:21]
    dst = torch.randperm(128, generator=g, device=dev)[:21]
    dst[::4] = -1
    decode.kv_quant_write(k, v, kv, dst, src=src)
    kept = dst >= 0
    assert int((kv.k_scale != 1).any(1).sum()) == int(kept.sum())
    k_out = torch.full((30, n_kv, d), 7.0, dtype=torch.bfloat16, device=dev)
    v_out = torch.full_like(k_out, 7.0)
    to = torch.randperm(30, generator=g, device=dev)[:int(kept.sum())]
    to[3] = -2
    decode.kv_quant_read(kv, dst[kept], dst=to, out=(k_out, v_out))
    assert status() == 0
    want_k, _ = quantise64(k[src[kept]])
    want_v, _ = quantise64(v[src[kept]])
    on = (to >= 0).cpu()
    assert torch.equal(k_out[to[to >= 0]].cpu().double(), want_k[on])
    assert torch.equal(v_out[to[to >= 0]].cpu().double(), want_v[on])
    rest = torch.ones(30, dtype=torch.bool)
    rest[to[to >= 0].cpu()] = False
    assert bool((k_out.cpu()[rest] == 7).all())


def test_kv_quant_bad_rows_are_flagged_and_skipped(dev):
    kv = decode.QuantKV(1, 2, 16, 1, 128).layer_kv(0)
    kv.k_scale.fill_(9)
    k = torch.ones(3, 1, 128, dtype=torch.bfloat16, device=dev)
    decode.kv_quant_write(k, k, kv, torch.tensor([0, 32, 1], device=dev))
    assert status() == BAD_INDEX
    decode.kv_quant_write(k, k, kv, torch.tensor([2, 4], device=dev),
                          src=torch.tensor([0, 3], device=dev))
    assert status() == BAD_INDEX
    assert [int(i) for i in (kv.k_scale != 9).nonzero()[:, 0]] == [0, 1, 2]
    got, _ = decode.kv_quant_read(kv, torch.tensor([0, 32, -1], device=dev))
    assert status() == BAD_INDEX
    assert bool((got[0] == 1).all()) and bool((got[1:] == 0).all())


def test_kv_quant_empty(dev):
    kv = decode.QuantKV(1, 1, 16, 2, 64).layer_kv(0)
    none = torch.empty(0, dtype=torch.int64, device=dev)
    k = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=dev)
    decode.kv_quant_write(k, k, kv, none)
    assert decode.kv_quant_read(kv, none)[0].shape == (0, 2, 64)
    assert status() == 0


# ---- decode attention ------------------------------------------------------------


class Case:
    def __init__(self, dev, n_q, n_kv, d, lengths, page=16, quant=False, seed=0, gain=2.0,
                 spare=3):
        g = torch.Generator(device=dev).manual_seed(seed)
        rows = len(lengths)
        self.lengths, self.page, self.n_kv, self.d = lengths, page, n_kv, d
        per = [-(-n // page) for n in lengths]
        n_pages = sum(per) + spare
        order = torch.randperm(n_pages, generator=g, device=dev).tolist()
        self.table = torch.zeros(rows, max(max(per), 1), dtype=torch.int32)
        for r, c in enumerate(per):
            self.table[r, :c] = torch.tensor(order[:c], dtype=torch.int32)
            order = order[c:]
        self.table = self.table.to(dev)
        self.used = torch.tensor(lengths, dtype=torch.int32, device=dev)
        self.q = (gain * torch.randn(rows, n_q, d, generator=g, device=dev)).to(torch.bfloat16)
        pools = [torch.randn(n_pages * page, n_kv, d, generator=g, device=dev)
                 * torch.exp(torch.randn(n_pages * page, n_kv, 1, generator=g, device=dev))
                 for _ in range(2)]
        pools[0] = torch.clamp(pools[0], -6, 6)
        # whatever the tables do not reach, or reach past a row's end, is NaN
        seen = torch.zeros(n_pages * page, dtype=torch.bool, device=dev)
        for r in range(rows):
            seen[self.rows_of(r)] = True
        if quant:
            kv = decode.QuantKV(1, n_pages, page, n_kv, d)
            layer = kv.layer_kv(0)
            decode.kv_quant_write(pools[0].to(torch.bfloat16), pools[1].to(torch.bfloat16),
                                  layer, torch.arange(n_pages * page, device=dev))
            for c, s in ((layer.k, layer.k_scale), (layer.v, layer.v_scale)):
                c.view(torch.uint8)[~seen] = 0x7F
                s[~seen] = 255
            self.kv = layer
        else:
            self.kv = tuple(x.to(torch.bfloat16) for x in pools)
            for x in self.kv:
                x[~seen] = math.nan

    def rows_of(self, r):
        i = torch.arange(self.lengths[r], device=self.table.device)
        return self.table[r].long()[i // self.page] * self.page + i % self.page

    def values(self, r):
        """K and V of a row's keys in 64 bits, [n_kv, n, d]."""
        at = self.rows_of(r)
        if isinstance(self.kv, decode.QuantLayer):
            out = [(e4m3_value(c.view(torch.uint8)[at].view(torch.float8_e4m3fn))
                    * e8m0_value(s[at])[..., None])
                   for c, s in ((self.kv.k, self.kv.k_scale), (self.kv.v, self.kv.v_scale))]
        else:
            out = [x[at].cpu().double() for x in self.kv]
        return [x.permute(1, 0, 2) for x in out]

    def check(self, out, lse=None, scale=None, rows=None, rounded=True):
        rows = range(len(self.lengths)) if rows is None else rows
        scale = self.d ** -0.5 if scale is None else scale
        for r in rows:
            n = self.lengths[r]
            if n == 0:
                assert bool((out[r] == 0).all())
                assert lse is None or bool((lse[r] == -math.inf).all())
                continue
            k, v = self.values(r)
            q = self.q[r].cpu().double().view(self.n_kv, -1, self.d)
            z = (q @ k.transpose(1, 2)) * scale
            w = torch.softmax(z, -1)
            want = (w @ v).reshape(-1, self.d)
            size = (w @ v.abs()).reshape(-1, self.d)
            x = (q.abs() @ k.abs().transpose(1, 2)).amax(-1).reshape(-1, 1) * abs(scale)
            dx = self.d / 16 * 2 ** -20.8 * x
            quant = isinstance(self.kv, decode.QuantLayer)
            dw = (torch.expm1(2 * dx) + (2 ** -11 if quant else 2 ** -16) + 2 ** -20
                  + (n / 16 + 32) * 2 ** -21)
            bound = dw * size + (2 ** -8 * (1 + dw) * want.abs() if rounded else 0)
            err = (out[r].cpu().double() - want).abs()
            assert bool((err <= bound).all()), (r, n, float((err / bound).max()))
            if lse is not None:
                exact = torch.logsumexp(z, -1).reshape(-1, 1)
                tol = dx + (n / 16 + 32) * 2 ** -23 + 2 ** -22 * exact.abs()
                off = (lse[r].cpu().double().reshape(-1, 1) - exact).abs()
                assert bool((off <= tol).all()), (r, n, float((off / tol).max()))


LENGTHS = [1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 64, 0, 127, 128, 129, 255, 300, 1000]


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("n_q,n_kv,d,page", [
    (32, 8, 128, 16), (8, 1, 128, 16), (4, 2, 64, 16), (6, 2, 128, 32), (5, 1, 64, 8),
    (1, 1, 128, 64), (3, 3, 64, 16), (24, 2, 128, 16), (17, 1, 64, 32), (7, 7, 128, 8)])
def test_decode_attention(dev, n_q, n_kv, d, page, quant):
    case = Case(dev, n_q, n_kv, d, LENGTHS, page=page, quant=quant, seed=n_q + d + page)
    out, lse = decode.decode_attention(case.q, case.kv, case.table, case.used, page_tokens=page,
                                       with_lse=True)
    assert status() == 0
    case.check(out, lse)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("lengths", [[20011], [5000, 1, 9000], [4096] * 40, [16] * 700, [0, 0, 0],
                                     [33000, 0, 3] + [50] * 60])
def test_decode_attention_lengths(dev, lengths, quant):
    case = Case(dev, 8, 2, 128, lengths, quant=quant, seed=len(lengths))
    out, lse = decode.decode_attention(case.q, case.kv, case.table, case.used, with_lse=True)
    assert status() == 0
    rows = range(len(lengths)) if len(lengths) < 50 else (0, 1, 2, len(lengths) // 2,
                                                          len(lengths) - 1)
    case.check(out, lse, rows=rows)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("n_q,d,lengths", [(8, 128, [40000]), (9, 64, [21000, 5]),
                                           (3, 128, [600, 7000, 129] * 9)])
def test_decode_attention_items_that_many_blocks_share(dev, n_q, d, lengths, quant):
    """One KV head: a long row's parts come from every block."""
    case = Case(dev, n_q, 1, d, lengths, quant=quant, seed=n_q)
    out, lse = decode.decode_attention(case.q, case.kv, case.table, case.used, with_lse=True)
    assert status() == 0
    case.check(out, lse)


@pytest.mark.parametrize("quant", [False, True])
def test_decode_attention_sharp_and_flat_rows(dev, quant):
    """Keys that raise the running maximum at each step, one key far above the
    rest at either end, and products that are all equal."""
    n = 700
    case = Case(dev, 8, 2, 128, [n] * 4, quant=False, seed=5, gain=0.5)
    k, v = case.kv
    for r, size in ((0, torch.linspace(-8, 8, n)), (1, torch.linspace(8, -8, n)),
                    (2, torch.where(torch.arange(n) == n - 1, 30.0, 0.0))):
        at = case.rows_of(r)
        direction = case.q[r].view(2, 4, 128)[:, 0].float()
        k[at] = (size.to(dev)[:, None, None] * direction).to(torch.bfloat16)
    case.q[3] = 0
    if quant:
        layer = decode.QuantKV(1, k.shape[0] // 16, 16, 2, 128).layer_kv(0)
        decode.kv_quant_write(torch.nan_to_num(k), torch.nan_to_num(v), layer,
                              torch.arange(k.shape[0], device=dev))
        case.kv = layer
    out, lse = decode.decode_attention(case.q, case.kv, case.table, case.used, with_lse=True)
    assert status() == 0
    case.check(out, lse)


def test_decode_attention_value_scales_apart(dev):
    """8-bit values whose scales differ by 2^40 between keys, the large ones on
    keys of little weight and of much."""
    case = Case(dev, 4, 1, 128, [200, 200], quant=True, seed=8, gain=1.0)
    layer = case.kv
    at = case.rows_of(0)
    layer.v_scale[at[::3], 0] += 20
    layer.v_scale[at[1::3], 0] -= 20
    at = case.rows_of(1)
    layer.v_scale[at[150], 0] += 40
    out, lse = decode.decode_attention(case.q, layer, case.table, case.used, with_lse=True)
    assert status() == 0
    case.check(out, lse)


def test_decode_attention_extreme_queries(dev):
    """Queries of 2^60 and 2^-60 (the 8-bit path scales them into f16)."""
    for quant in (False, True):
        case = Case(dev, 8, 2, 128, [100, 100, 100], quant=quant, seed=9)
        case.q[0] = (case.q[0].float() * 2.0 ** 60).to(torch.bfloat16)
        case.q[1] = (case.q[1].float() * 2.0 ** -60).to(torch.bfloat16)
        out, lse = decode.decode_attention(case.q, case.kv, case.table, case.used,
                                           softmax_scale=2.0 ** -60, with_lse=True)
        case.check(out[:1], lse[:1], scale=2.0 ** -60, rows=[0])
        out, lse = decode.decode_attention(case.q, case.kv, case.table, case.used, with_lse=True)
        case.check(out, lse, rows=[1, 2])


def test_decode_attention_not_finite(dev):
    """-inf products leave a row empty; NaN keys, values and scales show."""
    case = Case(dev, 2, 1, 64, [20, 20, 20, 20], seed=2)
    k, v = case.kv
    case.q[0] = 1.0
    k[case.rows_of(0)] = -math.inf
    k[case.rows_of(1)[3], 0, 5] = math.nan
    v[case.rows_of(2)[3], 0, 5] = math.nan
    out, lse = decode.decode_attention(case.q, case.kv, case.table, case.used, with_lse=True)
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    assert bool(out[1].isnan().all()) and bool(lse[1].isnan().all())
    nans = out[2].isnan()
    assert bool(nans[:, 5].all()) and int(nans.sum()) == 2
    case.check(out, lse, rows=[3])
    for which in range(4):
        c = Case(dev, 2, 1, 64, [1, 20, 20], quant=True, seed=2)
        if which < 2:
            c.kv[2 + which][c.rows_of(0)[0], 0] = 255
            c.kv[2 + which][c.rows_of(1)[3], 0] = 255
        else:
            c.kv[which - 2].view(torch.uint8)[c.rows_of(0)[0], 0] = 0xFF
            c.kv[which - 2].view(torch.uint8)[c.rows_of(1)[3], 0] = 0x7F
        out, lse = decode.decode_attention(c.q, c.kv, c.table, c.used, with_lse=True)
        assert bool(out[:2].isnan().all())
        c.check(out, lse, rows=[2])


def test_decode_attention_strides_scale_and_out(dev):
    """q as a slice of a projection, a table that is a view, an output of the
    caller's, another softmax scale."""
    case = Case(dev, 8, 2, 128, [40, 300, 77], seed=3)
    qkv = torch.zeros(3, 12 * 128, dtype=torch.bfloat16, device=dev)
    qkv[:, :8 * 128] = case.q.view(3, -1)
    wide = torch.full((3, case.table.shape[1] + 5), 10 ** 6, dtype=torch.int32, device=dev)
    wide[:, :case.table.shape[1]] = case.table
    out = torch.full((3, 16, 128), 5.0, dtype=torch.bfloat16, device=dev)
    got = decode.decode_attention(qkv[:, :8 * 128].view(3, 8, 128), case.kv,
                                  wide[:, :case.table.shape[1]], case.used, softmax_scale=0.03,
                                  out=out[:, 4:12])
    assert got.data_ptr() == out[:, 4:12].data_ptr() and status() == 0
    case.check(out[:, 4:12], scale=0.03)
    assert bool((out[:, :4] == 5).all()) and bool((out[:, 12:] == 5).all())


@pytest.mark.parametrize("ue8m0", [False, True])
@pytest.mark.parametrize("quant", [False, True])
def test_decode_attention_quantised_output(dev, quant, ue8m0):
    """The fp8 output is the bf16 output, quantised per head by the engine's
    rule."""
    case = Case(dev, 12, 2, 128, [40, 0, 5000, 77], quant=quant, seed=6)
    rows, ld = 4, 6
    q8 = QuantRows(torch.zeros(rows, 12 * 128, dtype=torch.float8_e4m3fn, device=dev),
                   torch.zeros(12, ld, device=dev), ld)
    out = torch.empty(rows, 12, 128, dtype=torch.bfloat16, device=dev)
    got = decode.decode_attention(case.q, case.kv, case.table, case.used, out=out,
                                  quantised=(q8, ue8m0))
    assert got is out and status() == 0
    alone = decode.decode_attention(case.q, case.kv, case.table, case.used)
    assert torch.equal(alone, out)
    x = out.float().cpu().numpy()
    amax = np.maximum(np.abs(x).max(-1), np.float32(1e-10))
    scale = (amax / np.float32(448)).astype(np.float32)
    if ue8m0:
        m, e = np.frexp(scale)
        scale = np.ldexp(np.float32(1), np.where(m == 0.5, e - 1, e)).astype(np.float32)
    assert np.array_equal(q8.scale[:, :rows].cpu().numpy().T, scale)
    codes = torch.from_numpy((x / scale[..., None]).clip(-448, 448)).to(torch.float8_e4m3fn)
    assert torch.equal(q8.q.view(torch.uint8).cpu().view(rows, 12, 128), codes.view(torch.uint8))


def test_decode_attention_bad_pages_and_lengths(dev):
    """A page out of range leaves its keys out, a length past the table ends at
    it, a negative one is none; each is flagged."""
    case = Case(dev, 4, 2, 128, [48, 32, 16], seed=7)
    table = case.table.clone()
    table[0, 1] = 10 ** 9
    used = case.used.clone()
    used[1] = 10 ** 8
    used[2] = -4
    out = decode.decode_attention(case.q, case.kv, table, used)
    assert status() == BAD_INDEX
    assert bool((out[2] == 0).all())
    short = Case.__new__(Case)
    short.__dict__ = dict(case.__dict__)
    keep = torch.cat([case.rows_of(0)[:16], case.rows_of(0)[32:]])
    short.rows_of = lambda r: keep
    short.lengths = [32]
    short.check(out, rows=[0])


def test_decode_attention_on_another_stream_and_in_a_graph(dev):
    case = Case(dev, 8, 2, 128, [3000, 12, 700], seed=11)
    want = decode.decode_attention(case.q, case.kv, case.table, case.used)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = decode.decode_attention(case.q, case.kv, case.table, case.used)
    side.synchronize()
    assert torch.equal(want, other)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(case.q)
    with torch.cuda.graph(graph):
        decode.decode_attention(case.q, case.kv, case.table, case.used, out=out)
    for lengths in ([3000, 12, 700], [5, 0, 333]):
        case.lengths = lengths
        case.used.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        case.check(out)
    assert status() == 0


def test_no_rows(dev):
    """Zero rows and groups: empty results, nothing launched on them."""
    kv = (torch.zeros(32, 2, 128, dtype=torch.bfloat16, device=dev),) * 2
    q = torch.zeros(0, 8, 128, dtype=torch.bfloat16, device=dev)
    table = torch.zeros(0, 3, dtype=torch.int32, device=dev)
    out, lse = decode.decode_attention(q, kv, table, table[:, 0].contiguous(), with_lse=True)
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)
    got = decode.beam_select(torch.zeros(0, 50, device=dev), torch.zeros(0, 4, device=dev))
    assert [t.shape for t in got] == [(0, 4)] * 3
    pool = torch.zeros(1, 2, 32, 1, 64, dtype=torch.bfloat16, device=dev)
    parents = torch.zeros(0, 4, dtype=torch.int32, device=dev)
    table, rows = decode.beam_reorder((pool,), parents, parents[:, 0].contiguous(), table)
    assert table.shape == (0, 3) and rows.shape == (0,)
    assert status() == 0


def test_decode_attention_repeats_bit_for_bit(dev):
    case = Case(dev, 32, 8, 128, [9000, 100, 2500, 1], seed=12)
    first = decode.decode_attention(case.q, case.kv, case.table, case.used, with_lse=True)
    for _ in range(5):
        again = decode.decode_attention(case.q, case.kv, case.table, case.used, with_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("quant", [False, True])
def test_decode_attention_past_32_bit_offsets(dev, quant):
    """Pool rows whose byte offsets pass 2^32 (and element offsets 2^31)."""
    n_kv, d, page = 8, 128, 64
    n_pages = (2 ** 32 // (n_kv * d * (1 if quant else 2)) // page) + 40
    case = Case(dev, 8, 8, d, [130, 65], page=page, quant=quant, seed=13, spare=0)
    small = case.kv
    shift = n_pages - small[0].shape[0] // page
    def far(x):
        y = torch.empty(n_pages * page, *x.shape[1:], dtype=x.dtype, device=dev)
        y[shift * page:] = x
        return y
    big = [far(x.view(torch.uint8)).view(x.dtype) if quant else far(x) for x in small[:2]]
    if quant:
        big = decode.QuantLayer(*big, *(far(x) for x in small[2:]))
    out, lse = decode.decode_attention(case.q, big, case.table + shift, case.used,
                                       page_tokens=page, with_lse=True)
    assert status() == 0
    case.check(out, lse)


# ---- beams -----------------------------------------------------------------------


def select64(logits, scores, finished, pad, n_out):
    """(score, parent, token) by the definition, in 64 bits; lists per group,
    over all offers, best first."""
    x = logits.double().cpu().numpy()
    groups, beams = scores.shape
    result = []
    for gi in range(groups):
        offers = []
        for b in range(beams):
            s = float(scores[gi, b])
            if finished is not None and finished[gi, b]:
                offers += [(s if r == 0 else -math.inf, b, r, pad) for r in range(n_out)]
                continue
            row = x[gi * beams + b]
            broken = np.isnan(row).any() or (row == math.inf).any()
            row = np.where(np.isnan(row), -math.inf, row)
            order = np.argsort(-row, kind="stable")[:n_out]
            m = row.max()
            dead = broken or m == -math.inf
            lse = m + math.log(np.exp(row - m).sum()) if not dead else 0.0
            for r, tok in enumerate(order):
                val = -math.inf if dead or row[tok] == -math.inf else s + (row[tok] - lse)
                offers.append((val if not math.isnan(val) else -math.inf, b, r, int(tok)))
        offers.sort(key=lambda o: (-o[0], o[1], o[2]))
        result.append(offers)
    return result


def check_select(got, logits, scores, finished=None, pad=0):
    score, parent, token = (t.cpu() for t in got)
    n_out = score.shape[1]
    want = select64(logits, scores.cpu(), None if finished is None else finished.cpu(), pad,
                    n_out)
    for gi, offers in enumerate(want):
        place = {(o[1], o[3], o[2]): o[0] for o in offers}
        for r in range(n_out):
            exact = offers[r][0]
            s = float(score[gi, r])
            if exact == -math.inf:
                assert s == -math.inf
            else:
                tol = 2 ** -19 + 2 ** -22 * (abs(exact) + abs(s) + 32)
                assert abs(s - exact) <= tol, (gi, r, s, exact)
            near = [o for j, o in enumerate(offers) if j != r and j in (r - 1, r + 1)
                    and o[0] != -math.inf and o[1] != offers[r][1]
                    and abs(o[0] - exact) <= 2 ** -17 and o[0] != exact]
            if not near:
                assert (int(parent[gi, r]), int(token[gi, r])) == (offers[r][1], offers[r][3]), (
                    gi, r, offers[:n_out], parent[gi], token[gi])
        assert place


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups,beams,vocab,n_out", [
    (1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 33, 5), (3, 4, 4096, 4), (1, 4, 151936, 4),
    (5, 8, 1000, 16), (2, 32, 257, 32), (1, 2, 40, 32), (9, 2, 12345, 1), (40, 8, 20000, 8),
    (1, 1, 100003, 32)])
def test_beam_select(dev, groups, beams, vocab, n_out, dtype):
    g = torch.Generator(device=dev).manual_seed(groups + vocab)
    logits = (3 * torch.randn(groups * beams, vocab, generator=g, device=dev)).to(dtype)
    scores = -5 + torch.randn(groups, beams, generator=g, device=dev)
    got = decode.beam_select(logits, scores, n_out=n_out)
    check_select(got, logits, scores)


def test_beam_select_ties_masks_and_finished(dev):
    """Equal logits and equal beams go to the lowest token and beam; masked
    tokens, beams without an allowed token, broken and finished beams."""
    beams, vocab = 4, 5000
    logits = torch.full((6 * beams, vocab), -math.inf, device=dev)
    scores = torch.zeros(6, beams, device=dev)
    finished = torch.zeros(6, beams, dtype=torch.bool, device=dev)
    logits[0:4] = 1.0                                   # group 0: all equal
    logits[4:8, 17::500] = 2.0                          # group 1: ten tokens, equal beams
    logits[8, 3] = 1.0                                  # group 2: one token, dead beams
    logits[12:16] = torch.randn(beams, vocab, device=dev)
    logits[13, 4000] = math.nan                         # group 3: NaN and +inf beams
    logits[14, 1] = math.inf
    logits[16:20] = torch.randn(beams, vocab, device=dev)
    finished[4, 1] = finished[4, 3] = True              # group 4: finished beams
    scores[4] = torch.tensor([-30.0, -2.0, -30.0, -3.0])
    logits[17] = math.nan                               # not read
    finished[5] = True                                  # group 5: all finished
    scores[5] = torch.tensor([-1.0, -5.0, -3.0, -3.0])
    got = decode.beam_select(logits, scores, finished=finished, pad=99)
    check_select(got, logits, scores, finished, 99)
    score, parent, token = (t.tolist() for t in got)
    assert parent[0] == [0, 0, 0, 0] and token[0] == [0, 1, 2, 3]
    assert token[1] == [17, 517, 1017, 1517] and parent[1] == [0, 0, 0, 0]
    assert score[2][0] == 0.0 and score[2][1:] == [-math.inf] * 3
    assert set(parent[3]) <= {0, 3}
    assert (parent[4][:2], token[4][:2], score[4][:2]) == ([1, 3], [99, 99], [-2.0, -3.0])
    assert parent[5] == [0, 2, 3, 1] and token[5] == [99] * 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["ascending", "descending", "blocks", "constant"])
def test_beam_select_adverse_orders(dev, kind, dtype):
    vocab = 30011
    x = {"ascending": torch.arange(vocab) / 1000.0, "descending": -torch.arange(vocab) / 1000.0,
         "blocks": (torch.arange(vocab) // 64 % 7).float(),
         "constant": torch.full((vocab,), -3.5)}[kind]
    logits = x.to(dtype).to(dev).repeat(6, 1)
    scores = torch.tensor([[-1.0, -1.5, -1.25], [0.0, 0.0, 0.0]], device=dev)
    for n_out in (1, 3, 32):
        check_select(decode.beam_select(logits, scores, n_out=n_out), logits, scores)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups,beams,vocab,n_out", [(15, 8, 20000, 8), (4, 32, 17001, 32),
                                                      (64, 1, 40001, 5), (37, 4, 16385, 3)])
def test_beam_select_wide_blocks(dev, groups, beams, vocab, n_out, dtype):
    """Enough rows of a long vocabulary for the wide blocks: random logits, and
    for some rows the orders and masks that the list does not hold."""
    g = torch.Generator(device=dev).manual_seed(groups + vocab)
    logits = 3 * torch.randn(groups * beams, vocab, generator=g, device=dev)
    logits[1] = torch.arange(vocab, device=dev) / 1000.0
    logits[2] = -1.5
    logits[3] = -math.inf
    logits[4, 7::3000] = math.nan
    logits[5] = -math.inf
    logits[5, 11::4000] = 0.5
    logits[6] = torch.arange(vocab, device=dev) // 100 % 5
    logits = logits.to(dtype)
    scores = -5 + torch.randn(groups, beams, generator=g, device=dev)
    check_select(decode.beam_select(logits, scores, n_out=n_out), logits, scores)


@pytest.mark.parametrize("groups,beams,vocab,n_out", [
    (1, 2, 300, 2), (1, 1, 9000, 1), (300, 2, 45000, 2), (1, 1, 148 * 150000, 1),
    (60, 2, 300000, 1)])
def test_beam_select_short_lists(dev, groups, beams, vocab, n_out):
    """Lists that one warp ranks, within a run and at its end, call after call:
    the same choice each time."""
    g = torch.Generator(device=dev).manual_seed(groups + vocab)
    logits = 3 * torch.randn(groups * beams, vocab, generator=g, device=dev)
    scores = -5 + torch.randn(groups, beams, generator=g, device=dev)
    got = [decode.beam_select(logits, scores, n_out=n_out) for _ in range(50)]
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
    check_select(got[0], logits, scores)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_beam_select_strided_rows(dev, dtype):
    """Rows at a stride that leaves them at every alignment."""
    g = torch.Generator(device=dev).manual_seed(3)
    wide = (2 * torch.randn(8, 9001, generator=g, device=dev)).to(dtype)
    for start, vocab in ((0, 9000), (1, 8999), (3, 4001), (5, 77)):
        logits = wide[:, start:start + vocab]
        scores = torch.randn(2, 4, generator=g, device=dev)
        check_select(decode.beam_select(logits, scores), logits, scores)


def reorder_by_hand(held, parents, used, table, page):
    out, nxt = table.clone(), []
    groups, beams = parents.shape
    for gi in range(groups):
        base, par = gi * beams, parents[gi].tolist()
        idle = [b for b in range(beams) if b not in par]
        full, tail = divmod(int(used[gi]), page)
        for j, p in enumerate(par):
            donor = idle.pop(0) if p in par[:j] else p
            out[base + j, :full] = table[base + p, :full]
            out[base + j, full:] = table[base + donor, full:]
            if donor != p and tail:
                a, b = int(table[base + p, full]) * page, int(table[base + donor, full]) * page
                for old, new in held:
                    new[:, :, b:b + tail] = old[:, :, a:a + tail]
            nxt.append(int(out[base + j, full]) * page + tail if full < table.shape[1] else -1)
    return out, nxt


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("groups,beams,page,used", [
    (1, 1, 16, [5]), (3, 4, 16, [0, 33, 48]), (2, 8, 8, [7, 24]), (4, 32, 16, [1, 15, 16, 31]),
    (2, 5, 64, [64, 100])])
def test_beam_reorder(dev, groups, beams, page, used, quant):
    g = torch.Generator().manual_seed(beams + page)
    width = max(used) // page + 2
    rows = groups * beams
    # shared full pages, then each beam's own
    table = torch.zeros(rows, width, dtype=torch.int32)
    n_pages = rows * width + 2
    ids = torch.randperm(n_pages, generator=g).tolist()
    for gi in range(groups):
        full = used[gi] // page
        shared = [ids.pop() for _ in range(full)]
        for j in range(beams):
            table[gi * beams + j] = torch.tensor(shared + [ids.pop() for _ in range(width - full)])
    parents = torch.randint(0, beams, (groups, beams), generator=g, dtype=torch.int32)
    if quant:
        kv = decode.QuantKV(3, n_pages, page, 3, 64)
        kv.codes.view(torch.uint8).copy_(torch.randint(0, 127, kv.codes.shape, generator=g))
        kv.scales.copy_(torch.randint(0, 255, kv.scales.shape, generator=g))
        pools = kv.pools
        plain = [kv.codes.view(torch.uint8).cpu(), kv.scales.cpu()]
    else:
        pools = (torch.randn(3, 2, n_pages * page, 3, 64, generator=g).to(torch.bfloat16).to(dev),)
        plain = [pools[0].cpu()]
    held = [(p, p.clone()) for p in plain]
    want, nxt = reorder_by_hand(held, parents, used, table, page)
    got, next_row = decode.beam_reorder(pools, parents.to(dev),
                                        torch.tensor(used, dtype=torch.int32, device=dev),
                                        table.to(dev), page_tokens=page)
    assert status() == 0
    assert torch.equal(got.cpu(), want) and next_row.tolist() == nxt
    for (_, new), now in zip(held, pools):
        now = now.view(torch.uint8) if quant and now.dtype != torch.uint8 else now
        assert torch.equal(now.cpu(), new)


def test_beam_reorder_bad_parents_and_full_tables(dev):
    pools = (torch.zeros(1, 2, 64, 1, 64, dtype=torch.bfloat16, device=dev),)
    table = torch.tensor([[0, 1], [0, 2]], dtype=torch.int32, device=dev)
    used = torch.tensor([32], dtype=torch.int32, device=dev)
    got, nxt = decode.beam_reorder(pools, torch.tensor([[1, 1]], dtype=torch.int32, device=dev),
                                   used, table)
    assert status() == 0 and nxt.tolist() == [-1, -1]
    assert got.tolist() == [[0, 2], [0, 2]]
    decode.beam_reorder(pools, torch.tensor([[0, 2]], dtype=torch.int32, device=dev), used, table)
    assert status() == BAD_INDEX
    decode.beam_reorder(pools, torch.tensor([[0, 0]], dtype=torch.int32, device=dev),
                        torch.tensor([40], dtype=torch.int32, device=dev), table)
    assert status() == BAD_INDEX
    bad = torch.tensor([[0, 1], [0, 99]], dtype=torch.int32, device=dev)
    decode.beam_reorder(pools, torch.tensor([[0, 0]], dtype=torch.int32, device=dev),
                        torch.tensor([20], dtype=torch.int32, device=dev), bad)
    assert status() == BAD_INDEX
