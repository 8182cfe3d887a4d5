"""Refusals of the generation operators: bad arguments raise ValueError before
any launch (no GPU is touched, so these run on the CPU-only test host)."""

import ctypes

import pytest
import torch

from quail_b200 import _native as nat
from quail_b200 import decode

OK, OFF = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1008)


@pytest.fixture(scope="module", autouse=True)
def lib():
    if not nat.LIBRARY.exists():
        from quail_b200 import build
        build.build()
    return nat.load()


def refused(match, name, *args):
    with pytest.raises(ValueError, match=match):
        nat.call(name, *args)


WRITE = dict(k=OK, v=OK, k_ld=256, v_ld=256, src=None, dst=OK, n=4, src_rows=4, n_kv=2, d=128,
             kc=OK, vc=OK, ks=OK, vs=OK, pool=64, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(d=96), "head_dim"), (dict(n=-1), "counts"), (dict(n_kv=0), "counts"),
    (dict(n_kv=2000), "counts"), (dict(k_ld=248), "cover"), (dict(v_ld=260), "multiples of 8"),
    (dict(k=OFF), "aligned"), (dict(vc=OFF), "aligned"), (dict(ks=None), "NULL"),
    (dict(dst=None), "dst"), (dict(src_rows=3), "fewer source rows")])
def test_kv_quant_write_refuses(change, match):
    refused(match, "qb_kv_quant_write", *dict(WRITE, **change).values())


READ = dict(kc=OK, vc=OK, ks=OK, vs=OK, pool=64, src=OK, dst=None, n=4, n_kv=2, d=128, k=OK,
            v=OK, k_ld=256, v_ld=256, rows=4, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(d=32), "head_dim"), (dict(n=1 << 31), "counts"), (dict(v_ld=255), "cover"),
    (dict(kc=OFF), "aligned"), (dict(src=None), "src"), (dict(rows=3), "fewer output rows")])
def test_kv_quant_read_refuses(change, match):
    refused(match, "qb_kv_quant_read", *dict(READ, **change).values())


ATTN = dict(q=OK, q_ld=1024, rows=4, n_q=8, n_kv=2, d=128, k=OK, v=OK, ks=None, vs=None,
            n_pages=8, page=16, table=OK, width=4, table_ld=4, used=OK, scale=0.1)
ATTN_OUT = dict(ws=OK, ws_bytes=1 << 30, out=OK, out_ld=1024, q_out=None, scale_out=None, scale_ld=0, ue8m0=0, lse=None,
                stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(d=80), "head_dim"), (dict(n_q=7), "multiple of n_kv"), (dict(n_kv=0), "multiple"),
    (dict(rows=70000), "rows"), (dict(page=12), "power of two"), (dict(page=4), "power of two"),
    (dict(q_ld=1020), "q_ld"), (dict(q=OFF), "alignment"), (dict(out=None), "no output"),
    (dict(out_ld=1000), "out_ld"), (dict(table=None), "NULL"), (dict(ks=OK), "together"),
    (dict(k=OFF), "aligned"), (dict(width=0), "width"), (dict(table_ld=3), "width"),
    (dict(n_pages=0), "width"), (dict(width=1 << 40), "width"),
    (dict(ws=None), "workspace"), (dict(ws=OFF), "workspace"),
    (dict(q_out=OK), "fp8 output"), (dict(q_out=OK, scale_out=OK, scale_ld=3), "fp8 output")])
def test_decode_attention_refuses(change, match):
    args = dict(ATTN, **ATTN_OUT)
    args.update(change)
    refused(match, "qb_decode_attention", *args.values())


SELECT = dict(logits=OK, bf16=0, ld=100, groups=2, beams=4, vocab=100, scores=OK, finished=None,
              pad=0, n_out=4, ws=OK, ws_bytes=1 << 20, so=OK, po=OK, to=OK, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(beams=33), "beams"), (dict(n_out=0), "outputs"), (dict(n_out=33), "outputs"),
    (dict(vocab=3, ld=3), "vocab"), (dict(vocab=2**31 - 1, ld=2**31), "vocab"),
    (dict(ld=99), "logits_ld"), (dict(logits=None), "NULL"),
    (dict(ws=None), "workspace"), (dict(ws_bytes=8), "workspace")])
def test_beam_select_refuses(change, match):
    refused(match, "qb_beam_select", *dict(SELECT, **change).values())


REORDER = dict(parents=OK, used=OK, groups=2, beams=4, table=OK, width=4, page=16, n_pages=64,
               pool=OK, slabs=4, row_bytes=256, pool2=None, row_bytes2=0,
               out=ctypes.c_void_p(0x2000), next_row=None, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(beams=0), "beams"), (dict(groups=20000), "rows"), (dict(page=0), "page"),
    (dict(groups=1 << 62), "rows"), (dict(width=(1 << 62) + 1), "table"),
    (dict(row_bytes=24), "multiples of 16"), (dict(pool=OFF), "aligned"),
    (dict(pool2=OK), "row_bytes2"), (dict(out=None), "NULL"), (dict(out=OK), "table_in")])
def test_beam_reorder_refuses(change, match):
    refused(match, "qb_beam_reorder", *dict(REORDER, **change).values())


def test_python_refusals():
    """Shapes and types, before the tensors' device is looked at; CPU tensors
    last."""
    bf = dict(dtype=torch.bfloat16)
    kv = decode.QuantKV(1, 2, 16, 2, 128, device="cpu").layer_kv(0)
    k, dst = torch.zeros(3, 2, 128, **bf), torch.arange(3)
    for match, args in (
            ("bf16", (k.float(), k, kv, dst)), ("heads", (k[:, :1], k[:, :1], kv, dst)),
            ("contiguous", (k.transpose(0, 1).contiguous().transpose(0, 1), k, kv, dst)),
            ("differ", (k, k[:2], kv, dst)), ("dst", (k, k, kv, dst.int())),
            ("dst", (k, k, kv, dst[:2])), ("e4m3", (k, k, kv._replace(k=k), dst)),
            ("CUDA", (k, k, kv, dst))):
        with pytest.raises(ValueError, match=match):
            decode.kv_quant_write(*args)
    with pytest.raises(ValueError, match="dst needs out"):
        decode.kv_quant_read(kv, dst, dst=dst)
    for out in ((k, None), (None, k)):
        with pytest.raises(ValueError, match="pair"):
            decode.kv_quant_read(kv, dst, out=out)
    q, table = torch.zeros(3, 4, 128, **bf), torch.zeros(3, 2, dtype=torch.int32)
    used, pools = torch.zeros(3, dtype=torch.int32), (torch.zeros(32, 2, 128, **bf),) * 2
    for match, args in (
            ("q must", (q.float(), pools, table, used)),
            ("head size", (torch.zeros(3, 4, 64, **bf), pools, table, used)),
            ("table", (q, pools, table[:2], used)), ("table", (q, pools, table.long(), used)),
            ("used", (q, pools, table, used[:1])),
            ("bf16 pools", (q, (pools[0], pools[1].float()), table, used)),
            ("CUDA", (q, pools, table, used)), ("CUDA", (q, kv, table, used))):
        with pytest.raises(ValueError, match=match):
            decode.decode_attention(*args)
    with pytest.raises(ValueError, match="whole pages"):
        decode.decode_attention(q, pools, table, used, page_tokens=64)
    logits, scores = torch.zeros(4, 10), torch.zeros(2, 2)
    for match, args, kw in (
            ("scores", (logits, scores.double()), {}), ("logits", (logits[:3], scores), {}),
            ("logits", (logits.half(), scores), {}),
            ("finished", (logits, scores), dict(finished=torch.zeros(2, 3, dtype=torch.bool))),
            ("CUDA", (logits, scores), {})):
        with pytest.raises(ValueError, match=match):
            decode.beam_select(*args, **kw)
    parents = torch.zeros(2, 2, dtype=torch.int32)
    pool, table, used = torch.zeros(1, 2, 32, 2, 64, **bf), torch.zeros(4, 2, dtype=torch.int32), \
        torch.zeros(2, dtype=torch.int32)
    for match, args, kw in (
            ("parents", ((pool,), parents.long(), used, table), {}),
            ("used", ((pool,), parents, used[:1], table), {}),
            ("table", ((pool,), parents, used, table[:3]), {}),
            ("one pool", ((), parents, used, table), {}),
            ("whole pages", ((pool,), parents, used, table), dict(page_tokens=64)),
            ("pools", ((torch.zeros(1, 2, 64, 2, 64, **bf)[:, :, ::2],), parents, used, table), {}),
            ("CUDA", ((pool,), parents, used, table), {})):
        with pytest.raises(ValueError, match=match):
            decode.beam_reorder(*args, **kw)
