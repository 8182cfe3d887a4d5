"""The operators of generation: continuing rows whose KV is already paged.

- ``QuantKV`` / ``kv_quant_write`` / ``kv_quant_read``: an 8-bit paged KV
  cache (e4m3 codes, one power-of-two scale per row and head), quantised as
  it is written and read back as bf16;
- ``decode_attention``: attention of one new token per row over its paged
  cache, bf16 (an arena's layer) or 8-bit;
- ``beam_select`` / ``beam_reorder``: beam search's choice over beams and
  vocabulary, and the page tables and started pages following it.

Every function launches libquailb200 kernels on the current CUDA stream of
its inputs' device and returns without waiting; outputs come from torch's
caching allocator unless they are passed in. Shapes and types are checked
here (ValueError); sizes, strides and alignment by the library.
"""

import ctypes
import functools
from typing import NamedTuple

import torch

from quail_b200 import _native as nat


class QuantLayer(NamedTuple):
    """One layer of an 8-bit cache: e4m3 codes [rows, n_kv, d] and exponent
    bytes [rows, n_kv] (scale 2^(byte - 127)) of K and V."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


class QuantKV:
    """The pools of an 8-bit paged KV cache, page for page like KVArena's:
    page p holds pool rows p * page_tokens .. (p + 1) * page_tokens.

    HBM layout: codes (n_layers, 2, rows, n_kv, d_head) e4m3, scales
    (n_layers, 2, rows, n_kv) uint8.
    """

    def __init__(self, n_layers, n_pages, page_tokens, n_kv, d_head, device="cuda"):
        rows = n_pages * page_tokens
        self.n_layers, self.n_pages, self.page_tokens = n_layers, n_pages, page_tokens
        self.n_kv, self.d_head = n_kv, d_head
        self.codes = torch.empty((n_layers, 2, rows, n_kv, d_head), dtype=torch.float8_e4m3fn,
                                 device=device)
        self.scales = torch.empty((n_layers, 2, rows, n_kv), dtype=torch.uint8, device=device)

    def layer_kv(self, layer: int) -> QuantLayer:
        return QuantLayer(self.codes[layer, 0], self.codes[layer, 1], self.scales[layer, 0],
                          self.scales[layer, 1])

    @property
    def pools(self):
        """What beam_reorder moves: the codes and their scales."""
        return self.codes, self.scales


_bf16, _f32, _i32, _i64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _launch(name, device, args):
    """One library call (the arguments before the stream) on the current stream
    of CUDA device `device`. nat.call without its look-ups: a call's host time is
    what a small one costs."""
    if device != _current_device():
        with torch.cuda.device(device):
            return _launch(name, device, args)
    status = getattr(nat.load(), name)(*args, _raw_stream(device))
    if status:
        nat.check(status, name)
    nat.LAUNCHES["count"] += 1


def _device(who, first, *others):
    """The index of the one CUDA device that holds the tensors (None skipped)."""
    device = first.get_device()
    if device < 0:
        raise ValueError(f"{who}: CUDA tensors are needed")
    for t in others:
        if t is not None and t.get_device() != device:
            raise ValueError(f"{who}: tensors on different devices")
    return device


def _heads(who, name, x):
    """(rows, heads, d, row stride) of bf16 rows of heads [rows, n, d], each
    row's heads contiguous."""
    shape = x.shape
    if len(shape) != 3 or x.dtype != _bf16:
        raise ValueError(f"{who}: {name} must be bf16 [rows, n, d]")
    rows, n, d = shape
    ld, head, one = x.stride()
    if one != 1 or (head != d and n > 1):
        raise ValueError(f"{who}: the heads of a row of {name} must be contiguous")
    # a single row's stride may be anything; the library wants one that covers it
    return rows, n, d, ld if rows > 1 else -(-n * d // 8) * 8


def _quant_layer(who, kv):
    k, v, ks, vs = kv
    shape = k.shape
    if not (len(shape) == 3 and v.shape == shape and ks.shape == vs.shape == shape[:2]
            and k.dtype == v.dtype == torch.float8_e4m3fn
            and ks.dtype == vs.dtype == torch.uint8
            and k.is_contiguous() and v.is_contiguous()
            and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError(f"{who}: the cache needs contiguous e4m3 codes [rows, n_kv, d] and "
                         "uint8 scales [rows, n_kv]")
    return shape


def _index(who, name, x, n=None):
    shape = x.shape
    if x.dtype != _i64 or len(shape) != 1 or not x.is_contiguous() or (
            n is not None and shape[0] != n):
        raise ValueError(f"{who}: {name} must be a contiguous int64 vector as long as the rows")


def _rows_of(who, k, v, n_kv, d):
    """(rows, k's and v's row strides) of bf16 K and V of the cache's heads."""
    rows, n, width, k_ld = _heads(who, "k", k)
    v_rows, n_v, v_width, v_ld = _heads(who, "v", v)
    if n != n_kv or n_v != n_kv or width != d or v_width != d:
        raise ValueError(f"{who}: the heads of k and v are not the cache's")
    if rows != v_rows:
        raise ValueError(f"{who}: k and v differ in rows")
    return rows, k_ld, v_ld


def kv_quant_write(k, v, kv: QuantLayer, dst, src=None):
    """Quantise K and V rows into an 8-bit cache as they are written.

    k, v: bf16 [rows, n_kv, d], the heads of a row contiguous, rows at any
    stride that is a multiple of 8 elements (slices of a qkv projection, or an
    arena's pools). dst: int64 [n] pool rows, all different, a negative one
    writing nothing; src: int64 [n] rows of k and v, or None for 0 .. n - 1.
    """
    who = "kv_quant_write"
    pool_rows, n_kv, d = _quant_layer(who, kv)
    rows, k_ld, v_ld = _rows_of(who, k, v, n_kv, d)
    if src is not None:
        _index(who, "src", src)
    n = rows if src is None else src.shape[0]
    _index(who, "dst", dst, n)
    device = _device(who, k, v, dst, src, *kv)
    _launch("qb_kv_quant_write", device, (
        k.data_ptr(), v.data_ptr(), k_ld, v_ld, None if src is None else src.data_ptr(),
        dst.data_ptr(), n, rows, n_kv, d, kv.k.data_ptr(), kv.v.data_ptr(),
        kv.k_scale.data_ptr(), kv.v_scale.data_ptr(), pool_rows))


def kv_quant_read(kv: QuantLayer, src, dst=None, out=None):
    """(k, v) bf16 of an 8-bit cache's rows src (int64 [n]), the values that the
    codes stand for. out: (k, v) to write into, row dst[i] (int64 [n]; negative:
    not written) or row i, for instance an arena's pools and the rows of its
    pages; fresh [n, n_kv, d] tensors otherwise."""
    who = "kv_quant_read"
    pool_rows, n_kv, d = _quant_layer(who, kv)
    _index(who, "src", src)
    n = src.shape[0]
    if out is None:
        if dst is not None:
            raise ValueError(f"{who}: dst needs out")
        k, v = kv.k.new_empty((2, n, n_kv, d), dtype=torch.bfloat16).unbind(0)
        rows, k_ld, v_ld = n, n_kv * d, n_kv * d
    else:
        k, v = out
        rows, k_ld, v_ld = _rows_of(who, k, v, n_kv, d)
        if dst is not None:
            _index(who, "dst", dst, n)
    device = _device(who, k, v, src, dst, *kv)
    _launch("qb_kv_quant_read", device, (
        kv.k.data_ptr(), kv.v.data_ptr(), kv.k_scale.data_ptr(), kv.v_scale.data_ptr(),
        pool_rows, src.data_ptr(), None if dst is None else dst.data_ptr(), n, n_kv, d,
        k.data_ptr(), v.data_ptr(), k_ld, v_ld, rows))
    return k, v


_workspaces = {}   # (use, device, stream) -> a workspace


def _stream_workspace(use, device, need):
    """The current stream's own zeroed workspace of `need` bytes or more, kept
    (each call leaves its counters zero). A graph that is being captured must
    not share it (the graph may be replayed beside the stream), so there a call
    gets a fresh one, whose zeroing the graph repeats: pass workspace= to spare
    that."""
    key = use, device, torch._C._cuda_getCurrentRawStream(device)
    held = _workspaces.get(key)
    if held is not None and held.shape[0] >= need and (
            not torch.cuda.is_current_stream_capturing()):
        return held
    held = torch.zeros(need, dtype=torch.uint8, device=torch.device("cuda", device))
    if not torch.cuda.is_current_stream_capturing():
        _workspaces[key] = held
    return held


_attention_bytes = {}   # device -> bytes


def _decode_bytes(device):
    need = _attention_bytes.get(device)
    if need is None:
        out = ctypes.c_int64(0)
        with torch.cuda.device(device):
            nat.call("qb_decode_attention_workspace", ctypes.byref(out))
        need = _attention_bytes[device] = out.value
    return need


def decode_workspace(device="cuda"):
    """A workspace for decode_attention calls that follow one another (one
    stream, one captured graph): its size does not depend on a call's, and each
    call leaves it as it found it."""
    index = torch.empty(0, device=device).get_device()
    return torch.zeros(_decode_bytes(index), dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=256)
def _select_bytes(groups, beams, vocab, n_out):
    need = ctypes.c_int64(0)
    nat.call("qb_beam_select_workspace", groups, beams, vocab, n_out, ctypes.byref(need))
    return need.value


def beam_workspace(groups, beams, vocab, n_out=None, device="cuda"):
    """A workspace for beam_select calls of these sizes that follow one
    another."""
    need = _select_bytes(groups, beams, vocab, beams if n_out is None else n_out)
    return torch.zeros(need, dtype=torch.uint8, device=device)


def decode_attention(q, kv, table, used, *, page_tokens=16, softmax_scale=None, out=None,
                     with_lse=False, quantised=None, workspace=None):
    """Attention of one new token per row over its paged KV cache.

    q: bf16 [rows, n_q, d]; kv: an arena's (k, v) pools of one layer (bf16
    [pool rows, n_kv, d]) or a QuantLayer; table: int32 [rows, width] page ids;
    used: int32 [rows] keys of each row, the new token's included (0: zeros).
    softmax_scale: d ** -0.5 when None. Returns the bf16 output [rows, n_q, d]
    (out, when given), with with_lse a pair of it and the f32 log-sum-exp
    [rows, n_q]. quantised: an engine.QuantRows to fill with the output
    quantised per head (d = 128), in place of the bf16 output unless out is
    given too; the library's UE8M0 mode when it is a (QuantRows, True) pair.
    workspace: from decode_workspace, for calls that never overlap; the current
    stream's own when None.
    """
    who = "decode_attention"
    rows, n_q, d, q_ld = _heads(who, "q", q)
    if len(kv) == 4:
        pool_rows, n_kv, width = _quant_layer(who, kv)
        k, v, ks, vs = kv
    else:
        k, v = kv
        ks = vs = None
        shape = k.shape
        if not (len(shape) == 3 and v.shape == shape and k.dtype == v.dtype == _bf16
                and k.is_contiguous() and v.is_contiguous()):
            raise ValueError(f"{who}: bf16 pools must be contiguous [rows, n_kv, d]")
        pool_rows, n_kv, width = shape
    if width != d:
        raise ValueError(f"{who}: q's head size is not the cache's")
    if page_tokens <= 0 or pool_rows % page_tokens:
        raise ValueError(f"{who}: the pools are not whole pages")
    shape = table.shape
    if len(shape) != 2 or shape[0] != rows or table.dtype != _i32 or table.stride(1) != 1:
        raise ValueError(f"{who}: table must be int32 [rows, pages]")
    table_width = shape[1]
    if used.shape != (rows,) or used.dtype != _i32 or not used.is_contiguous():
        raise ValueError(f"{who}: used must be int32 [rows]")
    q8 = q8_scale = None
    q8_ld, ue8m0, out_ld = 0, False, 0
    if quantised is not None:
        if isinstance(quantised, tuple):
            quantised, ue8m0 = quantised
        q8, q8_scale, q8_ld = quantised.q, quantised.scale, quantised.ld
        if not (q8.shape == (rows, n_q * d) and q8.is_contiguous()
                and q8_scale.shape[0] == n_q and q8_scale.is_contiguous()):
            raise ValueError(f"{who}: quantised must hold [rows, n_q * d] codes and [n_q, ld] "
                             "scales")
    if out is not None:
        if out.shape != q.shape:
            raise ValueError(f"{who}: out must have q's shape")
        out_ld = _heads(who, "out", out)[3]
    device = _device(who, q, k, v, ks, vs, table, used, out, q8, q8_scale, workspace)
    if out is None and q8 is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        out_ld = n_q * d
    lse = q.new_empty((rows, n_q), dtype=_f32) if with_lse else None
    if workspace is None:
        workspace = _stream_workspace("attention", device, _decode_bytes(device))
    _launch("qb_decode_attention", device, (
        q.data_ptr(), q_ld, rows, n_q, n_kv, d, k.data_ptr(), v.data_ptr(),
        None if ks is None else ks.data_ptr(), None if vs is None else vs.data_ptr(),
        pool_rows // page_tokens, page_tokens, table.data_ptr(), table_width,
        table.stride(0) if rows > 1 else table_width, used.data_ptr(),
        d ** -0.5 if softmax_scale is None else softmax_scale, workspace.data_ptr(),
        workspace.shape[0], None if out is None else out.data_ptr(), out_ld,
        None if q8 is None else q8.data_ptr(), None if q8 is None else q8_scale.data_ptr(),
        q8_ld, ue8m0, None if lse is None else lse.data_ptr()))
    result = quantised if out is None else out
    return (result, lse) if with_lse else result


def beam_select(logits, scores, *, finished=None, pad=0, n_out=None, workspace=None):
    """Beam search's choice over beams and vocabulary.

    logits: f32 or bf16 [groups * beams, vocab] (rows at any stride); scores:
    f32 [groups, beams]; finished: bool or uint8 [groups, beams] or None (such a
    beam continues only as itself, by the token pad). n_out: continuations per
    group, the beams' number when None. Returns (scores f32, parents int32,
    tokens int64), each [groups, n_out], best first; a parent is a beam's place
    in its group. workspace: from beam_workspace, for calls that never overlap;
    the current stream's own when None.
    """
    who = "beam_select"
    shape = scores.shape
    if len(shape) != 2 or scores.dtype != _f32 or not scores.is_contiguous():
        raise ValueError(f"{who}: scores must be contiguous f32 [groups, beams]")
    groups, beams = shape
    n_out = beams if n_out is None else n_out
    dtype, shape = logits.dtype, logits.shape
    if len(shape) != 2 or shape[0] != groups * beams or logits.stride(1) != 1 or (
            dtype != _f32 and dtype != _bf16):
        raise ValueError(f"{who}: logits must be f32 or bf16 [groups * beams, vocab]")
    if finished is not None and not (
            finished.shape == scores.shape and finished.is_contiguous()
            and finished.dtype in (torch.bool, torch.uint8)):
        raise ValueError(f"{who}: finished must be contiguous bool or uint8 [groups, beams]")
    device = _device(who, logits, scores, finished, workspace)
    vocab = shape[1]
    if workspace is None:
        workspace = _stream_workspace("select", device,
                                      _select_bytes(groups, beams, vocab, n_out))
    score = torch.empty_like(scores) if n_out == beams else scores.new_empty((groups, n_out))
    parent = scores.new_empty((groups, n_out), dtype=_i32)
    token = scores.new_empty((groups, n_out), dtype=_i64)
    _launch("qb_beam_select", device, (
        logits.data_ptr(), dtype == _bf16, logits.stride(0) if groups * beams > 1 else vocab,
        groups, beams, vocab, scores.data_ptr(),
        None if finished is None else finished.data_ptr(), pad, n_out, workspace.data_ptr(),
        workspace.shape[0], score.data_ptr(), parent.data_ptr(), token.data_ptr()))
    return score, parent, token


def beam_reorder(pools, parents, used, table, *, page_tokens=16):
    """The beams' paged KV after a choice: page tables that follow the parents,
    and the started pages' tokens copied where siblings part.

    pools: the KV pools of all layers, in place: (arena.pools,) or
    QuantKV.pools, each [n_layers, 2, pool rows, ...] contiguous; parents: int32
    [groups, beams]; used: int32 [groups] tokens that every beam of the group
    holds; table: int32 [groups * beams, width], the entries before used //
    page_tokens full pages (beams may share them), the rest a beam's own.
    Returns (table, next_row): a new table, and int64 [groups * beams] the pool
    row of each beam's next token (-1 when its table is full).
    """
    who = "beam_reorder"
    shape = parents.shape
    if len(shape) != 2 or parents.dtype != _i32 or not parents.is_contiguous():
        raise ValueError(f"{who}: parents must be contiguous int32 [groups, beams]")
    groups, beams = shape
    if used.shape != (groups,) or used.dtype != _i32 or not used.is_contiguous():
        raise ValueError(f"{who}: used must be int32 [groups]")
    shape = table.shape
    if len(shape) != 2 or shape[0] != groups * beams or table.dtype != _i32 or (
            not table.is_contiguous()):
        raise ValueError(f"{who}: table must be contiguous int32 [groups * beams, pages]")
    width = shape[1]
    if len(pools) not in (1, 2):
        raise ValueError(f"{who}: one pool, or codes and scales")
    pool = pools[0]
    second = pools[1] if len(pools) == 2 else None
    shape = pool.shape
    if len(shape) < 4 or not pool.is_contiguous() or second is not None and not (
            second.dim() >= 4 and second.shape[:3] == shape[:3] and second.is_contiguous()):
        raise ValueError(f"{who}: pools must be contiguous [n_layers, 2, rows, ...]")
    rows = shape[2]
    if page_tokens <= 0 or rows % page_tokens:
        raise ValueError(f"{who}: the pools are not whole pages")
    device = _device(who, pool, second, parents, used, table)
    out = torch.empty_like(table)
    next_row = table.new_empty(groups * beams, dtype=_i64)
    _launch("qb_beam_reorder", device, (
        parents.data_ptr(), used.data_ptr(), groups, beams, table.data_ptr(), width, page_tokens,
        rows // page_tokens, pool.data_ptr(), shape[0] * shape[1],
        pool.stride(2) * pool.element_size(), None if second is None else second.data_ptr(),
        0 if second is None else second.stride(2) * second.element_size(), out.data_ptr(),
        next_row.data_ptr()))
    return out, next_row
