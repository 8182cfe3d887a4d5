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


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _same_device(who, first, *tensors):
    for t in tensors:
        if t is not None and t.device != first.device:
            raise ValueError(f"{who}: tensors on different devices")
    if first.device.type != "cuda":
        raise ValueError(f"{who}: CUDA tensors are needed")


def _heads(who, name, x, n_kv=None, d=None):
    """x as bf16 rows of heads [rows, n, d], each row's heads contiguous."""
    _need(x.dim() == 3 and x.dtype == torch.bfloat16, f"{who}: {name} must be bf16 [rows, n, d]")
    _need(n_kv is None or (x.shape[1] == n_kv and x.shape[2] == d),
          f"{who}: {name}'s heads are not the cache's")
    _need(x.stride(2) == 1 and (x.shape[1] == 1 or x.stride(1) == x.shape[2]),
          f"{who}: the heads of a row of {name} must be contiguous")


def _row_stride(x):
    # a single row's stride may be anything; the library wants one that covers it
    return x.stride(0) if x.shape[0] > 1 else -(-x.shape[1] * x.shape[2] // 8) * 8


def _quant_layer(who, kv):
    rows, n_kv, d = kv.k.shape
    for c, s in ((kv.k, kv.k_scale), (kv.v, kv.v_scale)):
        _need(c.shape == (rows, n_kv, d) and s.shape == (rows, n_kv)
              and c.dtype == torch.float8_e4m3fn and s.dtype == torch.uint8
              and c.is_contiguous() and s.is_contiguous(),
              f"{who}: the cache needs contiguous e4m3 codes [rows, n_kv, d] and uint8 scales "
              f"[rows, n_kv]")
    return rows, n_kv, d


def _index(who, name, x, n=None):
    _need(x.dtype == torch.int64 and x.dim() == 1 and x.is_contiguous()
          and (n is None or x.shape[0] == n), f"{who}: {name} must be a contiguous int64 vector "
          "as long as the rows")


def kv_quant_write(k, v, kv: QuantLayer, dst, src=None):
    """Quantise K and V rows into an 8-bit cache as they are written.

    k, v: bf16 [rows, n_kv, d], the heads of a row contiguous, rows at any
    stride that is a multiple of 8 elements (slices of a qkv projection, or an
    arena's pools). dst: int64 [n] pool rows, all different, a negative one
    writing nothing; src: int64 [n] rows of k and v, or None for 0 .. n - 1.
    """
    who = "kv_quant_write"
    pool_rows, n_kv, d = _quant_layer(who, kv)
    _heads(who, "k", k, n_kv, d)
    _heads(who, "v", v, n_kv, d)
    _need(k.shape == v.shape, f"{who}: k and v differ in rows")
    _index(who, "dst", dst, k.shape[0] if src is None else src.shape[0])
    if src is not None:
        _index(who, "src", src)
    _same_device(who, k, v, dst, src, *kv)
    nat.call("qb_kv_quant_write", k.data_ptr(), v.data_ptr(), _row_stride(k), _row_stride(v),
             None if src is None else src.data_ptr(), dst.data_ptr(), dst.shape[0], k.shape[0],
             n_kv, d, kv.k.data_ptr(), kv.v.data_ptr(), kv.k_scale.data_ptr(),
             kv.v_scale.data_ptr(), pool_rows, _stream(k.device))


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
        _need(dst is None, f"{who}: dst needs out")
        k = torch.empty((n, n_kv, d), dtype=torch.bfloat16, device=kv.k.device)
        v = torch.empty_like(k)
    else:
        k, v = out
        _heads(who, "k", k, n_kv, d)
        _heads(who, "v", v, n_kv, d)
        _need(k.shape == v.shape, f"{who}: k and v differ in rows")
    if dst is not None:
        _index(who, "dst", dst, n)
    _same_device(who, kv.k, k, v, src, dst, *kv)
    nat.call("qb_kv_quant_read", kv.k.data_ptr(), kv.v.data_ptr(), kv.k_scale.data_ptr(),
             kv.v_scale.data_ptr(), pool_rows, src.data_ptr(),
             None if dst is None else dst.data_ptr(), n, n_kv, d, k.data_ptr(), v.data_ptr(),
             _row_stride(k), _row_stride(v), k.shape[0], _stream(k.device))
    return k, v


def _decode_args(who, q, kv, table, used, page_tokens):
    _heads(who, "q", q)
    if isinstance(kv, QuantLayer):
        pool_rows, n_kv, d = _quant_layer(who, kv)
        k, v, ks, vs = kv
    else:
        k, v = kv
        ks = vs = None
        _need(k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype == torch.bfloat16
              and k.is_contiguous() and v.is_contiguous(),
              f"{who}: bf16 pools must be contiguous [rows, n_kv, d]")
        pool_rows, n_kv, d = k.shape
    _need(q.shape[2] == d, f"{who}: q's head size is not the cache's")
    _need(pool_rows % page_tokens == 0, f"{who}: the pools are not whole pages")
    _need(table.dim() == 2 and table.dtype == torch.int32 and table.shape[0] == q.shape[0]
          and table.stride(1) == 1, f"{who}: table must be int32 [rows, pages]")
    _need(used.dim() == 1 and used.dtype == torch.int32 and used.shape[0] == q.shape[0]
          and used.is_contiguous(), f"{who}: used must be int32 [rows]")
    _same_device(who, q, k, v, ks, vs, table, used)
    return k, v, ks, vs, pool_rows, n_kv, d


def decode_attention(q, kv, table, used, *, page_tokens=16, softmax_scale=None, out=None,
                     with_lse=False, quantised=None):
    """Attention of one new token per row over its paged KV cache.

    q: bf16 [rows, n_q, d]; kv: an arena's (k, v) pools of one layer (bf16
    [pool rows, n_kv, d]) or a QuantLayer; table: int32 [rows, width] page ids;
    used: int32 [rows] keys of each row, the new token's included (0: zeros).
    softmax_scale: d ** -0.5 when None. Returns the bf16 output [rows, n_q, d]
    (out, when given), with with_lse a pair of it and the f32 log-sum-exp
    [rows, n_q]. quantised: an engine.QuantRows to fill with the output
    quantised per head (d = 128), in place of the bf16 output unless out is
    given too; the library's UE8M0 mode when it is a (QuantRows, True) pair.
    """
    who = "decode_attention"
    k, v, ks, vs, pool_rows, n_kv, d = _decode_args(who, q, kv, table, used, page_tokens)
    rows, n_q = q.shape[0], q.shape[1]
    ue8m0 = False
    if isinstance(quantised, tuple):
        quantised, ue8m0 = quantised
    if out is None and quantised is None:
        out = torch.empty((rows, n_q, d), dtype=torch.bfloat16, device=q.device)
    elif out is not None:
        _heads(who, "out", out)
        _need(out.shape == q.shape, f"{who}: out must have q's shape")
        _same_device(who, q, out)
    if quantised is not None:
        _need(quantised.q.shape == (rows, n_q * d) and quantised.q.is_contiguous()
              and quantised.scale.shape[0] == n_q and quantised.scale.is_contiguous(),
              f"{who}: quantised must hold [rows, n_q * d] codes and [n_q, ld] scales")
        _same_device(who, q, quantised.q, quantised.scale)
    lse = torch.empty((rows, n_q), dtype=torch.float32, device=q.device) if with_lse else None
    nat.call("qb_decode_attention", q.data_ptr(), _row_stride(q), rows, n_q, n_kv, d,
             k.data_ptr(), v.data_ptr(), None if ks is None else ks.data_ptr(),
             None if vs is None else vs.data_ptr(), pool_rows // page_tokens, page_tokens,
             table.data_ptr(), table.shape[1], table.stride(0) if rows > 1 else table.shape[1],
             used.data_ptr(), d ** -0.5 if softmax_scale is None else softmax_scale,
             None if out is None else out.data_ptr(), 0 if out is None else _row_stride(out),
             None if quantised is None else quantised.q.data_ptr(),
             None if quantised is None else quantised.scale.data_ptr(),
             0 if quantised is None else quantised.ld, int(ue8m0),
             None if lse is None else lse.data_ptr(), _stream(q.device))
    result = quantised if out is None else out
    return (result, lse) if with_lse else result


def beam_select(logits, scores, *, finished=None, pad=0, n_out=None):
    """Beam search's choice over beams and vocabulary.

    logits: f32 or bf16 [groups * beams, vocab] (rows at any stride); scores:
    f32 [groups, beams]; finished: bool or uint8 [groups, beams] or None (such a
    beam continues only as itself, by the token pad). n_out: continuations per
    group, the beams' number when None. Returns (scores f32, parents int32,
    tokens int64), each [groups, n_out], best first; a parent is a beam's place
    in its group.
    """
    who = "beam_select"
    _need(scores.dim() == 2 and scores.dtype == torch.float32 and scores.is_contiguous(),
          f"{who}: scores must be contiguous f32 [groups, beams]")
    groups, beams = scores.shape
    n_out = beams if n_out is None else n_out
    _need(logits.dim() == 2 and logits.shape[0] == groups * beams
          and logits.dtype in (torch.float32, torch.bfloat16) and logits.stride(1) == 1,
          f"{who}: logits must be f32 or bf16 [groups * beams, vocab]")
    if finished is not None:
        _need(finished.shape == scores.shape and finished.is_contiguous()
              and finished.dtype in (torch.bool, torch.uint8),
              f"{who}: finished must be contiguous bool or uint8 [groups, beams]")
    _same_device(who, logits, scores, finished)
    vocab = logits.shape[1]
    need = nat.ctypes.c_int64(0)
    nat.call("qb_beam_select_workspace", groups, beams, vocab, n_out, nat.ctypes.byref(need))
    dev = logits.device
    workspace = torch.empty(max(need.value, 16), dtype=torch.uint8, device=dev)
    out = (torch.empty((groups, n_out), dtype=torch.float32, device=dev),
           torch.empty((groups, n_out), dtype=torch.int32, device=dev),
           torch.empty((groups, n_out), dtype=torch.int64, device=dev))
    nat.call("qb_beam_select", logits.data_ptr(), int(logits.dtype == torch.bfloat16),
             logits.stride(0) if logits.shape[0] > 1 else vocab, groups, beams, vocab,
             scores.data_ptr(), None if finished is None else finished.data_ptr(), pad, n_out,
             workspace.data_ptr(), workspace.shape[0], out[0].data_ptr(), out[1].data_ptr(),
             out[2].data_ptr(), _stream(dev))
    return out


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
    _need(parents.dim() == 2 and parents.dtype == torch.int32 and parents.is_contiguous(),
          f"{who}: parents must be contiguous int32 [groups, beams]")
    groups, beams = parents.shape
    _need(used.shape == (groups,) and used.dtype == torch.int32 and used.is_contiguous(),
          f"{who}: used must be int32 [groups]")
    _need(table.dim() == 2 and table.dtype == torch.int32 and table.is_contiguous()
          and table.shape[0] == groups * beams,
          f"{who}: table must be contiguous int32 [groups * beams, pages]")
    _need(len(pools) in (1, 2), f"{who}: one pool, or codes and scales")
    rows = pools[0].shape[2]
    _need(rows % page_tokens == 0, f"{who}: the pools are not whole pages")
    row_bytes = [0, 0]
    for i, pool in enumerate(pools):
        _need(pool.dim() >= 4 and pool.shape[:3] == pools[0].shape[:3] and pool.is_contiguous(),
              f"{who}: pools must be contiguous [n_layers, 2, rows, ...]")
        row_bytes[i] = pool.stride(2) * pool.element_size()
    _same_device(who, pools[0], parents, used, table, *pools[1:])
    out = torch.empty_like(table)
    next_row = torch.empty(groups * beams, dtype=torch.int64, device=table.device)
    nat.call("qb_beam_reorder", parents.data_ptr(), used.data_ptr(), groups, beams,
             table.data_ptr(), table.shape[1], page_tokens, rows // page_tokens,
             pools[0].data_ptr(), pools[0].shape[0] * pools[0].shape[1], row_bytes[0],
             pools[1].data_ptr() if len(pools) > 1 else None, row_bytes[1], out.data_ptr(),
             next_row.data_ptr(), _stream(table.device))
    return out, next_row
