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
caching allocator unless they are passed in. Shapes and types are checked by
csrc/torch_ops.cpp, sizes, strides and alignment by the library: ValueError.
"""

import ctypes
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

    @classmethod
    def over(cls, arena):
        """An 8-bit cache whose codes lie in an arena's own memory: the arena's page
        p is the 8-bit pages 2p and 2p + 1, for whoever has reserved it. Only the
        scale bytes are allocated, 1 / d_head of the arena's bytes."""
        kv = cls.__new__(cls)
        kv.n_layers, kv.n_pages, kv.page_tokens = (arena.n_layers, 2 * arena.n_pages,
                                                   arena.page_tokens)
        kv.n_kv, kv.d_head = arena.n_kv, arena.d_head
        rows = kv.n_pages * kv.page_tokens
        kv.codes = arena.pools.view(torch.float8_e4m3fn).view(kv.n_layers, 2, rows, kv.n_kv,
                                                              kv.d_head)
        kv.scales = torch.empty((kv.n_layers, 2, rows, kv.n_kv), dtype=torch.uint8,
                                device=arena.pools.device)
        return kv

    def layer_kv(self, layer: int) -> QuantLayer:
        return QuantLayer(self.codes[layer, 0], self.codes[layer, 1], self.scales[layer, 0],
                          self.scales[layer, 1])

    @property
    def pools(self):
        """What beam_reorder moves: the codes and their scales."""
        return self.codes, self.scales


_ENTRIES = ("qb_kv_quant_write", "qb_kv_quant_read", "qb_decode_attention_workspace",
            "qb_decode_attention", "qb_beam_select_workspace", "qb_beam_select",
            "qb_beam_reorder")
_bound = None


def _ops():
    """The compiled calls, bound to the loaded library's entry points."""
    global _bound
    if _bound is None:
        lib = nat.load()
        try:
            from quail_b200 import _torch_ops
        except ImportError as e:
            raise ImportError("quail_b200/_torch_ops.so is missing or not of this torch: build "
                              "it with `python -m quail_b200.build`") from e
        _torch_ops.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value
                         for n in _ENTRIES})
        _bound = _torch_ops
    return _bound


def kv_quant_write(k, v, kv: QuantLayer, dst, src=None):
    """Quantise K and V rows into an 8-bit cache as they are written.

    k, v: bf16 [rows, n_kv, d], the heads of a row contiguous, rows at any
    stride that is a multiple of 8 elements (slices of a qkv projection, or an
    arena's pools). dst: int64 [n] pool rows, all different, a negative one
    writing nothing; src: int64 [n] rows of k and v, or None for 0 .. n - 1.
    """
    _ops().kv_quant_write(k, v, *kv, dst, src)
    nat.LAUNCHES["count"] += 1


def kv_quant_read(kv: QuantLayer, src, dst=None, out=None):
    """(k, v) bf16 of an 8-bit cache's rows src (int64 [n]), the values that the
    codes stand for. out: (k, v) to write into, row dst[i] (int64 [n]; negative:
    not written) or row i, for instance an arena's pools and the rows of its
    pages; fresh [n, n_kv, d] tensors otherwise."""
    k, v = (None, None) if out is None else out
    result = _ops().kv_quant_read(*kv, src, dst, k, v)
    nat.LAUNCHES["count"] += 1
    return result


def decode_workspace(device="cuda"):
    """A workspace for decode_attention calls that follow one another (one
    stream, one captured graph): its size does not depend on a call's, and each
    call leaves it as it found it."""
    return _ops().decode_workspace(torch.empty(0, device=device).device)


def beam_workspace(groups, beams, vocab, n_out=None, device="cuda"):
    """A workspace for beam_select calls of these sizes that follow one
    another."""
    return _ops().beam_workspace(groups, beams, vocab, beams if n_out is None else n_out,
                                 torch.empty(0, device=device).device)


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
    stream's own when None (in a captured graph a fresh one, zeroed by each
    replay).
    """
    k, v, k_scale, v_scale = kv if len(kv) == 4 else (*kv, None, None)
    codes = scale = None
    ld, ue8m0 = 0, False
    if quantised is not None:
        if isinstance(quantised, tuple):
            quantised, ue8m0 = quantised
        codes, scale, ld = quantised.q, quantised.scale, quantised.ld
    got, lse = _ops().decode_attention(
        q, k, v, k_scale, v_scale, table, used, page_tokens,
        q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale, out, with_lse, codes,
        scale, ld, ue8m0, workspace)
    nat.LAUNCHES["count"] += 1
    result = quantised if got is None else got
    return (result, lse) if with_lse else result


def beam_select(logits, scores, *, finished=None, pad=0, n_out=None, workspace=None):
    """Beam search's choice over beams and vocabulary.

    logits: f32 or bf16 [groups * beams, vocab] (rows at any stride); scores:
    f32 [groups, beams]; finished: bool or uint8 [groups, beams] or None (such a
    beam continues only as itself, by the token pad). n_out: continuations per
    group, the beams' number when None. Returns (scores f32, parents int32,
    tokens int64), each [groups, n_out], best first; a parent is a beam's place
    in its group. workspace: from beam_workspace, for calls that never overlap;
    the current stream's own when None (in a captured graph a fresh one, zeroed
    by each replay).
    """
    result = _ops().beam_select(logits, scores, finished, pad, n_out, workspace)
    nat.LAUNCHES["count"] += 1
    return result


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
    if len(pools) not in (1, 2):
        raise ValueError("beam_reorder: one pool, or codes and scales")
    result = _ops().beam_reorder(pools[0], pools[1] if len(pools) == 2 else None, parents, used,
                                 table, page_tokens)
    nat.LAUNCHES["count"] += 1
    return result
