"""The generation operators' measured cases: decode attention over the paged
KV cache, the 8-bit KV cache's write and read back, and a beam-search step
(selection over beams and vocabulary, then the reordering of the beams' pages).

Each case runs either in its plain form (elementary torch operations in 32
bits) or, where ``own`` is true, through quail_b200.decode, the calls a user
makes. Shapes are this repository's model configurations (32 or 64 query
heads over 8 KV heads of 128, the tiny test model's 4 over 2, configuration
0's heads of 64, a vocabulary of 151,936, 16-token pages) with the lengths of
its filter and long-document workloads, and odd neighbours of them.
"""

import math

import numpy as np
import torch

own = False

E4M3_MAX = 448.0


# ---- cases --------------------------------------------------------------------


def decode(name, rows, n_q, n_kv, head_dim, lo, hi, cache, page=16, empty=False):
    case = dict(op="decode", rows=rows, n_q=n_q, n_kv=n_kv, head_dim=head_dim, lo=lo, hi=hi,
                cache=cache, page=page, empty=empty)
    return dict(case, name=name) if name else case


def kv(name, rows, n_kv, head_dim, pool_rows, strided=False, skip=False):
    case = dict(op="kv", rows=rows, n_kv=n_kv, head_dim=head_dim, pool_rows=pool_rows,
                strided=strided, skip=skip)
    return dict(case, name=name) if name else case


def beam(name, groups, beams, vocab, dtype, layers, n_kv, head_dim, tokens, masked=False,
         finished=False):
    case = dict(op="beam", groups=groups, beams=beams, vocab=vocab, dtype=dtype, layers=layers,
                n_kv=n_kv, head_dim=head_dim, tokens=tokens, masked=masked, finished=finished)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one row of a short prompt: the call's latency
        decode("decode one short row", 1, 32, 8, 128, 37, 37, "bf16"),
        # the rows of one filter chunk, each with its own document
        decode("decode filter rows", 256, 32, 8, 128, 96, 2112, "bf16"),
        # one document at the rotary cache's end: the split over the length
        decode("decode one long row", 1, 32, 8, 128, 40960, 40960, "bf16"),
        # long documents under the 64-head model, from the 8-bit cache
        decode("decode long rows 8-bit", 16, 64, 8, 128, 4096, 16384, "fp8"),
        # a serving batch, the largest
        decode("decode serving batch", 128, 32, 8, 128, 4096, 16384, "bf16"),
        # odd head counts, heads of 64, 32-token pages, rows with no key yet
        decode("decode odd heads 8-bit", 37, 10, 2, 64, 1, 1031, "fp8", page=32, empty=True),
        # one new token of each row of a decode batch
        kv("kv decode append", 64, 8, 128, 16384),
        # a full filter chunk's K and V, parked in 8 bits and restored
        kv("kv filter chunk", 110371, 8, 128, 131072),
        # K and V as slices of a wider projection, padding rows skipped
        kv("kv strided odd", 4099, 2, 64, 8192, strided=True, skip=True),
        # one request's four beams
        beam("beam one request", 1, 4, 151936, "float32", 36, 8, 128, 213),
        # a batch of requests, bf16 logits (equal ones occur)
        beam("beam batch", 16, 8, 151936, "bfloat16", 36, 8, 128, 85),
        # a small vocabulary under a mask, with finished and dead beams
        beam("beam masked odd", 7, 5, 4099, "float32", 2, 2, 64, 50, masked=True, finished=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "kv", "beam"])
    head_dim = rng.choice([64, 128, 128])
    n_kv = rng.choice([1, 2, 3, 4, 8, 8])
    if op == "decode":
        group = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 12, 16])
        rows = _log_int(rng, 1, 256)
        hi = _log_int(rng, 1, 32768)
        # at most 128 rows of the longest documents' mean length at 8 heads of 128
        hi = max(1, min(hi, 2 ** 27 // (rows * n_kv * head_dim) * 8))
        lo = max(1, hi // rng.choice([1, 2, 4, 16]))
        return decode(None, rows, group * n_kv, n_kv, head_dim, lo, hi,
                      rng.choice(["bf16", "fp8"]), page=rng.choice([8, 16, 16, 32, 64]),
                      empty=rng.choice([False, True]))
    if op == "kv":
        rows = _log_int(rng, 1, 110000)
        return kv(None, rows, n_kv, head_dim, rows + rng.randrange(16, 4096),
                  strided=rng.choice([False, True]), skip=rng.choice([False, True]))
    beams = rng.choice([1, 2, 3, 4, 5, 8, 8, 11, 16])
    groups = _log_int(rng, 1, max(1, 192 // beams))
    return beam(None, groups, beams, _log_int(rng, 100, 152000),
                rng.choice(["float32", "bfloat16"]), rng.choice([1, 2, 5, 24]), n_kv, head_dim,
                _log_int(rng, 1, 400), masked=rng.choice([False, True]),
                finished=rng.choice([False, True]))


# ---- inputs -------------------------------------------------------------------


def _lengths(case):
    """Tokens of each row: log-uniform over [lo, hi], fixed by the case."""
    rng = np.random.default_rng([case["rows"], case["lo"], case["hi"]])
    n = np.exp(rng.uniform(np.log(case["lo"]), np.log(case["hi"] + 0.999), case["rows"]))
    n = np.clip(n.astype(np.int64), case["lo"], case["hi"])
    if case["empty"]:
        n[::5] = 0          # rows that hold no key
    return n


def _codes(x):
    """(e4m3 codes, exponent bytes) of x over its last axis: the least power of
    two that brings the largest element to 448 or below."""
    amax = x.abs().amax(-1).clamp_min(1e-10)
    bits = (amax / E4M3_MAX).view(torch.int32)
    byte = (bits >> 23) + ((bits & 0x7FFFFF) != 0).int()
    # 2^(127 - byte), from its bits: a quotient by a power of two is exact
    q = x * ((254 - byte) << 23).view(torch.float32)[..., None]
    return q.to(torch.float8_e4m3fn), byte.to(torch.uint8)


def _decode_state(case, g, dev):
    n, page = _lengths(case), case["page"]
    d, n_q, n_kv, rows = case["head_dim"], case["n_q"], case["n_kv"], case["rows"]
    perm = torch.randperm(rows, generator=g, device=dev)
    used = torch.from_numpy(n.astype(np.int32)).to(dev)[perm]
    pages = (used.long() + page - 1) // page
    width = int(-(-max(int(n.max()), 1) // page))
    # pages in a random order, each owned by one row; entries past a row's pages are 0
    n_pages = int((-(-n // page)).sum()) + 3
    order = torch.randperm(n_pages, generator=g, device=dev)
    slot = torch.cumsum(pages, 0) - pages
    at = torch.arange(width, device=dev)[None, :]
    held = at < pages[:, None]
    ids = order[torch.where(held, slot[:, None] + at, 0)]
    table = torch.where(held, ids, 0).to(torch.int32)

    # a mixture of diffuse and sharp heads, rows of V of different size
    gain = torch.exp(0.5 + 0.5 * torch.randn(rows, n_q, 1, generator=g, device=dev))
    q = (gain * torch.randn(rows, n_q, d, generator=g, device=dev)).to(torch.bfloat16)
    pools = []
    for k in range(2):
        x = torch.randn(n_pages * page, n_kv, d, generator=g, device=dev, dtype=torch.bfloat16)
        if k:
            x *= torch.exp(0.5 * torch.randn(n_pages * page, n_kv, 1, generator=g, device=dev,
                                             dtype=torch.bfloat16))
        pools.append(x)
    # rows past a row's tokens hold whatever was there: NaN
    last = torch.clamp(pages - 1, min=0)
    spare = torch.arange(page, device=dev)[None, :] >= (used.long() - last * page)[:, None]
    where = (table.gather(1, last[:, None]).long() * page + torch.arange(page, device=dev))
    where = where[spare & (pages > 0)[:, None]]
    state = dict(op="decode", q=q, table=table, used=used, page=page, case=case)
    if case["cache"] == "fp8":
        (kc, ks), (vc, vs) = (_codes(x.float()) for x in pools)
        for c, s in ((kc, ks), (vc, vs)):
            c.view(torch.uint8)[where] = 0x7F
            s[where] = 0xFF
        state.update(k=kc, v=vc, k_scale=ks, v_scale=vs)
    else:
        for x in pools:
            x[where] = float("nan")
        state.update(k=pools[0], v=pools[1])
    return state


def _kv_state(case, g, dev):
    rows, n_kv, d, pool = case["rows"], case["n_kv"], case["head_dim"], case["pool_rows"]
    if case["strided"]:     # q | k | v of one projection: four query heads for each KV head
        width = 6 * n_kv * d
        qkv = torch.randn(rows, width, generator=g, device=dev, dtype=torch.bfloat16)
        k = qkv[:, 4 * n_kv * d:5 * n_kv * d].view(rows, n_kv, d)
        v = qkv[:, 5 * n_kv * d:].view(rows, n_kv, d)
    else:
        k, v = (torch.randn(rows, n_kv, d, generator=g, device=dev, dtype=torch.bfloat16)
                for _ in range(2))
    # rows of different size, channels that stand out
    for x in (k, v):
        x *= torch.exp(torch.randn(rows, n_kv, 1, generator=g, device=dev)).to(torch.bfloat16)
        x[:, :, 5] *= 12
    dst = torch.randperm(pool - 1, generator=g, device=dev)[:rows]
    back = dst[torch.randperm(rows, generator=g, device=dev)]
    if case["skip"]:
        dst = torch.where(torch.arange(rows, device=dev) % 7 == 3, -1, dst)
    codes = [torch.zeros(pool, n_kv, d, dtype=torch.float8_e4m3fn, device=dev) for _ in range(2)]
    scales = [torch.full((pool, n_kv), 127, dtype=torch.uint8, device=dev) for _ in range(2)]
    return dict(op="kv", k=k, v=v, dst=dst, back=back, k_codes=codes[0], v_codes=codes[1],
                k_scale=scales[0], v_scale=scales[1])


def _beam_state(case, g, dev):
    groups, beams, vocab, page = case["groups"], case["beams"], case["vocab"], 16
    rows = groups * beams
    x = 3 * torch.randn(rows, vocab, generator=g, device=dev)
    if case["masked"]:      # nine tokens of ten are not allowed; some beams have none left
        x[torch.rand(rows, vocab, generator=g, device=dev) < 0.9] = float("-inf")
        if beams > 1:
            x.view(groups, beams, vocab)[::3, -1] = float("-inf")
    scores = -10 + torch.randn(groups, beams, generator=g, device=dev)
    finished = None
    if case["finished"]:
        finished = torch.rand(groups, beams, generator=g, device=dev) < 0.2
    # full pages of a group's beams are shared, the last one and the next are a beam's own
    first = case["tokens"] // page
    n_pages = groups * first + 2 * rows
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    shared = order[:groups * first].view(groups, 1, first).expand(groups, beams, first)
    table = torch.cat([shared, order[groups * first:].view(groups, beams, 2)], 2)
    pools = torch.randn(case["layers"], 2, n_pages * page, case["n_kv"], case["head_dim"],
                        generator=g, device=dev, dtype=torch.bfloat16)
    used = torch.full((groups,), case["tokens"], dtype=torch.int32, device=dev)
    return dict(op="beam", logits=x.to(getattr(torch, case["dtype"])), scores=scores,
                finished=finished, table=table.reshape(rows, first + 2).contiguous(),
                pools=pools, used=used, page=page, pad=1)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    make = dict(decode=_decode_state, kv=_kv_state, beam=_beam_state)[case["op"]]
    return make(case, g, dev)


# ---- one pass -----------------------------------------------------------------


def _exp2_byte(b):
    """2^(b - 127) of an E8M0 byte (255: NaN)."""
    x = torch.where(b == 0, 0x00400000, b.int() << 23).view(torch.float32)
    return torch.where(b == 255, float("nan"), x)


def _plain_decode(s):
    q, table, used, page = s["q"], s["table"], s["used"], s["page"]
    rows, n_q, d = q.shape
    n_kv, width = s["k"].shape[1], table.shape[1]
    at = torch.arange(width * page, device=q.device)
    src = table.long()[:, at // page] * page + at % page
    seen = at[None, :] < used[:, None]

    def rows_of(pool, scale):
        x = pool.view(torch.uint8)[src].view(pool.dtype) if scale is not None else pool[src]
        x = x.float()
        if scale is not None:
            x = x * _exp2_byte(scale[src])[..., None]
        return torch.where(seen[:, :, None, None], x, 0.0).permute(0, 2, 1, 3)
    k = rows_of(s["k"], s.get("k_scale"))                    # [rows, n_kv, keys, d]
    x = q.float().view(rows, n_kv, n_q // n_kv, d) @ k.transpose(2, 3) * d ** -0.5
    del k
    x = torch.where(seen[:, None, None, :], x, float("-inf"))
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    out = p @ rows_of(s["v"], s.get("v_scale"))
    out = torch.where(total > 0, out / total, 0.0)
    lse = (m + torch.log(total)).view(rows, n_q)
    return dict(out=out.reshape(rows, n_q, d).to(torch.bfloat16), lse=lse)


def _plain_kv(s):
    end = s["k_scale"].shape[0] - 1                      # a row that nothing reads
    dst = torch.where(s["dst"] < 0, end, s["dst"])
    out = []
    for x, codes, scale in ((s["k"], s["k_codes"], s["k_scale"]),
                            (s["v"], s["v_codes"], s["v_scale"])):
        c, b = _codes(x.float())
        codes.view(torch.uint8)[dst] = c.view(torch.uint8)
        scale[dst] = b
        got = codes.view(torch.uint8)[s["back"]].view(torch.float8_e4m3fn).float()
        out.append((got * _exp2_byte(scale[s["back"]])[..., None]).to(torch.bfloat16))
    return dict(k=out[0], v=out[1])


def _offers(x, scores, finished, pad, n_out):
    """Each beam's n_out largest logits (equal ones: lowest token first) with
    their scores; a finished beam offers itself alone."""
    groups, beams = scores.shape
    broken = torch.isnan(x).any(-1)
    x = torch.where(torch.isnan(x), float("-inf"), x)
    m = x.amax(-1, keepdim=True)
    top, token = torch.sort(x, dim=-1, descending=True, stable=True)
    lse = m + torch.log(torch.exp(x - torch.where(m == float("-inf"), 0.0, m)).sum(-1, True))
    s = scores.reshape(-1, 1) + (top[:, :n_out] - lse)
    s = torch.where(torch.isnan(s) | broken[:, None], float("-inf"), s)
    token = token[:, :n_out]
    if finished is not None:
        f = finished.reshape(-1, 1)
        own_score = torch.full_like(s, float("-inf"))
        own_score[:, :1] = scores.reshape(-1, 1)
        s, token = torch.where(f, own_score, s), torch.where(f, pad, token)
    return s.view(groups, beams * n_out), token.reshape(groups, beams * n_out)


def _plain_beam(s):
    groups, n = s["scores"].shape
    score, token = _offers(s["logits"].float(), s["scores"], s["finished"], s["pad"], n)
    score, at = torch.sort(score, dim=-1, descending=True, stable=True)
    score, at = score[:, :n], at[:, :n]
    parent = at // n
    # the first child of a beam keeps its own pages, the others take those of
    # the beams without children, in order
    same = parent[:, :, None] == parent[:, None, :]
    later = (same & (torch.arange(n, device=at.device)[None, :, None]
                     > torch.arange(n, device=at.device)[None, None, :])).any(-1)
    childless = ~(parent[:, :, None] == torch.arange(n, device=at.device)).any(1)
    free = torch.sort((~childless).int(), dim=-1, stable=True)[1]
    donor = torch.where(later, free.gather(1, (torch.cumsum(later.int(), 1) - 1).clamp_min(0)),
                        parent)
    first = torch.arange(groups, device=at.device)[:, None] * n
    old, page = s["table"].long(), s["page"]
    width = old.shape[1]
    full = (s["used"].long() // page)[:, None, None]
    kept = torch.arange(width, device=at.device)[None, None, :] < full
    table = torch.where(kept, old[first + parent], old[first + donor])
    # the started page's tokens follow a child that moved
    tail = full.expand(groups, n, 1)
    src = old[first + parent].gather(2, tail)
    dst = table.gather(2, tail)
    slots = torch.arange(page, device=at.device)
    moved = later[:, :, None] & (slots[None, None, :] < (s["used"].long() % page)[:, None, None])
    src, dst = src * page + slots, dst * page + slots
    src = torch.where(moved, src, dst).reshape(-1)
    s["pools"][:, :, dst.reshape(-1)] = s["pools"][:, :, src]
    place = s["used"].long()[:, None, None] // page
    following = table.gather(2, place.expand(groups, n, 1))[:, :, 0] * page + (
        s["used"].long() % page)[:, None]
    return dict(score=score, parent=parent.to(torch.int32),
                token=token.gather(1, at), table=table.view(groups * n, width).to(torch.int32),
                next_row=following.reshape(-1), pools=s["pools"])


def run(state):
    op = state["op"]
    if not own:
        return dict(decode=_plain_decode, kv=_plain_kv, beam=_plain_beam)[op](state)
    from quail_b200 import decode as ops
    if op == "decode":
        if "k_scale" in state:
            cache = ops.QuantLayer(state["k"], state["v"], state["k_scale"], state["v_scale"])
        else:
            cache = (state["k"], state["v"])
        out, lse = ops.decode_attention(state["q"], cache, state["table"], state["used"],
                                        page_tokens=state["page"], with_lse=True)
        return dict(out=out, lse=lse)
    if op == "kv":
        cache = ops.QuantLayer(state["k_codes"], state["v_codes"], state["k_scale"],
                               state["v_scale"])
        ops.kv_quant_write(state["k"], state["v"], cache, state["dst"])
        k, v = ops.kv_quant_read(cache, state["back"])
        return dict(k=k, v=v)
    score, parent, token = ops.beam_select(state["logits"], state["scores"],
                                           finished=state["finished"], pad=state["pad"])
    table, next_row = ops.beam_reorder((state["pools"],), parent, state["used"], state["table"],
                                       page_tokens=state["page"])
    return dict(score=score, parent=parent, token=token, table=table, next_row=next_row,
                pools=state["pools"])


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    if case["op"] == "decode":
        tokens = int(_lengths(case).sum())
        n_q, n_kv, d = case["n_q"], case["n_kv"], case["head_dim"]
        row = 2 * n_kv * (d + 1 if case["cache"] == "fp8" else 2 * d)
        ids = int((-(-_lengths(case) // case["page"])).sum())
        return dict(bytes=tokens * row + 4 * ids + case["rows"] * (4 * n_q * d + 4 * n_q + 4),
                    flops=4 * tokens * n_q * d)
    if case["op"] == "kv":
        # read K and V, write the codes and scales; read those, write K and V
        head = case["rows"] * case["n_kv"] * 2
        return dict(bytes=2 * head * (3 * case["head_dim"] + 1) + 16 * case["rows"],
                    flops=4 * head * case["head_dim"])
    groups, n, vocab = case["groups"], case["beams"], case["vocab"]
    rows = groups * n
    size = 4 if case["dtype"] == "float32" else 2
    # the children that move, were every parent as likely as another
    moved = rows * (1 - 1 / n) ** n
    token = case["layers"] * 2 * case["n_kv"] * case["head_dim"] * 2
    copied = 2 * moved * (case["tokens"] % 16) * token
    tables = 2 * 4 * rows * (case["tokens"] // 16 + 2)
    return dict(bytes=rows * vocab * size + copied + tables + 28 * rows,
                flops=4 * rows * vocab)


# ---- the definitions in 64 bits ------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "decode":
        return _exact_decode(s)
    if case["op"] == "kv":
        return _exact_kv(s)
    return _exact_beam(s)


def _binade(x):
    """The power of two at or below each x > 0, from the bits of a double."""
    return (x.view(torch.int64) >> 52 << 52).view(torch.float64)


def _exact_decode(s):
    q, page = s["q"].double(), s["page"]
    rows, n_q, d = q.shape
    n_kv = s["k"].shape[1]
    out = torch.zeros(rows, n_q, d, dtype=torch.float64, device=q.device)
    lse = torch.full((rows, n_q), -math.inf, dtype=torch.float64, device=q.device)
    for r, n in enumerate(s["used"].tolist()):
        if n == 0:
            continue
        ids = s["table"][r, :-(-n // page)].long()
        at = (ids[:, None] * page + torch.arange(page, device=q.device)).reshape(-1)[:n]
        parts = []
        for name in ("k", "v"):
            x = s[name]
            if name + "_scale" in s:
                power = ((s[name + "_scale"][at].long() + 896) << 52).view(torch.float64)
                x = x.view(torch.uint8)[at].view(torch.float8_e4m3fn).double() * power[..., None]
            else:
                x = x[at].double()
            parts.append(x.transpose(0, 1))                  # [n_kv, keys, d]
        z = q[r].view(n_kv, n_q // n_kv, d) @ parts[0].transpose(1, 2) / math.sqrt(d)
        lse[r] = torch.logsumexp(z, -1).reshape(-1)
        out[r] = (torch.softmax(z, -1) @ parts[1]).reshape(n_q, d)
    return dict(out=out, lse=lse)


def _exact_kv(s):
    """What the rows read back hold, from the rows written: a place's code is
    the nearest multiple of its binade's step (ties to even)."""
    pool = s["k_scale"].shape[0]
    source = torch.full((pool,), -1, dtype=torch.int64, device=s["dst"].device)
    kept = s["dst"] >= 0
    source[s["dst"][kept]] = torch.arange(s["dst"].shape[0], device=source.device)[kept]
    source = source[s["back"]]
    got = {}
    for name in ("k", "v"):
        x = s[name].double()
        largest = x.abs().amax(-1, keepdim=True).clamp_min(1e-10)
        unit = _binade(largest / E4M3_MAX)
        unit = torch.where(unit * E4M3_MAX < largest, 2 * unit, unit)
        y = x / unit
        step = _binade(y.abs().clamp_min(2.0 ** -6)) / 8
        y = torch.round(y / step) * step * unit
        y = y[source.clamp_min(0)]
        y[source < 0] = 0
        got[name] = y
    return got


def _exact_beam(s):
    x = s["logits"].double()
    groups, n = s["scores"].shape
    value = torch.log_softmax(x, -1).nan_to_num(nan=-math.inf)
    best = torch.topk(value, n, -1)[0].view(groups, n, n) + s["scores"].double()[..., None]
    if s["finished"] is not None:
        alone = torch.full_like(best, -math.inf)
        alone[..., 0] = s["scores"].double()
        best = torch.where(s["finished"][..., None], alone, best)
    score = torch.topk(best.reshape(groups, n * n), n, -1)[0]
    return dict(score=score, parent=None, token=None, table=None, next_row=None, pools=None)
