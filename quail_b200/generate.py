"""Continuing rows from their paged KV: prefill, then one token a step for every
beam of every row.

``Generator`` runs the generation operators (quail_b200.decode) with the
prefill's own pipeline and arena:

    prefill     pack_chunk + Qwen3Pipeline.forward_chunk write the prompts' KV
                into the arena, as a filter's documents
    choose      the output head (tied embeddings), beam_select, beam_reorder
    step        embed + norm + quant, qkv GEMM + q/k norm + rotary, the new
                token's KV written (bf16 into the arena, or 8-bit into a
                QuantKV over its memory), decode_attention quantised for
                o_proj, the MLP, the final norm

A row's beams share the full pages of its prompt (the arena's borrowing) and
own the started page and those its new tokens will fill, reserved up front;
beam_reorder keeps each page with one owner as beams die and part. Nothing is
read back between steps but, every few steps, whether all beams have ended.
"""

from dataclasses import dataclass

import numpy as np

from quail_b200 import decode
from quail_b200.loop import HostChunk, pack_chunk

POLL_STEPS = 8   # steps between looks at whether every beam has ended


@dataclass
class Completion:
    """One row's beams, best first: token ids (the ending token included) and
    the sum of their log-probabilities."""

    tokens: list
    scores: list


class Generator:
    """Beam search (greedy with one beam) on one executor's model.

    Args:
        executor: api.B200Executor; its arena must have pages for the rows
            generated at once, free or held by retained keys, which are evicted
            in their order as far as needed.
        kv: "bf16" decodes over the arena's pools; "fp8" over an 8-bit cache in
            pages of the arena's memory, at half the bytes a token and a step.
            The prompts then pass through bf16 pages, a prefill chunk at a time;
            where a few rows' cache and the longest prompt do not fit together,
            the cache gets memory of its own for the call.
    """

    def __init__(self, executor, kv="bf16"):
        if kv not in ("bf16", "fp8"):
            raise ValueError(f"kv {kv!r}: bf16 or fp8")
        self.executor = executor
        self.torch = executor.torch
        self.pipeline = executor.pipeline
        self.arena = executor.arena
        self.weights = executor.weights
        self.kv = kv
        self.quant = None   # the 8-bit cache of a call
        self.workspace = decode.decode_workspace(executor.device)

    # ---- pages ------------------------------------------------------------------

    def _reserve(self, prompts, new_tokens, beams):
        """The arena keys that hold the rows' pages. bf16: one a beam, row by row:
        beam 0 holds the prompt, the others borrow its full pages; each owns pages
        for its own tokens. 8-bit: one for all of them, or none."""
        arena, keys, self.quant = self.arena, [], None
        pages = sum(sum(self._beam_pages(p, new_tokens, beams)) for p in prompts)
        # The arena's pages that a way of placing them asks for, and takes, and
        # whether an 8-bit cache lies inside: two of its pages in one of the arena's,
        # beside the longest prompt's bf16 ones. Else those alone are the arena's, and
        # the cache lies beside it where the arena could hold the rows in bf16.
        half, longest = -(-pages // 2), arena.pages_needed(max(len(p) for p in prompts))
        ways = [(pages, longest if self.kv == "fp8" else pages, False)]
        if self.kv == "fp8":
            ways.insert(0, (half + longest, half + longest, True))
        room = arena.free_pages
        fit = next((w for w in ways if w[0] <= room), None)
        if fit is None:   # with what is kept for later operators
            room += arena.evictable_pages()
            fit = next((w for w in ways if w[0] <= room), None)
        if fit is None:
            raise RuntimeError(
                f"the arena is short of pages for {len(prompts)} rows of {beams} beams and "
                f"{new_tokens} tokens (free: {arena.free_pages})")
        _, need, inside = fit
        arena.evict_retained(need - arena.free_pages)

        def hold(key, tokens, **kw):
            arena.alloc(key, tokens, **kw)
            keys.append(key)
        try:
            if inside:
                self.quant = decode.QuantKV.over(arena)
                hold(("generate", "8-bit"), half * arena.page_tokens)
            elif self.kv == "fp8":
                self.quant = decode.QuantKV(arena.n_layers, pages, arena.page_tokens, arena.n_kv,
                                            arena.d_head, device=arena.pools.device)
            else:
                for i, prompt in enumerate(prompts):
                    n, full = len(prompt), len(prompt) // arena.page_tokens * arena.page_tokens
                    for b in range(beams):
                        borrow = (("generate", (i, 0)), full) if b and full else None
                        hold(("generate", (i, b)), n, capacity_tokens=n + new_tokens,
                             borrow=borrow)
        except Exception:
            self._release(keys)
            raise
        return keys

    def _beam_pages(self, prompt, new_tokens, beams):
        """(the pages that a row's beams share, those they own together)."""
        full = len(prompt) // self.arena.page_tokens
        return full, beams * (self.arena.pages_needed(len(prompt) + new_tokens) - full)

    def _tables(self, prompts, new_tokens, beams, keys):
        """The page ids of every beam, row by row."""
        if self.quant is None:
            return [self.arena.owned_pages(key) for key in keys]
        ids = iter(range(self.quant.n_pages))
        if keys:
            ids = iter([2 * p + half for p in self.arena.owned_pages(keys[0]) for half in (0, 1)])
        tables = []
        for prompt in prompts:
            shared, own = self._beam_pages(prompt, new_tokens, beams)
            full = [next(ids) for _ in range(shared)]
            tables += [full + [next(ids) for _ in range(own // beams)] for _ in range(beams)]
        return tables

    def _release(self, keys):
        for key in reversed(keys):   # borrowers before the key they borrow from
            self.arena.free_key(key)

    # ---- the passes ----------------------------------------------------------------

    def _chunks(self, prompts):
        """(first, end) of the prompts that one forward pass takes: up to the
        executor's budget and, where they only pass through the arena, its free
        pages."""
        room = None if self.quant is None else self.arena.free_pages
        first = tokens = pages = 0
        for i, prompt in enumerate(prompts):
            more = self.arena.pages_needed(len(prompt))
            if i > first and (tokens + len(prompt) > self.executor.budget
                              or (room is not None and pages + more > room)):
                yield first, i
                first, tokens, pages = i, 0, 0
            tokens += len(prompt)
            pages += more
        yield first, len(prompts)

    def _prefill(self, prompts, keys=None, tables=None):
        """Normed last rows [prompts, hidden]; every prompt token's KV written, to
        the pages of its key (bf16) or of its table (8-bit)."""
        normed = []
        for first, end in self._chunks(prompts):
            chunk = prompts[first:end]
            if self.quant is None:
                normed.append(self._forward(chunk, keys[first:end]))
                continue
            held = []
            try:
                for i, prompt in enumerate(chunk):
                    self.arena.alloc(("generate", i), len(prompt))
                    held.append(("generate", i))
                normed.append(self._forward(chunk, held))
                self._quantise(chunk, held, tables[first:end])
            finally:
                # (used again in stream order)
                self._release(held)
        return self.torch.cat(normed)

    def _forward(self, prompts, keys):
        groups = []
        for key, prompt in zip(keys, prompts):
            ids = np.asarray(prompt, dtype=np.int64)
            groups.append(dict(key=key, prefix=ids[:-1], f=len(ids) - 1, suffixes=[ids[-1:]],
                               write_suffix_tokens=1))
        chunk = pack_chunk(self.arena, groups, attention_mode="tree")
        assert isinstance(chunk, HostChunk)
        return self.pipeline.forward_chunk(chunk.upload(self.torch, self.executor.device))

    def _quantise(self, prompts, keys, tables):
        """The prompts' KV from their keys' bf16 rows to the 8-bit rows of their
        tables."""
        arena, torch = self.arena, self.torch
        page = np.arange(arena.page_tokens)
        src = np.concatenate([arena.capacity_rows(key)[:len(p)] for key, p in zip(keys, prompts)])
        dst = np.concatenate([(np.asarray(t)[:, None] * arena.page_tokens + page).reshape(-1)
                              [:len(p)] for t, p in zip(tables, prompts)])
        src, dst = (torch.from_numpy(x).to(self.executor.device) for x in (src, dst))
        for layer in range(arena.n_layers):
            k, v = arena.layer_kv(layer)
            decode.kv_quant_write(k, v, self.quant.layer_kv(layer), dst, src=src)

    def step(self, tokens, positions, rows, table, used):
        """One token of every beam: normed rows [beams, hidden].

        tokens, positions, rows: int64 [n] ids, positions and the pool rows the
        tokens' KV goes to; table: int32 [n, pages]; used: int32 [n] keys, the
        new one included.
        """
        torch, eng, w, cfg = self.torch, self.pipeline.engine, self.weights, self.weights.config
        arena, quant, n = self.arena, self.quant, tokens.shape[0]
        hidden = residual = None
        for index, layer in enumerate(self.pipeline.layers):
            if index == 0:
                residual, x = eng.embed_norm_quant(tokens, w.embed, layer.input_ln)
            else:
                x = eng.norm_quant(hidden, layer.input_ln, residual)
            row_dst = rows if quant is None else None
            if self.pipeline.fused_qkv:
                q, k, v = eng.gemm_qknorm_rope(x, layer.qkv_w, layer.qkv_s, positions, w.cos_sin,
                                               layer.q_norm, layer.k_norm, index, row_dst)
            else:
                qkv = eng.gemm(x, layer.qkv_w, layer.qkv_s)
                q, k, v = eng.qk_norm_rope(qkv, positions, w.cos_sin, layer.q_norm, layer.k_norm,
                                           index, row_dst)
            if quant is None:
                kv = arena.layer_kv(index)
            else:
                kv = quant.layer_kv(index)
                decode.kv_quant_write(k.view(n, cfg.n_kv, cfg.head_dim),
                                      v.view(n, cfg.n_kv, cfg.head_dim), kv, rows)
            o_in = eng.quant_rows(n, cfg.n_q * cfg.head_dim)
            decode.decode_attention(q.view(n, cfg.n_q, cfg.head_dim), kv, table, used,
                                    page_tokens=arena.page_tokens,
                                    softmax_scale=eng.softmax_scale,
                                    quantised=(o_in, eng.use_ue8m0), workspace=self.workspace)
            hidden = eng.gemm(o_in, layer.o_w, layer.o_s)
            x = eng.norm_quant(hidden, layer.post_ln, residual)
            x = eng.gemm_silu_quant(x, layer.gate_up_w, layer.gate_up_s)
            hidden = eng.gemm(x, layer.down_w, layer.down_s)
        every = torch.arange(n, dtype=torch.int64, device=tokens.device)
        return eng.final_norm(hidden, residual, every, w.final_norm)

    def logits(self, normed):
        """The tied output head over the whole vocabulary, f32: in bf16 logits of
        16 and more are steps of 1/8 apart, and so would the scores be."""
        return self.torch.mm(normed, self.weights.embed.t(), out_dtype=self.torch.float32)

    def generate(self, prompts, max_new_tokens, beams=1, eos=None):
        """Completion per prompt (token ids, at least one each): up to
        max_new_tokens tokens for each of `beams` beams; a beam ends at the
        token eos."""
        if max_new_tokens < 1 or not 1 <= beams <= 32:
            raise ValueError("at least one new token and 1 to 32 beams")
        prompts = [list(p) for p in prompts]
        if not all(prompts):
            raise ValueError("an empty prompt")
        longest = max((len(p) for p in prompts), default=0) + max_new_tokens
        if longest > self.weights.config.max_pos:
            raise ValueError(f"{longest} positions: the rotary cache has "
                             f"{self.weights.config.max_pos}")
        if not prompts:
            return []
        keys = self._reserve(prompts, max_new_tokens, beams)
        try:
            with self.torch.cuda.device(self.executor.device):
                return self._search(prompts, keys, max_new_tokens, beams, eos)
        finally:
            self._release(keys)
            self.quant = None

    def _search(self, prompts, keys, max_new_tokens, beams, eos):
        torch, dev, arena = self.torch, self.executor.device, self.arena
        groups, pad = len(prompts), 0 if eos is None else eos
        pages = self._tables(prompts, max_new_tokens, beams, keys)
        table = torch.from_numpy(arena.block_table_rows(pages)).to(dev)
        used = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=dev)
        pools = (arena.pools,) if self.quant is None else self.quant.pools

        normed = self._prefill(prompts, keys[::beams], pages[::beams])
        # every beam's first token comes from the prompt's own row
        scores, parents, tokens = decode.beam_select(
            self.logits(normed), torch.zeros(groups, 1, device=dev), n_out=beams)
        chosen, came = [tokens], [parents]
        finished = None
        for step in range(1, max_new_tokens):
            if eos is not None:
                ended = tokens == eos
                if finished is not None:
                    ended |= finished.gather(1, parents.long())
                finished = ended
                if step % POLL_STEPS == 0 and bool(finished.all()):
                    break
            table, rows = decode.beam_reorder(pools, parents, used, table,
                                              page_tokens=arena.page_tokens)
            each = used.repeat_interleave(beams)
            normed = self.step(tokens.view(-1), each.long(), rows, table, each + 1)
            used = used + 1
            scores, parents, tokens = decode.beam_select(self.logits(normed), scores,
                                                         finished=finished, pad=pad)
            chosen.append(tokens)
            came.append(parents)
        return self._trace(chosen, came, scores, eos)

    def _trace(self, chosen, came, scores, eos):
        """The beams' tokens, from the last step back by their parents."""
        chosen = self.torch.stack(chosen).cpu().numpy()
        came = self.torch.stack(came).cpu().numpy()
        scores = scores.cpu().numpy()
        steps, groups, beams = chosen.shape
        out = []
        for g in range(groups):
            rows = []
            for b in range(beams):
                tokens, at = [], b
                for t in range(steps - 1, -1, -1):
                    tokens.append(int(chosen[t, g, at]))
                    at = int(came[t, g, at])
                tokens.reverse()
                if eos is not None and eos in tokens:
                    tokens = tokens[:tokens.index(eos) + 1]
                rows.append(tokens)
            out.append(Completion(rows, [float(s) for s in scores[g]]))
        return out
