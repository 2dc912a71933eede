"""Greedy serving of many sequences from a paged KV cache: prompts and chunks of any lengths together with sequences
that decode, in one forward pass over their packed rows.

The reference engine holds one sequence in a contiguous cache (qwen3-8b-fp8_rtx-5090/generate.py:55-58, model.py:208-211).
Here the cache is a pool of pages (`DecodeOps.paged_qkv`), so a sequence costs the pages it fills, sequences come and go,
and one pass mixes whole prompts, chunks of long prompts and decode steps:

  embed rows -> per layer: W_qkv (batched FP8 linear, 128 rows a call) -> paged_qkv (head norms, rotary positions, K and V
  into the pages) -> packed_attention (every sequence of the pass begins here) or paged_attention -> W_o, residual, W_gu,
  SwiGLU, W_down, residual -> the last row of each sequence through the final norm, the FP8 head and the argmax.

`beam_search` lets beams share their pages: `paged_plan` (pages, offsets) -> the pass with `shared_attention` -> `beam_select` ->
`paged_fork` (the beams in their new order), all on the device, a captured graph a step.

`paged_kv_read` hands a sequence to a contiguous-cache engine (`export`). `capture` records the decode step of a fixed set
of sequences as a CUDA graph: their lengths and tables are device data.
"""
from __future__ import annotations

import torch

from kernels import ops
from model import FP8, Linear, Qwen3FP8Decode, pack_fp8_tiles, rope_angles, unpack_fp8

GEMM_ROWS = 128   # rows of one batched-linear call


class PagedEngine:
    """pages: pages of the pool (each page_size positions of every layer); max_rows: token rows of one pass; max_seqs:
    sequences of one pass; max_len: the longest sequence (the rotary tables' length); kv_dtype: "bf16" or "fp8";
    rope_scaling: see `model.rope_angles` (contexts past the trained length; "ramp": "dims" for what Qwen3's configurations
    mean). The model's own contiguous cache is not used.

    A pass in which every sequence begins attends over the projection's own rows, any other over the cache: with an fp8
    cache a prompt's logits depend on whether it entered whole (unquantised keys and values) or in chunks."""

    def __init__(self, model: Qwen3FP8Decode, pages: int, page_size: int = 64, max_rows: int = 512, max_seqs: int = 64,
                 max_len: int | None = None, kv_dtype: str = "bf16", rope_scaling: dict | None = None, pdl: bool = True):
        m = self.m = model
        if not isinstance(m.lm_head, Linear):
            raise ValueError("PagedEngine needs the FP8 lm_head (the batched linear takes FP8 weights)")
        if kv_dtype not in ("bf16", "fp8"):
            raise ValueError(f"kv_dtype must be bf16 or fp8, got {kv_dtype!r}")
        self.k = ops()
        self.k.set_pdl(pdl)
        cfg, dev = m.cfg, m.device
        nq, nkv, hd, layers = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, len(m.layers)
        self.page_size, self.max_rows, self.max_seqs = page_size, max_rows, max_seqs
        self.max_len = max_len or m.max_seq
        self.width = -(-self.max_len // page_size)
        dt = FP8 if kv_dtype == "fp8" else torch.bfloat16
        self.k_pages, self.v_pages = (torch.zeros(layers, pages, nkv, page_size, hd, dtype=dt, device=dev) for _ in range(2))
        self.k_scale, self.v_scale = ((torch.zeros(layers, pages, nkv, page_size, device=dev) for _ in range(2))
                                      if kv_dtype == "fp8" else ([None] * layers, [None] * layers))
        self.cos, self.sin = rope_angles(self.max_len, hd, cfg.rope_theta, dev, rope_scaling)
        bf = dict(dtype=torch.bfloat16, device=dev)
        self.resid = torch.empty(max_rows, cfg.hidden, **bf)
        self.qkv = torch.empty(max_rows, (nq + 2 * nkv) * hd, **bf)
        self.q = torch.empty(max_rows, nq, hd, **bf)
        # keys before quantisation, for packed_attention: rows as far apart as the values' in qkv
        self.kb = torch.empty(max_rows, nq + 2 * nkv, hd, **bf)[:, :nkv]
        self.attn = torch.empty(max_rows, nq * hd, **bf)
        self.y = torch.empty(max_rows, cfg.hidden, **bf)
        self.gu = torch.empty(max_rows, 2 * cfg.inter, **bf)
        self.h = torch.empty(max_rows, cfg.inter, **bf)
        self.logits = torch.empty(max_seqs, cfg.vocab, **bf)
        self.best = torch.zeros(max_seqs, dtype=torch.int64, device=dev)
        # scratch of its own: the decode graph runs on it, beside passes of any number of rows
        self.ws = self.k.attention_workspace(dev)
        self.linear_ws = self.k.gemm_scratch(dev, min(max_rows, GEMM_ROWS),
                                             [((nq + 2 * nkv) * hd, cfg.hidden), (cfg.hidden, nq * hd), (2 * cfg.inter, cfg.hidden),
                                              (cfg.hidden, cfg.inter), (cfg.vocab, cfg.hidden)])
        self.w = [tuple(pack_fp8_tiles(unpack_fp8(lin.packed, lin.N, lin.K, lin.pairs)) for lin in (L.qkv, L.o, L.gu, L.down))
                  for L in m.layers]
        self.head_w = pack_fp8_tiles(unpack_fp8(m.lm_head.packed, m.lm_head.N, m.lm_head.K))
        self.free = list(range(pages - 1, -1, -1))
        self.tables: dict[int, list[int]] = {}    # sequence -> its pages
        self.lens: dict[int, int] = {}            # sequence -> positions in the cache
        self._next = 0
        self.graph = None
        self.beam_graph = True                    # beam_search replays a graph for each step

    # ---- sequences ---------------------------------------------------------------------------------------------
    def new(self) -> int:
        """A new, empty sequence."""
        s = self._next
        self._next += 1
        self.tables[s], self.lens[s] = [], 0
        return s

    def release(self, seq: int):
        """Give a sequence's pages back."""
        self.free.extend(reversed(self.tables.pop(seq)))
        del self.lens[seq]

    def reserve(self, seq: int, length: int):
        """Pages for `length` positions; RuntimeError (and nothing taken) where the pool has too few."""
        self._reserve([(seq, length)])

    def _reserve(self, wants):
        """Pages for all of [(sequence, positions)], or none."""
        top = max(length for _, length in wants)
        if top > self.max_len:
            raise RuntimeError(f"sequence of {top} positions: the engine was built for {self.max_len}")
        need = [max(0, -(-length // self.page_size) - len(self.tables[s])) for s, length in wants]
        if sum(need) > len(self.free):
            raise RuntimeError(f"out of pages: {sum(need)} wanted, {len(self.free)} free")
        for (s, _), n in zip(wants, need):
            for _ in range(n):
                self.tables[s].append(self.free.pop())

    def _int32(self, rows):
        return torch.tensor(rows, dtype=torch.int32).to(self.m.device, non_blocking=True)

    def _table(self, seqs):
        """The sequences' pages; -1, which no kernel takes for a page, past them."""
        return self._int32([(self.tables[s] + [-1] * self.width)[:self.width] for s in seqs])

    # ---- the pass ----------------------------------------------------------------------------------------------
    def _linear(self, x, w, scale, out, norm_w=None):
        for r in range(0, x.shape[0], GEMM_ROWS):
            self.k.fp8_gemm_rows(x[r:r + GEMM_ROWS], w, scale, out[r:r + GEMM_ROWS], norm_w=norm_w, eps=self.m.cfg.eps,
                                 scratch=self.linear_ws)

    def _forward(self, tokens, cu, lens, table, max_q, whole, last, sharing=None):
        """One pass over T packed rows (device tensors); `whole`: every sequence begins in this pass. Leaves each
        sequence's logits and argmax key in rows 0 .. B-1 of `logits` and `best`; last: its last row, or None where
        every row is one. sharing: (groups, shared, workspace) of sequences that share their first positions."""
        m, k, cfg = self.m, self.k, self.m.cfg
        T, B = tokens.shape[0], lens.shape[0]
        nq, nkv, hd = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
        resid, qkv, q, kb, attn, y, gu, h = (t[:T] for t in (self.resid, self.qkv, self.q, self.kb, self.attn, self.y, self.gu, self.h))
        v = qkv.view(T, nq + 2 * nkv, hd)[:, nq + nkv:]
        scale = hd ** -0.5
        k.embed_rows(tokens, m.embed, resid)
        for li, L in enumerate(m.layers):
            wq, wo, wgu, wd = self.w[li]
            kp, vp, ks, vs = self.k_pages[li], self.v_pages[li], self.k_scale[li], self.v_scale[li]
            self._linear(resid, wq, L.qkv.scale, qkv, L.ln1)
            k.paged_qkv(qkv, cu, lens, table, kp, vp, q, self.cos, self.sin, q_norm=L.q_norm, k_norm=L.k_norm, eps=cfg.eps,
                        k_scale=ks, v_scale=vs, k_out=kb if whole else None)
            if whole:
                k.packed_attention(q, kb, v, cu, attn, scale, max_q, workspace=self.ws)
            elif sharing:
                k.shared_attention(q, cu, lens, table, *sharing[:2], kp, vp, attn, scale, max_q, k_scale=ks, v_scale=vs, workspace=sharing[2])
            else:
                k.paged_attention(q, cu, lens, table, kp, vp, attn, scale, max_q, k_scale=ks, v_scale=vs, workspace=self.ws)
            self._linear(attn, wo, L.o.scale, y)
            k.add_rows(resid, y)
            self._linear(resid, wgu, L.gu.scale, gu, L.ln2)
            k.swiglu_rows(gu, h)
            self._linear(h, wd, L.down.scale, y)
            k.add_rows(resid, y)
        x = resid if last is None else resid[last]
        logits = self.logits[:B]
        self._linear(x, self.head_w, m.lm_head.scale, logits, m.norm)
        k.argmax_rows(logits, self.best[:B])

    @torch.no_grad()
    def step(self, batch):
        """One pass. batch: [(sequence, new tokens), ...], each with at least one token; at most max_rows tokens and max_seqs
        sequences together. Appends them to the sequences and returns the next token of each (a host list). The
        logits of batch[i] are in logits[i]."""
        seqs, toks = [s for s, _ in batch], [list(t) for _, t in batch]
        n = [len(t) for t in toks]
        if not batch or min(n) < 1 or sum(n) > self.max_rows or len(batch) > self.max_seqs or len(set(seqs)) < len(seqs):
            raise ValueError(f"a pass takes 1 to {self.max_seqs} different sequences with 1 to {self.max_rows} tokens together")
        self._reserve([(s, self.lens[s] + c) for s, c in zip(seqs, n)])
        whole = all(self.lens[s] == 0 for s in seqs)
        cu = [0]
        for c in n:
            cu.append(cu[-1] + c)
        lens = [self.lens[s] + c for s, c in zip(seqs, n)]
        last = None if max(n) == 1 else torch.tensor([c - 1 for c in cu[1:]]).to(self.m.device, non_blocking=True)
        self._forward(self._int32([t for x in toks for t in x]), self._int32(cu), self._int32(lens), self._table(seqs), max(n),
                      whole, last)
        self.lens.update(zip(seqs, lens))
        return self._tokens(len(batch))

    def _tokens(self, B):
        """The packed argmax keys hold ~index in their low words."""
        t = (0xFFFFFFFF - (self.best[:B] & 0xFFFFFFFF)).tolist()
        self.check()
        return t

    @torch.no_grad()
    def generate(self, prompts, gen_len: int, chunk: int | None = None):
        """Greedy generation of gen_len tokens for each prompt (lists of ids): prompts enter in chunks of at most `chunk`
        tokens (default: what a pass takes) beside the sequences that already decode, in their order and as soon as the pool
        has pages for a prompt and its gen_len tokens; a finished sequence's pages go to those that wait. Returns the lists
        of ids."""
        prompts = [list(p) for p in prompts]
        chunk = min(chunk or self.max_rows, self.max_rows)
        if chunk < 1 or not all(len(p) for p in prompts):
            raise ValueError(f"chunks of {chunk} tokens, {sum(not len(p) for p in prompts)} empty prompts")
        if gen_len < 1:
            return [[] for _ in prompts]
        longest = max((len(p) for p in prompts), default=0) + gen_len - 1
        if longest > self.max_len:
            raise RuntimeError(f"sequence of {longest} positions: the engine was built for {self.max_len}")
        need = [-(-(len(p) + gen_len - 1) // self.page_size) for p in prompts]
        if max(need, default=0) > len(self.free):
            raise RuntimeError(f"out of pages: {max(need)} wanted by one prompt, {len(self.free)} free")
        running: list[int] = []
        try:
            return self._generate(running, prompts, need, gen_len, chunk)
        finally:
            for s in running:
                self.release(s)

    def _generate(self, running, prompts, need, gen_len, chunk):
        """`running`: the sequences that hold pages, kept up to date for the caller."""
        out: list[list[int]] = [[] for _ in prompts]
        waiting = list(range(len(prompts)))
        todo, of = {}, {}                        # sequence -> tokens still to enter; its prompt's place
        while waiting or running:
            while waiting and need[waiting[0]] <= len(self.free):
                i, s = waiting.pop(0), self.new()
                running.append(s)
                todo[s], of[s] = prompts[i], i
                self.reserve(s, len(prompts[i]) + gen_len - 1)   # to its end: it cannot run out on the way
            batch, room = [], self.max_rows
            for s in running:                    # those that decode, then prompts
                if not todo[s] and len(batch) < self.max_seqs and room:
                    batch.append((s, out[of[s]][-1:]))
                    room -= 1
            for s in running:
                if todo[s] and room and len(batch) < self.max_seqs:
                    take = todo[s][:min(chunk, room)]
                    todo[s] = todo[s][len(take):]
                    batch.append((s, take))
                    room -= len(take)
            for (s, _), tok in zip(batch, self.step(batch)):
                if not todo[s]:
                    out[of[s]].append(tok)
                    if len(out[of[s]]) == gen_len:
                        running.remove(s)
                        self.release(s)
        return out

    # ---- beam search -------------------------------------------------------------------------------------------
    @torch.no_grad()
    def beam_search(self, prompts, beams: int, gen_len: int, eos: int | None = None, length_penalty: float = 1.0):
        """The `beams` best continuations of each prompt (lists of ids) by beam search, of up to gen_len tokens: per prompt a
        list of (ids, score), best first, score = sum of log-probabilities / (number of ids) ** length_penalty (at least 0).
        Each step takes the 2 * beams best candidates of a prompt's beams: those of the first `beams` that are `eos` become
        hypotheses (the eos is their last id), the first `beams` others go on. Prompts enter as many at a time as passes and
        pool can hold; the beams of a prompt share its pages, and each other's."""
        prompts, K = [list(p) for p in prompts], 2 * beams
        limit = min(self.max_seqs, self.max_rows)
        if not 1 <= beams <= min(32, limit) or gen_len < 1 or not length_penalty >= 0:
            raise ValueError(f"{beams} beams (1 to {min(32, limit)}), {gen_len} tokens, length penalty {length_penalty}")
        if not all(len(p) for p in prompts) or self.m.cfg.vocab < K:
            raise ValueError(f"{sum(not len(p) for p in prompts)} empty prompts, {beams} beams over {self.m.cfg.vocab} tokens")
        longest = max((len(p) for p in prompts), default=0) + gen_len - 1
        if longest > self.max_len:
            raise RuntimeError(f"sequence of {longest} positions: the engine was built for {self.max_len}")
        # a prompt's pages, and for each beam what it writes: from the page that the prompt ends in, which forks copy
        need = [len(p) // self.page_size + beams * (-(-(len(p) + gen_len - 1) // self.page_size) - len(p) // self.page_size + 1)
                for p in prompts]
        if max(need, default=0) > len(self.free):
            raise RuntimeError(f"out of pages: {max(need)} wanted by one prompt, {len(self.free)} free")
        out, at = [], 0
        while at < len(prompts):
            n = 1
            while at + n < len(prompts) and (n + 1) * beams <= limit and sum(need[at:at + n + 1]) <= len(self.free):
                n += 1
            out += self._beam_batch(prompts[at:at + n], sum(need[at:at + n]), beams, gen_len, eos, length_penalty)
            at += n
        return out

    def _beam_batch(self, prompts, pages, beams, gen_len, eos, alpha):
        N, K, R, V, dev = len(prompts), 2 * beams, len(prompts) * beams, self.m.cfg.vocab, self.m.device
        k, seqs, pool = self.k, [], []
        i32 = dict(dtype=torch.int32, device=dev)
        try:
            logits = torch.empty(N, V, dtype=torch.bfloat16, device=dev)
            for i, p in enumerate(prompts):      # prompts alone or in chunks
                seqs.append(self.new())
                for c in range(0, len(p), self.max_rows):
                    self.step([(seqs[i], p[c:c + self.max_rows])])
                logits[i] = self.logits[0]
            held = [x for s in seqs for x in self.tables[s]]
            pool = [self.free.pop() for _ in range(pages - len(held))]
            refs = torch.ones(self.k_pages.shape[1], **i32)
            if pool:
                refs[torch.tensor(pool, device=dev)] = 0
            table, table2 = self._table(seqs), torch.empty(R, self.width, **i32)
            lens = self._int32([len(p) for p in prompts])
            lens2, info = torch.empty(R, **i32), torch.zeros(2, **i32)
            # per request: the candidates of a step, the hypotheses that ended; per step: each beam's parent and token
            cand = (torch.empty(N, K, device=dev), torch.empty(N, K, **i32), torch.empty(N, K, **i32))
            ws = k.beam_workspace(dev, R, V, K)
            scores, token, parents = torch.empty(R, device=dev), torch.empty(R, **i32), torch.empty(R, **i32)
            ended = torch.full((N, beams), -float("inf"), device=dev)
            ended_at = torch.zeros(N, beams, dtype=torch.int64, device=dev)   # step * R + parent row
            hist = torch.zeros(2, gen_len, R, **i32)
            step = torch.zeros(1, dtype=torch.int64, device=dev)
            rank = torch.arange(K, device=dev)
            weight = torch.arange(1, gen_len + 1, device=dev, dtype=torch.float64).pow(-alpha).float()   # of a hypothesis of n tokens
            first_row = (torch.arange(N, device=dev, dtype=torch.int32) * beams)[:, None]

            def choose(rows_logits, rows_scores, cu, parent_of):
                """The candidates of a step -> hypotheses that ended, the beams that go on (their parents, tokens and scores)."""
                k.beam_select(rows_logits, rows_scores, cu, *cand, workspace=ws)
                s, parent, tok = cand
                none = parent < 0
                over = torch.zeros_like(none) if eos is None else (tok == eos) & ~none
                new = torch.where(over & (rank < beams), s * weight[step], -float("inf"))
                best, i = torch.cat((ended, new), 1).topk(beams, dim=1)
                ended.copy_(best)
                ended_at.copy_(torch.cat((ended_at, step * R + parent_of(parent)), 1).gather(1, i))
                on = torch.where(over, rank + K, rank).topk(beams, dim=1, largest=False, sorted=True).indices   # (keys are all different)
                scores.copy_(s.gather(1, on).flatten())
                parents.copy_(parent_of(parent).gather(1, on).flatten())
                token.copy_(tok.clamp(min=0).gather(1, on).flatten())   # (a beam without a candidate: score -inf)
                hist[0].index_copy_(0, step, parents[None])
                hist[1].index_copy_(0, step, token[None])
                step.add_(1)

            # the prompts' own logits: the first tokens; every beam of a request continues its prompt
            choose(logits, torch.zeros(N, device=dev), torch.arange(N + 1, **i32),
                   lambda p: torch.arange(N, **i32)[:, None].expand(N, K).contiguous())
            k.paged_fork(refs, lens, parents, table, table2, lens2, self.k_pages, self.v_pages, *self._scales(), info=info)
            table = torch.empty_like(table2)
            cu, cu_new, ones = torch.arange(N + 1, **i32) * beams, torch.empty(R + 1, **i32), torch.ones(R, **i32)
            seq_lens, shared = torch.empty(R, **i32), torch.empty(N, **i32)
            sharing = (cu, shared, k.shared_workspace(dev, R, self.m.cfg.n_heads))

            def one():
                k.paged_plan(refs, lens2, ones, table2, cu_new, seq_lens, self.page_size, groups=cu, shared=shared, info=info)
                table.copy_(table2)
                self._forward(token, cu_new, seq_lens, table, 1, False, None, sharing)
                choose(self.logits[:R], scores, cu, lambda p: torch.where(p < 0, first_row, p))
                k.paged_fork(refs, seq_lens, parents, table, table2, lens2, self.k_pages, self.v_pages, *self._scales(), info=info)

            graph, done = None, 1
            while done < gen_len:
                if graph is None and done > 1 and self.beam_graph:   # (the first step warmed everything up)
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        one()
                graph.replay() if graph else one()
                done += 1
                if eos is not None and done % 8 == 0:   # a beam's score only falls, its weight ends at weight[-1]
                    top = scores.view(N, beams).amax(1)
                    if bool((ended.amin(1) >= torch.maximum(top * weight[-1], top * weight[done - 1])).all()):
                        break
            live = scores.view(N, beams) * weight[done - 1]
            result = self._hypotheses(hist[:, :done].tolist(), ended.tolist(), ended_at.tolist(), live.tolist(), done, beams, eos)
            self.check()
            return result
        finally:
            torch.cuda.synchronize()
            self.free.extend(reversed(pool))
            for s in seqs:
                self.release(s)

    def _scales(self):
        return (self.k_scale, self.v_scale) if isinstance(self.k_scale, torch.Tensor) else (None, None)

    @staticmethod
    def _hypotheses(hist, ended, ended_at, live, steps, beams, eos):
        """Beams and what ended, followed back through the steps' parents: the best of each request, [(ids, score)]."""
        parents, tokens = hist
        R = len(parents[0])

        def back(step, row):                     # the ids of beam `row` after the first `step` steps
            ids = []
            for t in range(step - 1, -1, -1):
                ids.append(tokens[t][row])
                row = parents[t][row]
            return ids[::-1]

        out = []
        for b in range(len(ended)):
            found = [(s, 0, back(at // R, at % R) + [eos]) for s, at in zip(ended[b], ended_at[b]) if s > -float("inf")]
            found += [(s, 1, back(steps, b * beams + w)) for w, s in enumerate(live[b]) if s > -float("inf")]
            found.sort(key=lambda h: -h[0])
            out.append([(ids, s) for s, _, ids in found[:beams]])
        return out

    # ---- decode graph ------------------------------------------------------------------------------------------
    @torch.no_grad()
    def capture(self, seqs, tokens, steps: int):
        """Record one decode step of these sequences as a CUDA graph, with pages reserved for `steps` more positions.
        `tokens`: the token each continues with. Then `decode`."""
        B, dev = len(seqs), self.m.device
        if not 0 < B <= min(self.max_seqs, self.max_rows, GEMM_ROWS):
            raise ValueError(f"1 to {min(self.max_seqs, self.max_rows, GEMM_ROWS)} sequences")
        if steps < 1:                            # (the warm-up writes the next position, which has to be reserved)
            raise ValueError(f"{steps} steps to capture")
        if len(set(seqs)) < B or len(tokens) != B:
            raise ValueError(f"{B} sequences, {len(set(seqs))} of them different, and {len(tokens)} tokens")
        self._reserve([(s, self.lens[s] + steps) for s in seqs])
        self.graph = None
        self.g_seqs, self.g_steps, self.g_done = list(seqs), steps, 0
        self.g_at = {s: self.lens[s] for s in seqs}                     # where the next replay finds them
        self.token = self._int32(tokens)
        self.state = self._int32([[self.lens[s], 0] for s in seqs])     # [position of the next row, step]
        self.out_tokens = torch.zeros(B, steps, dtype=torch.int32, device=dev)
        self.g_lens = torch.zeros(B, dtype=torch.int32, device=dev)
        self.g_cu, self.g_table = self._int32(list(range(B + 1))), self._table(seqs)   # the graph reads them: kept

        def one():
            torch.add(self.state[:, 0], 1, out=self.g_lens)
            self._forward(self.token, self.g_cu, self.g_lens, self.g_table, 1, False, None)
            self.k.finalize(self.best[:B], self.token, self.out_tokens, self.state)

        token, state = self.token.clone(), self.state.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):            # warm-up; rewrites the rows at the current positions with the same values
            one()
        torch.cuda.current_stream().wait_stream(side)
        self.token.copy_(token)
        self.state.copy_(state)
        self.out_tokens.zero_()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            one()

    def decode(self, steps: int):
        """Replay `steps` captured steps; returns the new tokens of each sequence (host lists). The graph holds its own copy of
        the sequences' pages and positions: once one of them was released, or went on in a `step`, ValueError (and nothing
        is replayed) until the next capture."""
        if self.graph is None:
            raise ValueError("no capture to replay")
        if not 0 <= steps <= self.g_steps - self.g_done:
            raise ValueError(f"{steps} steps: {self.g_steps - self.g_done} steps left of the capture")
        gone = [s for s in self.g_seqs if self.lens.get(s) != self.g_at[s]]
        if gone:
            raise ValueError(f"sequences {gone} of the capture were released or went on since: capture again")
        for _ in range(steps):
            self.graph.replay()
        self.g_done += steps
        for s in self.g_seqs:
            self.g_at[s] += steps
            self.lens[s] = self.g_at[s]
        t = self.out_tokens[:, self.g_done - steps:self.g_done].tolist()
        self.check()
        return t

    # ---- out of the pages --------------------------------------------------------------------------------------
    @torch.no_grad()
    def export(self, seq: int, k_cache: torch.Tensor, v_cache: torch.Tensor):
        """A sequence's rows into one sequence of a contiguous bf16 cache, [layers, n_kv, max_seq, 128] (a `Qwen3FP8Decode`'s
        k_cache[:, b]), from where the contiguous engines go on."""
        n, cfg = self.lens[seq], self.m.cfg
        for t in (k_cache, v_cache):
            if t.dim() != 4 or tuple(t.shape[:2]) != (len(self.m.layers), cfg.n_kv_heads) or t.shape[2] < n or t.shape[3] != cfg.head_dim:
                raise ValueError(f"export wants caches [{len(self.m.layers)}, {cfg.n_kv_heads}, {n} or more, {cfg.head_dim}], got "
                                 f"{tuple(t.shape)}")
        cu, table = self._int32([0, n]), self._table([seq])
        for li in range(len(self.m.layers)):
            self.k.paged_kv_read(cu, table, self.k_pages[li], self.v_pages[li], k_cache[li, :, :n].transpose(0, 1),
                                 v_cache[li, :, :n].transpose(0, 1), k_scale=self.k_scale[li], v_scale=self.v_scale[li])

    def recover(self):
        """After a failed pass, with no launch in flight: zero the counters of the attention workspace and of the linears'
        scratch, and clear the error word. The sequences of the failed pass have to be prefilled again."""
        torch.cuda.synchronize()
        self.ws.zero_()
        self.linear_ws.zero_()
        torch.cuda.synchronize()
        self.k.device_error()

    def check(self):
        """Raise RuntimeError if a kernel recorded a device error since the last check (see `generate.Engine.check`)."""
        err = self.k.device_error()
        if err:
            raise RuntimeError(f"paged pass failed on the device (error word {err:#x}: 1 = a wait timed out, 2 = a bad position, "
                               "page, token or logit, 8 = too few pages)")
