"""Greedy decoding over a paged KV cache, with continuous batching.

The reference pads a ragged batch to its longest prompt, shares one write
slot across rows and masks the holes with a bias (SE:1162-1204,
SE:1263-1335); "PagedAttention & Continuous Batching" is on its roadmap
(README.md:144).  ``PagedDecodeEngine`` runs the same model step over page
pools (``paged.PagedKvCache``):

* every row appends at its own slot (its current length) and attends over
  exactly its own slots, so no bias and no holes;
* a row only holds the pages its request needs;
* ``serve`` admits a waiting request into a row as soon as that row's request
  finishes: the row's pages go back to the pool, the new prompt is prefilled
  into fresh pages of the same row, and the captured step keeps replaying
  for all rows (first come, first served).  Requests with a common prefix fork
  its pages and extend them by their own prompts, and a long prefix is read once
  for all rows in each step;
* ``generate_drafted`` runs a row's last token and drafted ones in one pass and
  keeps those that the model would have drawn;
* all three hold their cache in 8 bits on request (``kv_code``, ``paged8``).

The captured step is the dense engine's step with the paged kernels: for 1..4
rows the fused weight-streaming kernels (QKV + RoPE + paged append, paged
split-K attention, merge + o_proj, gate/up, down, lm_head + argmax), for 5..32
rows their wide forms, above that torch projections around the paged attention
kernels.  Slots, positions,
tokens and the step counter advance on the device inside the graph.
"""

from __future__ import annotations

from collections import deque

import torch
import torch.nn.functional as F

from . import ops, paged, paged8, prefill_ops, step_ops, verify, wide_ops
from .engine import DecodeEngine
from .rope import cos_sin


def lookup_drafts(tokens, n: int, longest: int = 3) -> list:
    """Up to ``n`` tokens that followed an earlier occurrence of the sequence's
    end (its last ``longest`` tokens, else fewer): of the last occurrence with n
    tokens behind it, or of the one with the most, as in a text that repeats
    itself within n tokens."""
    back = list(tokens)[::-1] if longest > 0 else []
    length = behind = i = 0               # of the best occurrence; i tokens stand behind one found
    while (length < longest or behind < n) and back:
        try:
            i = back.index(back[0], i + 1)
        except ValueError:
            break
        k = 1
        while k < longest and i + k < len(back) and back[i + k] == back[k]:
            k += 1
        if k > length or (k == length and behind < n):
            length, behind = k, i
    return back[max(behind - n, 0):behind][::-1]


class PagedDecodeEngine(DecodeEngine):
    """``DecodeEngine`` whose decode step reads and writes a paged KV cache."""

    def new_paged_cache(self, max_rows: int, n_pages: int, page_size: int, pages_per_row: int,
                        code: str | None = None) -> paged.PagedKvCache:
        """A cache in fp16, or in 8 bits of ``code`` (``paged8.CODES``)."""
        cfg = self.cfg
        kind, more = (paged.PagedKvCache, ()) if code is None else (paged8.PagedKv8Cache, (code,))
        return kind(cfg.layers, cfg.kv_heads, n_pages, page_size, max_rows, pages_per_row, self.device, *more)

    # ------------------------------------------------------------------ prefill
    @torch.no_grad()
    def prefill_paged(self, prompts, kv: paged.PagedKvCache, rows):
        """Prompts (list of 1-D id tensors) into rows ``rows`` of ``kv`` (their
        pages mapped beforehand) -> last-token logits (len(rows), vocab).

        One packed varlen launch per layer (``_prefill_ragged`` semantics,
        SE:1162-1204): row b's tokens land in its slots [0, len_b).  A cache in 8
        bits is filled behind the pass, whose own attention is over the fp16
        keys and values."""
        rows = list(rows)
        if len(rows) != len(prompts):
            raise ValueError("one row per prompt")
        if isinstance(kv, paged8.PagedKv8Cache):
            return self._prefill_paged8(prompts, kv, rows)
        table = self._table_rows(kv, rows)
        return self._prefill_packed(
            prompts, lambda i, q, k, v, cu, n, cos, sin, lengths: paged.prefill_varlen_paged(
                q, k, v, cu, n, cos, sin, kv.pools[i][0], kv.pools[i][1], table, 0,
                lengths=lengths),
            lambda hidden, cu, longest: longest <= kv.capacity and self._native_layers(
                hidden, kv.pools, (kv.n_pages, kv.kv_heads, kv.page_size, self.cfg.head_dim),
                len(prompts), longest, cu=cu, block_table=table, n_pages=kv.n_pages,
                page_size=kv.page_size))

    def _prefill_paged8(self, prompts, kv: paged8.PagedKv8Cache, rows):
        """The prompts through dense fp16 caches of their own, which are then quantised:
        every layer's tokens of a row in one launch.  Prompts go together as far as
        those caches take a 64th of the GPU's memory, 2 GiB at least."""
        cfg = self.cfg
        lengths = [int(p.numel()) for p in prompts]
        if max(lengths) > kv.capacity:
            raise ValueError(f"a prompt exceeds the row capacity {kv.capacity}")
        slot_bytes = cfg.layers * 2 * cfg.kv_heads * cfg.head_dim * 2
        memory = max(2 << 30, torch.cuda.get_device_properties(self.device).total_memory // 64)
        logits, at = [], 0
        while at < len(prompts):
            n, longest = 1, lengths[at]
            while at + n < len(prompts) and (n + 1) * max(longest, lengths[at + n]) * slot_bytes <= memory:
                longest = max(longest, lengths[at + n])
                n += 1
            dense = torch.zeros((2, cfg.layers, n, cfg.kv_heads, longest, cfg.head_dim), device=self.device,
                                dtype=torch.float16)
            logits.append(self.prefill_ragged(prompts[at:at + n], list(zip(*dense))))
            zero = torch.zeros(1, device=self.device, dtype=torch.int64)
            for j in range(n):
                m = lengths[at + j]
                k, v = dense[:, :, j, :, :m].transpose(2, 3)
                cu = torch.tensor([0, m], device=self.device, dtype=torch.int32)
                r = rows[at + j]
                paged8.append_paged8(k, v, cu, m, zero, None, None, kv.all_pools, kv.table[r:r + 1], lengths=[m])
            at += n
        return torch.cat(logits)

    def _table_rows(self, kv: paged.PagedKvCache, rows):
        if rows == list(range(rows[0], rows[0] + len(rows))):
            return kv.table[rows[0]:rows[0] + len(rows)]
        return kv.table[torch.tensor(rows, device=self.device)]

    @torch.no_grad()
    def extend_paged(self, chunks, kv: paged.PagedKvCache, rows, contexts, last_only: bool = True):
        """New tokens (list of 1-D id tensors, one or more each) of rows that hold
        ``contexts`` (ints) slots already: appended behind them and run in one
        packed pass -> logits after each row's last token (len(rows), vocab), or
        after every token (packed) without ``last_only``.

        The slots must be mapped; pages of theirs that another row holds too are
        copied first (``PagedKvCache.own_slots``)."""
        cfg, dev = self.cfg, self.device
        rows, contexts = list(rows), [int(c) for c in contexts]
        lengths = [int(c.numel()) for c in chunks]
        if not rows or not len(rows) == len(chunks) == len(contexts) == len(set(rows)):
            raise ValueError("one chunk and one context for each of distinct rows")
        if min(lengths) < 1:
            raise ValueError("a chunk needs at least one token")
        for r, c, n in zip(rows, contexts, lengths):
            kv.own_slots(r, c, n)
        table = self._table_rows(kv, rows)
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        total, most = starts[-1], max(c + n for c, n in zip(contexts, lengths))
        ids = torch.cat([c.reshape(-1).to(dev) for c in chunks])
        cu = torch.tensor(starts, dtype=torch.int32, device=dev)
        ctx = torch.tensor(contexts, dtype=torch.int64, device=dev)
        hidden = F.embedding(ids, self.w["embed"])
        if not self._native_extension(hidden, kv, cu, max(lengths), ctx, most, table):
            pos = torch.cat([torch.arange(c, c + n, device=dev) for c, n in zip(contexts, lengths)])
            cos, sin = cos_sin(pos, self.inv_freq)
            qh, kvh, d = cfg.heads, cfg.kv_heads, cfg.head_dim
            for layer, pools in zip(self.w["layers"], kv.pools):
                proj = F.linear(self._rms(hidden, layer["input_norm"]), layer["qkv_weight"],
                                layer["qkv_bias"]).view(total, qh + 2 * kvh, d)
                new = (proj[:, :qh], proj[:, qh:qh + kvh], proj[:, qh + kvh:], cu, max(lengths), ctx, cos, sin)
                last = dict(lengths=lengths, max_slots=most, scale=self.scale)
                if isinstance(kv, paged8.PagedKv8Cache):
                    att = paged8.prefill_extend_paged8(*new, pools, table, **last)
                else:
                    att = paged.prefill_extend_paged(*new, *pools, table, **last)
                hidden = hidden + F.linear(att.reshape(total, qh * d), layer["o_weight"])
                hidden = hidden + self._mlp(self._rms(hidden, layer["post_norm"]), layer)
        return self._last_logits(hidden[cu[1:].long() - 1] if last_only else hidden)

    def _native_extension(self, hidden, kv, cu, longest: int, ctx, most: int, table) -> bool:
        """Every layer of an extension in one native call, or False where the
        model's or the caches' layout is one it does not take."""
        cfg = self.cfg
        if (hidden.dtype != torch.float16 or not hidden.is_cuda
                or prefill_ops.workspace_bytes(cfg, hidden.shape[0]) < 0):
            return False
        if isinstance(kv, paged8.PagedKv8Cache):
            layers = prefill_ops.layer_table(cfg, self.w["layers"], None, hidden.device, None)
            if layers is None:
                return False
            prefill_ops.extend_layers_paged8(cfg, layers, kv.pools, hidden, cu, longest, ctx, most,
                                             self.inv_freq, table)
            return True
        layers = prefill_ops.layer_table(cfg, self.w["layers"], kv.pools, hidden.device,
                                         (kv.n_pages, kv.kv_heads, kv.page_size, cfg.head_dim))
        if layers is None:
            return False
        prefill_ops.extend_layers(cfg, layers, hidden, cu, ctx, most, self.inv_freq, table, kv.n_pages,
                                  kv.page_size)
        return True

    # ------------------------------------------------------------------ decode
    def make_paged_context(self, kv: paged.PagedKvCache, batch: int, n_cols: int,
                           share_rows: bool = False, prefix=None):
        """Static buffers of the paged graph step over rows [0, batch) of ``kv``.

        ``pos[b]`` is row b's next slot (= its length so far) and its position;
        ``rows[:, step]`` receives each replay's tokens (``n_cols`` columns).
        ``share_rows``: attention may share its workgroups out by the rows'
        lengths (``ops.flash_decode_attention``); without it a row's results do
        not depend on the other rows.  Over caches in 8 bits it changes nothing:
        every row is cut into as many ranges.  ``prefix`` = (prefix_rows, prefix_len,
        prefix_table) of ``paged.flash_decode_attention_prefix_paged``: the step
        attends with it, the shared slots read once."""
        cfg = self.cfg
        dev = self.device
        fused = self.uses_fused_step(batch)
        if fused:
            splits = min(ops.choose_splits(batch, cfg.kv_heads, kv.capacity),
                         self.fused_max_splits(batch))
            flash = ops.make_flash_scratch(batch, cfg.kv_heads, cfg.groups, kv.capacity, dev,
                                           splits=splits, fused=False)
        else:
            flash = ops.make_flash_scratch(batch, cfg.kv_heads, cfg.groups, kv.capacity, dev)
        ctx = {
            "kv": kv,
            "table": kv.table[:batch],
            "flash": flash,
            "token": torch.zeros(batch, device=dev, dtype=torch.long),
            "pos": torch.full((batch,), -1, device=dev, dtype=torch.long),
            "step": torch.zeros(1, device=dev, dtype=torch.long),
            "rows": torch.zeros(batch, n_cols, device=dev, dtype=torch.long),
            "logits": torch.zeros(batch, cfg.vocab, device=dev, dtype=torch.float16),
            "fused": fused,
            "wide": self.uses_wide_step(batch),
            "share_rows": share_rows,
            "prefix": prefix,
        }
        self._step_buffers(ctx, batch)
        f16 = dict(device=dev, dtype=torch.float16)
        ctx["kv8"] = isinstance(kv, paged8.PagedKv8Cache)
        if ctx["kv8"]:
            if prefix is not None:
                raise ValueError("a prefix is read once for all rows over caches in fp16 only")
            # The step's keys and values pass through a page of fp16 for each row.
            ctx["new"] = tuple(torch.zeros(2, batch, cfg.kv_heads, paged.MIN_PAGE, cfg.head_dim, **f16))
            ctx["new_table"] = torch.arange(batch, device=dev, dtype=torch.int32).view(batch, 1)
            ctx["new_slot"] = torch.zeros(batch, device=dev, dtype=torch.long)
        if prefix is not None or ctx["kv8"]:
            ctx["att"] = torch.zeros(batch, cfg.kv_heads, cfg.groups, cfg.head_dim, **f16)
        return ctx

    def _write_to(self, ctx, i: int):
        """Where the QKV launch of layer i appends the step's keys and values: pools,
        table and slots."""
        if ctx["kv8"]:
            return (*ctx["new"], ctx["new_table"], ctx["new_slot"])
        return (*ctx["kv"].pools[i], ctx["table"], ctx["pos"])

    def _attend(self, ctx, i: int, grouped):
        """Attention of layer i's step over the slots up to the one just written."""
        kv, table, pos = ctx["kv"], ctx["table"], ctx["pos"]
        if ctx["kv8"]:
            return paged8.flash_decode_attention_paged8(grouped, kv.pools[i], table, pos, scale=self.scale,
                                                        out=ctx["att"], key=ctx["new"][0][:, :, 0],
                                                        value=ctx["new"][1][:, :, 0])
        if ctx["prefix"] is not None:
            return self._attend_prefix(ctx, grouped, *kv.pools[i])
        return paged.flash_decode_attention_paged(grouped, *kv.pools[i], table, None, ctx["flash"], kv_last=pos,
                                                  scale=self.scale, share_rows=ctx["share_rows"])

    def reads_prefix_once(self, batch: int, slots: int) -> bool:
        """Whether ``serve``'s steps attend ``batch`` rows with a common prefix of
        ``slots`` slots by ``flash_decode_attention_prefix_paged``, rather than each
        row alone over the pages it shares.

        Alone, a row's slots are cut into as many pieces as the step has for it, so
        its time grows with slots / pieces, however many of the rows are parked (4 of
        32 rows behind 16384 slots take what 32 take); together it hardly grows.  The
        fused step has four pieces for any row, the others CUs / (rows * kv heads).
        MI355X, us per layer of the step, alone / together, at heads / kv heads:
        fused, 2 rows of 14/2 2048 slots 27.2 / 27.6, 4096 30.6 / 28.9; of 16/8 2048
        28.2 / 29.7, 4096 31.8 / 31.6; 3 rows of 16/8 4096 32.0 / 32.2; 4 rows of
        14/2 4096 31.8 / 31.6, 6144 35.5 / 32.7; of 16/8 4096 33.0 / 35.7, 6144 36.9
        / 36.7.  Wide, by rows * kv heads * slots: 262144 (8 and 32 rows of 14/2)
        36.6 / 38.8 and 45.4 / 46.5, (8 of 16/8) 37.2 / 38.6, (16 of 8/1) 36.6 /
        39.8; 327680 (5 of 14/2, 5 of 16/8) 41.6 / 39.6 and 39.2 / 38.6; 524288 (16
        of 14/2, 8 of 16/8, 32 of 8/1) 46.1 / 43.5, 44.2 / 40.9 and 48.8 / 46.1."""
        if batch < 2:
            return False
        if self.uses_fused_step(batch):
            return slots >= (4096 if batch == 2 else 6144)
        return batch * self.cfg.kv_heads * slots >= 327680

    def _attend_prefix(self, ctx, grouped, kp, vp):
        rows, length, table = ctx["prefix"]
        return paged.flash_decode_attention_prefix_paged(grouped, kp, vp, ctx["table"], rows, length,
                                                         ctx["pos"], scale=self.scale, out=ctx["att"],
                                                         prefix_table=table)

    def _step(self, ctx):
        if "kv" not in ctx:
            return super()._step(ctx)
        if ctx["fused"]:
            self._step_fused_paged(ctx)
        elif ctx["wide"]:
            self._step_wide_paged(ctx)
        else:
            self._step_torch_paged(ctx)

    def _step_fused_paged(self, ctx):
        cfg = self.cfg
        b = ctx["token"].shape[0]
        eps = cfg.rms_eps
        kv, table, pos = ctx["kv"], ctx["table"], ctx["pos"]
        rope = (pos, self.inv_freq)                              # each row's own position
        hidden, q_rot, h = ctx["hidden"], ctx["q_rot"], ctx["h"]
        for i, layer in enumerate(self.w["layers"]):
            w_qkv, w_gate_up = self.projection_weights(i, b)
            if i == 0:
                paged.rms_qkv_rope_append_paged(self.w["embed"], layer["input_norm"], eps,
                                                w_qkv, layer["qkv_bias"], None, None,
                                                *self._write_to(ctx, i), q_rot, token=ctx["token"],
                                                hidden_out=hidden, positions=rope)
            else:
                paged.rms_qkv_rope_append_paged(hidden, layer["input_norm"], eps,
                                                w_qkv, layer["qkv_bias"], None, None,
                                                *self._write_to(ctx, i), q_rot, positions=rope)
            grouped = q_rot.view(b, cfg.kv_heads, cfg.groups, cfg.head_dim)
            # The slot just written is the row's last valid one.
            if ctx["prefix"] is not None:
                att = self._attend_prefix(ctx, grouped, *kv.pools[i])
                step_ops.gemv_residual(att.view(b, -1), layer["o_weight"], hidden)
            else:
                if ctx["kv8"]:
                    paged8.flash_decode_split_paged8(grouped, kv.pools[i], table, ctx["flash"], pos,
                                                     scale=self.scale, key=ctx["new"][0][:, :, 0],
                                                     value=ctx["new"][1][:, :, 0])
                else:
                    paged.flash_decode_split_paged(grouped, *kv.pools[i], table, None, ctx["flash"],
                                                   kv_last=pos, scale=self.scale)
                step_ops.attn_merge_o_proj(ctx["flash"], self.o_proj_weight(i, b), hidden)
            step_ops.rms_gate_up_swiglu(hidden, layer["post_norm"], eps, w_gate_up, h)
            step_ops.gemv_residual(h, layer["down_weight"], hidden)
        step_ops.rms_lm_head(hidden, self.w["final_norm"], eps, self.lm_head_weight(b), ctx["logits"],
                             ctx["keys"])
        step_ops.argmax_step(ctx["keys"], ctx["token"], ctx["rows"], ctx["step"], None, pos)

    def _step_wide_paged(self, ctx):
        def qkv(i, layer, w_qkv):
            wide_ops.rms_qkv_rope_append_paged(ctx["hidden"], layer["input_norm"], self.cfg.rms_eps,
                                               w_qkv, layer["qkv_bias"], (ctx["pos"], self.inv_freq),
                                               *self._write_to(ctx, i), ctx["q_rot"])

        self._wide_body(ctx, qkv, lambda i, grouped: self._attend(ctx, i, grouped), None)

    def _step_torch_paged(self, ctx):
        cfg = self.cfg
        b = ctx["token"].shape[0]
        pos = ctx["pos"]
        hidden = F.embedding(ctx["token"], self.w["embed"]).view(b, 1, cfg.hidden)
        cos, sin = cos_sin(pos, self.inv_freq)
        for i, layer in enumerate(self.w["layers"]):
            residual = hidden
            q, k, v = self._qkv(self._rms(hidden, layer["input_norm"]), layer)
            q_rot = paged.rope_append_paged(q, k, v, cos, sin, *self._write_to(ctx, i))
            grouped = q_rot.view(b, cfg.kv_heads, cfg.groups, cfg.head_dim)
            att = self._attend(ctx, i, grouped)
            hidden = residual + F.linear(att.reshape(b, 1, cfg.hidden), layer["o_weight"])
            residual = hidden
            hidden = residual + self._mlp(self._rms(hidden, layer["post_norm"]), layer)
        hidden = self._rms(hidden, self.w["final_norm"]).squeeze(1)
        logits = F.linear(hidden, self.w["lm_head"])
        nxt = torch.argmax(logits, dim=-1)
        ctx["logits"].copy_(logits)
        ctx["token"].copy_(nxt)
        ctx["rows"].index_copy_(1, ctx["step"], nxt.unsqueeze(1))
        pos.add_(pos >= 0)  # a parked row stays parked
        ctx["step"].add_(1)

    def capture_paged(self, ctx):
        """Capture the paged step into a hipGraph.  The two warm-ups run with
        every row parked at slot -1 (nothing is appended, nothing is read); the
        state is restored afterwards."""
        side = torch.cuda.Stream(self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        saved = {k: ctx[k].clone() for k in ("token", "pos", "step", "rows")}
        with torch.cuda.stream(side):
            for _ in range(2):
                ctx["pos"].fill_(-1)
                ctx["step"].fill_(0)
                self._step(ctx)
        torch.cuda.current_stream(self.device).wait_stream(side)
        torch.cuda.synchronize(self.device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            self._step(ctx)
        for k, v in saved.items():
            ctx[k].copy_(v)
        torch.cuda.synchronize(self.device)
        ctx["graph"] = graph
        return graph

    # ------------------------------------------------------------------ generation
    @torch.no_grad()
    def generate_paged(self, prompts, max_new_tokens: int, page_size: int = 64,
                       timing: dict | None = None, kv_code: str | None = None):
        """Greedy ids (B, max_new_tokens) for variable-length prompts, each row
        holding only the pages of its own prompt + new tokens: in fp16, or with
        ``kv_code`` "int8" or "e4m3" in 8 bits (``paged8``)."""
        b = len(prompts)
        lengths = [int(p.numel()) for p in prompts]
        need = [n + max(max_new_tokens - 1, 0) for n in lengths]
        ppr = -(-max(need) // page_size)
        n_pages = sum(-(-n // page_size) for n in need)
        kv = self.new_paged_cache(b, n_pages, page_size, ppr, kv_code)
        for r, n in enumerate(need):
            kv.map_row(r, n)
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(4)]
        ev[0].record()
        first = torch.argmax(self.prefill_paged(prompts, kv, range(b)), dim=-1)
        ev[1].record()
        ctx = self.make_paged_context(kv, b, max_new_tokens, share_rows=True)
        self.capture_paged(ctx)
        ctx["rows"][:, 0] = first
        ctx["token"].copy_(first)
        ctx["pos"].copy_(torch.tensor(lengths, device=self.device))
        ctx["step"].fill_(1)
        torch.cuda.synchronize(self.device)
        ev[2].record()
        for _ in range(1, max_new_tokens):
            ctx["graph"].replay()
        ev[3].record()
        torch.cuda.synchronize(self.device)
        if timing is not None:
            timing["prefill_ms"] = ev[0].elapsed_time(ev[1])
            timing["decode_ms"] = ev[2].elapsed_time(ev[3])
            timing["pages"] = n_pages
        self._ctx = ctx
        return ctx["rows"].clone()

    @torch.no_grad()
    def generate_drafted(self, prompts, max_new_tokens: int, draft_len: int = 4,
                         temperature: float = 0.0, seed: int = 0, drafter=lookup_drafts,
                         page_size: int = 64, stats: dict | None = None, kv_code: str | None = None):
        """``max_new_tokens`` ids for each of variable-length prompts (B, new), up
        to ``draft_len`` + 1 of them per pass.

        ``drafter(tokens, n)`` proposes up to n tokens after a row's tokens (a
        list of ints); the default looks them up in the row's own text.  A pass
        runs every unfinished row's last token and its drafts together
        (``extend_paged``), and ``verify.verify_drafts`` keeps what the model
        would have said: the argmax at ``temperature`` 0, else tokens distributed
        as softmax(logits / temperature) whatever the drafter proposes, from
        random numbers of a generator seeded with ``seed``.  ``stats`` (optional
        dict) receives the passes, drafts and accepted drafts.  With ``kv_code`` the
        cache is held in 8 bits; what a block of slots holds then depends a little
        on the drafts that were written to it, kept or not.

        It pays where drafts are mostly kept.  A pass is not captured and runs the
        prompt's kernels: MI355X, Qwen2.5-0.5B shape behind 500 tokens, ms per pass of
        5 positions a row / per captured step of ``generate_paged``: 1 row 1.54 /
        0.50, 4 rows 1.6-1.7 / 0.59, 8 rows 1.7-1.8 / 0.68, so a pass has to give each
        row about three tokens to break even."""
        b, dev = len(prompts), self.device
        if b < 1 or max_new_tokens < 1 or draft_len < 0 or min(int(p.numel()) for p in prompts) < 1:
            raise ValueError("need prompts of one token or more, max_new_tokens >= 1 and draft_len >= 0")
        gen = torch.Generator(dev).manual_seed(seed)
        text = [p.reshape(-1).tolist() for p in prompts]
        ends = [len(t) + max_new_tokens for t in text]
        ppr = -(-max(ends) // page_size)
        kv = self.new_paged_cache(b, sum(-(-n // page_size) for n in ends), page_size, ppr, kv_code)
        for r, n in enumerate(ends):
            kv.map_row(r, n)

        def draw(logits, chunks):
            lengths = [len(c) for c in chunks]
            cu = torch.tensor([sum(lengths[:i]) for i in range(len(chunks) + 1)], dtype=torch.int32,
                              device=dev)
            u, r = (torch.rand(n, generator=gen, device=dev) for n in (sum(lengths), len(chunks)))
            count, out = verify.verify_drafts(
                logits, torch.tensor([t for c in chunks for t in c], device=dev), cu, max(lengths), u, r,
                temperature=temperature, lengths=lengths)
            return [row[:n] for n, row in zip(count.tolist(), out.tolist())]

        passes = drafted = accepted = 0
        new = dict(enumerate(draw(self.prefill_paged(prompts, kv, range(b)), [t[-1:] for t in text])))
        while True:
            for r, ids in new.items():
                if not ids:
                    raise RuntimeError("the logits give no distribution to draw from")
                text[r] += ids
            open_rows = [r for r in range(b) if len(text[r]) < ends[r]]
            if not open_rows:
                break
            chunks = []
            for r in open_rows:
                n = min(draft_len, ends[r] - len(text[r]) - 1)
                ids = [int(t) for t in drafter(text[r], n)][:n] if n > 0 else []
                if any(not 0 <= t < self.cfg.vocab for t in ids):
                    raise ValueError("drafted tokens must be in the vocabulary")
                chunks.append(text[r][-1:] + ids)
            logits = self.extend_paged([torch.tensor(c) for c in chunks], kv, open_rows,
                                       [len(text[r]) - 1 for r in open_rows], last_only=False)
            new = dict(zip(open_rows, draw(logits, chunks)))
            passes += 1
            drafted += sum(len(c) - 1 for c in chunks)
            accepted += sum(max(0, len(ids) - 1) for ids in new.values())
        if stats is not None:
            stats.update(passes=passes, drafted=drafted, accepted=accepted)
        return torch.tensor([t[-max_new_tokens:] for t in text], device=dev)

    @torch.no_grad()
    def serve(self, prompts, max_new_tokens, max_batch: int = 4, page_size: int = 64,
              n_pages: int | None = None, stats: dict | None = None, prefix=None,
              kv_code: str | None = None):
        """Continuous batching: greedy ids for every prompt (list of 1-D tensors),
        ``max_new_tokens`` an int or one per prompt.

        Up to ``max_batch`` rows decode together in one captured step.  Whenever
        requests finish, their pages return to the pool and the next waiting
        requests (first come, first served) are prefilled, each on its own, into
        the freed rows; the graph then keeps replaying.  A request's tokens do
        not depend on the requests it shares the batch with, for one shape of
        the step: ``max_batch`` rows of the pages that the longest request
        needs.  A row with no request is parked at slot -1: it appends nothing and its output is
        ignored.  Returns a list of 1-D id tensors, one per prompt.

        ``prefix`` (1-D ids): every request is the prefix followed by its prompt.
        The prefix is prefilled once, each request's row forks its pages and
        extends them by the prompt, and the steps read the shared pages once for
        all rows where that is the faster way (``reads_prefix_once``).

        ``kv_code`` "int8" or "e4m3" holds the cache in 8 bits (``paged8``): half the
        bytes of a step's attention, twice the slots in a pool's memory.  Each row then
        reads a prefix by itself.
        """
        n_req = len(prompts)
        news = [max_new_tokens] * n_req if isinstance(max_new_tokens, int) else list(max_new_tokens)
        if len(news) != n_req or min(news) < 1:
            raise ValueError("one max_new_tokens >= 1 per prompt")
        common = 0 if prefix is None else int(prefix.numel())
        if prefix is not None and (common < 1 or min(int(p.numel()) for p in prompts) < 1):
            raise ValueError("a prefix and the prompts behind it need at least one token each")
        need = [common + int(p.numel()) + n - 1 for p, n in zip(prompts, news)]
        ppr = -(-max(need) // page_size)
        whole = common // page_size       # pages that rows share
        if n_pages is None:
            n_pages = max_batch * (ppr - whole) + -(-common // page_size)
        kv = self.new_paged_cache(max_batch + (common > 0), n_pages, page_size, ppr, kv_code)
        shared = None
        if common:
            # The row behind the batch holds the prefix for as long as the call runs.
            kv.map_row(max_batch, common)
            self.prefill_paged([prefix], kv, [max_batch])
        if common and kv_code is None and self.reads_prefix_once(max_batch, common):
            i32 = dict(device=self.device, dtype=torch.int32)
            shared = (torch.tensor([0, max_batch], **i32), torch.tensor([common], **i32),
                      kv.table[max_batch:])
        # Upper bound on replays: every request decoded back to back.
        ctx = self.make_paged_context(kv, max_batch, sum(n - 1 for n in news) + 1, prefix=shared)
        self.capture_paged(ctx)
        ctx["step"].fill_(0)
        queue = deque(range(n_req))
        active = {}                       # row -> (request, first replay, replays left)
        results = [None] * n_req
        replays, admitted = 0, 0

        def admit() -> int:
            """Prefill waiting requests into free rows (again while one-token
            requests free their rows at once); returns how many."""
            total = 0
            while True:
                n = admit_once()
                total += n
                if n == 0 or len(active) == max_batch or not queue:
                    return total

        def admit_once() -> int:
            nonlocal admitted
            free = [r for r in range(max_batch) if r not in active]
            batch = []
            while free and queue and kv.free_pages() >= -(-need[queue[0]] // page_size) - whole:
                r, i = free.pop(0), queue.popleft()
                if common:
                    kv.fork_row(max_batch, r, common)
                kv.map_row(r, need[i])
                batch.append((r, i))
            if not batch:
                return 0
            rows = [r for r, _ in batch]
            # One prefill per request: its projections then have the same
            # shapes whatever it is admitted with, so its tokens do not depend
            # on the other rows (the decode step is row-independent too: its
            # context shares no workgroups between rows).
            first = torch.cat([torch.argmax(
                self.extend_paged([prompts[i]], kv, [r], [common]) if common
                else self.prefill_paged([prompts[i]], kv, [r]), dim=-1) for r, i in batch])
            idx = torch.tensor(rows, device=self.device)
            ctx["token"].index_copy_(0, idx, first)
            lens = torch.tensor([common + int(prompts[i].numel()) for _, i in batch], device=self.device)
            ctx["pos"].index_copy_(0, idx, lens)
            for j, (r, i) in enumerate(batch):
                if news[i] == 1:
                    results[i] = first[j:j + 1].clone()
                    kv.release_row(r)
                    ctx["pos"][r] = -1
                else:
                    active[r] = (i, replays, news[i] - 1, first[j:j + 1].clone())
                admitted += 1
            return len(batch)

        admit()
        while active or queue:
            if not active:
                if admit() == 0:
                    raise RuntimeError("page pool too small for the next request")
                continue
            n = min(left for _, _, left, _ in active.values())
            for _ in range(n):
                ctx["graph"].replay()
            replays += n
            for r in list(active):
                i, t0, left, first = active[r]
                if left == n:
                    results[i] = torch.cat([first, ctx["rows"][r, t0:t0 + news[i] - 1]])
                    del active[r]
                    kv.release_row(r)
                    ctx["pos"][r] = -1
                else:
                    active[r] = (i, t0, left - n, first)
            admit()
        if common:
            kv.release_row(max_batch)
        torch.cuda.synchronize(self.device)
        if stats is not None:
            stats["replays"] = replays
            stats["requests"] = admitted
            stats["pages"] = n_pages
        self._ctx = ctx
        return results
