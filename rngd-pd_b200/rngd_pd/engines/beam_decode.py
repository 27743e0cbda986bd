"""Beam search over a paged 4-bit KV cache.

The reference decodes one greedy continuation per lane (BatchDecodeEngine.step,
src/rngd_pd/engines/decode_batch.py:422-442).  This engine keeps the W best of several searches at once in the
same 16 lanes.  A step is one decode step of all beams over their pages (rngd_decode_layers_kv4), the
selection among beams x vocabulary (rngd_pd.beam.select), and the forking of the pages of the beams that go on
(rngd_pd.kv4.fork): beams share the pages they have in common, a prompt is stored once.  All of it stays on the
GPU and is captured into one CUDA graph; the host reads nothing back until it asks for a result.
"""
import ctypes

import torch

from rngd_pd import _lib, beam, kv4
from rngd_pd.engines.decode_batch import MAXB, BatchDecodeEngine

BF = torch.bfloat16


class BeamDecodeEngine:
    def __init__(self, cfg, sd, beams=4, groups=4, pages=256, width=16, eos=-1, window=0, sinks=0, chip=0):
        """beams x groups <= 16 lanes; `sd` as for BatchDecodeEngine (a state dict, or another engine's weights).
        pages: of the pool, each 64 positions of all layers; width: pages a sequence may have.  window, sinks:
        what a token sees (kv4.attention)."""
        if not 1 <= beams <= beam.MAX_BEAMS or groups < 1 or beams * groups > MAXB:
            raise ValueError(f"{groups} groups of {beams} beams: at most {MAXB} lanes")
        if pages < 1 or width < 1 or window < 0 or sinks < 0 or eos >= cfg.vocab:
            raise ValueError(f"pages={pages} width={width} window={window} sinks={sinks} eos={eos}")
        self.cfg, self.W, self.G, self.B = cfg, beams, groups, beams * groups
        self.eos, self.width = eos, width
        self.window, self.sinks = (min(n, 2 ** 31 - 1) for n in (window, sinks))  # 32 bits in the library
        # the decode step's buffers (its lanes are not used: one group of the least width)
        self._e = BatchDecodeEngine(cfg, sd, B=self.B, S=128, group=cfg.n_layers, chip=chip)
        self.w, self.dev, self.stream = self._e.w, self._e.dev, self._e.stream
        with torch.cuda.device(self.dev):
            d, B = self.dev, self.B
            self.pool = kv4.alloc_pool(cfg.n_layers, pages, cfg.n_kv, cfg.head_dim, d)
            self.ref, self.table, self.lens = kv4.empty_state(B, width, pages, d)
            i32 = dict(dtype=torch.int32, device=d)
            self.parents = torch.full((B,), -1, **i32)          # of the next fork
            self.scores = torch.full((B,), float("-inf"), device=d)
            self.done = torch.ones(B, dtype=torch.bool, device=d)
            self.toks = self._e._toks
            self.short = torch.zeros(1, **i32)                  # pages that could not be given, of all steps
            self.missed = torch.zeros(groups, **i32)            # of each group's search: positions without a page
            self._first = width * torch.arange(B, **i32)        # each row's first entry of the table
            self._rows = torch.zeros((2, MAXB, cfg.n_kv, cfg.head_dim), dtype=BF, device=d)
            need = ctypes.c_size_t(0)
            _lib.call("rngd_decode_kv4_workspace", self._e._m, B, width, self.window, self.sinks, ctypes.byref(need))
            self._ws = torch.zeros(max(need.value, 16), dtype=torch.uint8, device=d)
        self._graph = None
        self._steps = []                                        # (tokens, parents) of the steps that are kept
        self._past = 0                                          # steps before them: no search reaches back so far
        self._begun = [None] * groups                           # first step of each group's search, first tokens
        self._held = [0] * groups                               # positions its beams hold
        self._broken = set()                                    # groups whose search a device wait spoilt
        torch.cuda.synchronize(self.dev)

    # ------------------------------------------------------------------ pages
    def _fork(self, parents, room):
        ref, table, lens, short = kv4.fork(self.pool, self.ref, self.table, self.lens, parents, room=room)
        self.ref.copy_(ref)
        self.table.copy_(table)
        self.lens.copy_(lens)
        self.short.add_(short)

    @_lib.on_device
    def begin(self, group, tokens, kv, logits):
        """Start a search in `group`: the prompt's tokens, its cache kv [L, 2, NKV, S, HD] bf16 as a prefill engine
        leaves it (FullPrefillEngine.prefill_kv_device), and the logits [V] after its last token.  What the group
        held is let go."""
        c = self.cfg
        P, n = len(tokens), self.width * kv4.PAGE
        self._check_group(group)
        if not 1 <= P < n:
            raise ValueError(f"a prompt of {P} tokens: 1..{n - 1}")
        if kv.dim() != 5 or kv.shape[:3] != (c.n_layers, 2, c.n_kv) or kv.shape[3] < P or kv.shape[4] != c.head_dim:
            raise ValueError(f"kv {tuple(kv.shape)}: expected [{c.n_layers}, 2, {c.n_kv}, >= {P}, {c.head_dim}]")
        if logits.shape != (c.vocab,) or logits.device != self.dev or kv.device != self.dev:
            raise ValueError(f"logits must be [{c.vocab}] on {self.dev}")
        s, W, r0 = self.stream, self.W, group * self.W
        s.wait_stream(torch.cuda.current_stream(self.dev))
        with torch.cuda.stream(s):
            kv.record_stream(s)
            logits.record_stream(s)
            self._release(r0)
            # pages for the prompt, in the group's first row; to the call all other rows are other holders
            zero = torch.zeros(1, dtype=torch.int32, device=self.dev)
            ref, table, _, short = kv4.fork(self.pool, self.ref, self.table[r0:r0 + 1], zero, room=P)
            self.ref.copy_(ref)
            self.table[r0] = table[0]
            self.short.add_(short)
            self.missed[group:group + 1].add_(short)
            k, v = (kv[:, i, :, :P].transpose(1, 2).unsqueeze(1) for i in (0, 1))
            kv4.store(self.pool, table, zero, k, v)
            self.lens[r0] = P
            # the first tokens: the W best after the prompt, all of them continue the first row
            one = torch.full((W,), float("-inf"), device=self.dev)
            one[0] = 0.0
            sc, pa, tk, dn = beam.select(logits.float().expand(W, -1).contiguous(), one,
                                         torch.zeros(W, dtype=torch.bool, device=self.dev), W, self.eos)
            rows = slice(r0, r0 + W)
            self.scores[rows], self.toks[rows], self.done[rows] = sc[0], tk[0], dn[0]
            self.parents[rows] = torch.where(sc[0] > float("-inf"), pa[0] + r0, -1)
            first = tk[0].clone()
        torch.cuda.current_stream(self.dev).wait_stream(s)
        self._begun[group] = (self._past + len(self._steps), first)
        self._held[group] = P
        self._forget()

    def _check_group(self, group):
        if not 0 <= group < self.G:
            raise IndexError(f"group {group} outside 0..{self.G - 1}")

    def _forget(self):
        """Drop the steps that came before the oldest search."""
        now = self._past + len(self._steps)
        oldest = min((b[0] for b in self._begun if b is not None), default=now)
        del self._steps[:oldest - self._past]
        self._past = oldest

    def _release(self, r0):
        """Empty the rows of the group whose first one is r0 (on the current stream)."""
        par = torch.arange(self.B, dtype=torch.int32, device=self.dev)
        rows = slice(r0, r0 + self.W)
        par[rows] = -1
        self._fork(par, 0)
        self.parents[rows] = -1
        self.scores[rows] = float("-inf")
        self.done[rows] = True
        self.missed[r0 // self.W] = 0
        self._broken.discard(r0 // self.W)

    # ------------------------------------------------------------------- step
    def _step(self):
        """Fork as selected, one decode step, select: all queued on the current stream."""
        e, m, h = self._e, self._e._m, _lib.stream_handle()
        self._fork(self.parents, 1)
        # a beam without a page for the position that comes now lost it in this fork: its group's search is spoilt
        live = self.lens > 0
        page = self.table.view(-1).index_select(0, self._first + self.lens // kv4.PAGE)
        self.missed.add_(((page < 0) & live).view(self.G, self.W).sum(1, dtype=torch.int32))
        e._pos.copy_(self.lens)
        io = e._io(self._rows[0], self._rows[1])
        cache = _lib.Kv4(pool=self.pool.data_ptr(), layer_bytes=self.pool.stride(0), P=self.pool.shape[1],
                         ld_table=self.width, table=self.table.data_ptr(), window=self.window, sinks=self.sinks,
                         rows=self._rows.data_ptr(), workspace=self._ws.data_ptr(), workspace_bytes=self._ws.numel())
        _lib.call("rngd_decode_embed", m, io, h)
        _lib.call("rngd_decode_layers_kv4", m, io, cache, 0, self.cfg.n_layers, h)
        _lib.call("rngd_decode_lmhead", m, io, h)
        self.lens.add_(live)
        sc, pa, tk, dn = beam.select(e._logits, self.scores, self.done, self.W, self.eos)
        self.scores.copy_(sc.view(-1))
        # a beam without continuation lets go of its pages
        self.parents.copy_(torch.where(self.scores > float("-inf"), pa.view(-1), -1))
        self.toks.copy_(tk.view(-1))
        self.done.copy_(dn.view(-1))

    @_lib.on_device
    def step(self, n=1):
        """n steps of every search.  Queued on the engine's stream; nothing is read back."""
        if n < 0:
            raise ValueError(f"{n} steps")
        for g in range(self.G):
            if self._begun[g] is not None and self._held[g] + n > self.width * kv4.PAGE:
                raise ValueError(f"group {g} holds {self._held[g]} positions: {n} more do not fit {self.width} pages")
        s = self.stream
        s.wait_stream(torch.cuda.current_stream(self.dev))
        with torch.cuda.stream(s):
            for _ in range(n):
                if self._graph is None and self._e.use_graph:
                    # one plain run on a copy of the state loads the kernels; then the step is captured
                    names = ("ref", "table", "lens", "parents", "scores", "done", "toks", "short", "missed")
                    keep = [getattr(self, x).clone() for x in names]
                    self._step()
                    for x, t in zip(names, keep):
                        getattr(self, x).copy_(t)
                    s.synchronize()
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
                        self._step()
                    self._graph = g
                if self._graph is not None:
                    self._graph.replay()
                else:
                    self._step()
                if any(b is not None for b in self._begun):
                    self._steps.append((self.toks.clone(), self.parents.clone()))
        for g in range(self.G):
            if self._begun[g] is not None:
                self._held[g] += n

    # ----------------------------------------------------------------- result
    @_lib.on_device
    def result(self, group):
        """The group's beams that have a continuation, best first: [(score, tokens)], tokens up to and with the
        first eos.  Raises where the pool ran out of pages during the group's search (others are not concerned)."""
        self._check_group(group)
        if self._begun[group] is None:
            raise ValueError(f"group {group} has no search")
        self.stream.synchronize()
        missed = int(self.missed[group].item())
        if missed:
            raise RuntimeError(f"the pool ran out in this search: {missed} times a page could not be given")
        if _lib.device_status():  # reading clears it
            self._broken.update(g for g in range(self.G) if self._begun[g] is not None)
        if group in self._broken:
            raise RuntimeError("a device wait ran out during this search")
        start, first = self._begun[group]
        r0 = group * self.W
        hist = [(t.tolist(), p.tolist()) for t, p in self._steps[start - self._past:]]
        scores, first = self.scores.tolist(), first.tolist()
        out = []
        for r in range(r0, r0 + self.W):
            if scores[r] == float("-inf"):
                continue
            seq, at = [], r
            for t, p in reversed(hist):
                seq.append(t[at])
                at = p[at]
            seq.append(first[at - r0])
            seq.reverse()
            if self.eos in seq:
                seq = seq[:seq.index(self.eos) + 1]
            out.append((scores[r], seq))
        return out

    @_lib.on_device
    def end(self, group):
        """Let go of the group's pages and beams."""
        self._check_group(group)
        s = self.stream
        s.wait_stream(torch.cuda.current_stream(self.dev))
        with torch.cuda.stream(s):
            self._release(group * self.W)
        self._begun[group] = None
        self._held[group] = 0
        self._forget()

    @_lib.on_device
    def compact(self):
        """Move the held pages to the front of the pool; returns how many there are (waits for it)."""
        with torch.cuda.stream(self.stream):
            ref, table, live = kv4.compact(self.pool, self.ref, self.table)
            self.ref.copy_(ref)
            self.table.copy_(table)
            return int(live.item())  # on the engine's stream, after what is queued there
