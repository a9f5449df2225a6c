"""Paged K/V cache: a batch of sequences over one pool of pages, and batched decode on top of it.

The reference keeps one contiguous cache for one sequence (gsd_lq_cpu_engine.c:186-330).  Here the positions
of every sequence are cut into pages of a common pool, so that sequences of any length share the memory,
a prompt's pages can be shared by several continuations, and a page is copied only when one of them writes
to it.  The page table and the reference counts live on the device: a decode step allocates its pages itself
and is captured as one CUDA graph.
"""
from __future__ import annotations

import math

import torch

from . import _lib as L
from . import ops
from .batch import BatchDecoder

KV_TYPES = {torch.float16: L.KV_F16, torch.bfloat16: L.KV_BF16}


class PagedKV:
    """A pool of pages k, v [layers][pages][page_size][kv heads][head_dim] (fp16 or bf16), the page table
    [sequences][blocks] and the pages' reference counts (int32, on the device).

    The calls are asynchronous on the current stream; calls on one pool must be ordered (one stream, or
    streams that wait for one another)."""

    def __init__(self, n_layers: int, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, n_seqs: int,
                 max_blocks: int, dtype=torch.float16, device=None):
        if min(n_layers, n_pages, page_size, n_kv_heads, n_seqs, max_blocks) < 1:
            raise ValueError("every size of a paged cache must be at least 1")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        shape = (n_layers, n_pages, page_size, n_kv_heads, head_dim)
        self._init(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                   torch.full((n_seqs, max_blocks), -1, dtype=torch.int32, device=device),
                   torch.zeros(n_pages, dtype=torch.int32, device=device))

    @classmethod
    def wrap(cls, k, v, table, refs):
        """A cache over the caller's tensors (not copied)."""
        self = cls.__new__(cls)
        self._init(k, v, table, refs)
        return self

    def _init(self, k, v, table, refs):
        for t, name in ((k, "k"), (v, "v"), (table, "table"), (refs, "refs")):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a tensor")
        if k.dtype not in KV_TYPES:
            raise TypeError(f"the pool must be float16 or bfloat16, not {k.dtype}")
        dev = k.device
        ops._check(k, "k", k.dtype, (None,) * 5, dev)
        ops._check(v, "v", k.dtype, tuple(k.shape), dev)
        ops._check(table, "table", torch.int32, (None, None), dev)
        ops._check(refs, "refs", torch.int32, (k.shape[1],), dev)
        self.k, self.v, self.table, self.refs, self.device = k, v, table, refs, dev
        self.n_layers, self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = k.shape
        self.n_seqs, self.max_blocks = table.shape
        if min(k.shape) < 1 or min(table.shape) < 1:
            raise ValueError("every size of a paged cache must be at least 1")
        if self.head_dim not in (32, 64, 128):
            raise ValueError("head_dim must be 32, 64 or 128")
        if self.n_seqs > L.PAGED_MAX_SEQS:
            raise ValueError(f"at most {L.PAGED_MAX_SEQS} sequences")
        i32 = dict(dtype=torch.int32, device=dev)
        # page pairs to copy: one per row of a reservation, half the pool's pages at most in a compaction
        n = max(L.PAGED_MAX_SEQS, self.n_pages // 2 + 1)
        self.src, self.dst = torch.full((n,), -1, **i32), torch.full((n,), -1, **i32)
        self.counts = torch.zeros(4, **i32)
        self._lists = tuple(t.data_ptr() for t in (self.src, self.dst, self.counts))
        self._to = torch.zeros(self.n_pages, **i32)
        self._desc = L.PagedKVDesc(k=k.data_ptr(), v=v.data_ptr(), kv_type=KV_TYPES[k.dtype], layers=self.n_layers,
                                   n_pages=self.n_pages, page_size=self.page_size, n_kv_heads=self.n_kv_heads,
                                   head_dim=self.head_dim, table=table.data_ptr(), refs=refs.data_ptr(),
                                   n_seqs=self.n_seqs, max_blocks=self.max_blocks)

    def desc(self) -> L.PagedKVDesc:
        return self._desc

    # ------------------------------------------------------------------ pages
    def fork(self, parent):
        """Sequence b takes over the pages of sequence parent[b], all at once; b itself: kept, -1: freed
        (gsdlq_pages_fork).  parent: int32 device tensor [n_seqs]."""
        ops._ints(parent, "parent", self.device, self.n_seqs)
        status = L.load().gsdlq_pages_fork(self._desc, parent.data_ptr(), ops._stream_on(self.device))
        if status:
            L.check(status, "gsdlq_pages_fork")

    def reserve(self, pos, row_seq=None):
        """A page of its own for every row's position (gsdlq_pages_reserve), with the contents copied where the
        page was shared (gsdlq_pages_copy).  pos, row_seq: int32 device tensors [rows], as in attention.
        Afterwards counts holds (pages copied, rows that got no page, pages taken)."""
        rows = ops._rows(self, pos, row_seq, self.device)
        if rows > L.PAGED_MAX_SEQS:
            raise ValueError(f"at most {L.PAGED_MAX_SEQS} rows")
        stream, (src, dst, counts) = ops._stream_on(self.device), self._lists
        status = L.load().gsdlq_pages_reserve(self._desc, None if row_seq is None else row_seq.data_ptr(),
                                              pos.data_ptr(), rows, src, dst, rows, counts, stream)
        if status:
            L.check(status, "gsdlq_pages_reserve")
        self._copy(src, dst, counts, rows, stream)

    def compact(self, max_moves: int | None = None):
        """Move the pages in use to the front of the pool, the highest first, at most ``max_moves`` of them
        (gsdlq_pages_compact, gsdlq_pages_copy).  Afterwards counts holds (pages moved, pages in use, 1 + the
        highest page in use)."""
        most = self.n_pages // 2 + 1 if max_moves is None else min(int(max_moves), self.n_pages // 2 + 1)
        if most < 1:
            raise ValueError("max_moves must be at least 1")
        stream, (src, dst, counts) = ops._stream_on(self.device), self._lists
        status = L.load().gsdlq_pages_compact(self._desc, src, dst, most, counts, self._to.data_ptr(),
                                              4 * self.n_pages, stream)
        if status:
            L.check(status, "gsdlq_pages_compact")
        self._copy(src, dst, counts, most, stream)

    def copy_pages(self, src, dst, counts):
        """Copy page src[i] over page dst[i] in every layer, i < counts[0] (gsdlq_pages_copy): int32 device
        tensors.  A page must not be a destination twice, nor a source and a destination."""
        n = ops._ints(src, "src", self.device)
        ops._ints(dst, "dst", self.device, n)
        if ops._ints(counts, "counts", self.device) < 1 or n < 1:
            raise ValueError("src, dst and counts must not be empty")
        self._copy(src.data_ptr(), dst.data_ptr(), counts.data_ptr(), n, ops._stream_on(self.device))

    def _copy(self, src, dst, counts, n, stream):
        status = L.load().gsdlq_pages_copy(self._desc, src, dst, counts, n, stream)
        if status:
            L.check(status, "gsdlq_pages_copy")

    def resized(self, n_pages: int) -> "PagedKV":
        """This cache in a pool of ``n_pages`` pages, larger or (after compact) smaller: a new pool with the pages'
        contents and counts, and the same table tensor, so that this one, and the jobs, graphs and decoders made over
        it, must not be used any more.  Waits for the device."""
        keep = min(int(n_pages), self.n_pages)
        if n_pages < 1:
            raise ValueError("at least one page")
        if bool((self.refs[keep:] > 0).any()) or bool((self.table >= keep).any()):
            raise ValueError("pages in use lie behind the new end: compact first")
        shape = (self.n_layers, int(n_pages)) + tuple(self.k.shape[2:])
        k, v = (torch.zeros(shape, dtype=self.k.dtype, device=self.k.device) for _ in range(2))
        k[:, :keep], v[:, :keep] = self.k[:, :keep], self.v[:, :keep]
        refs = torch.zeros(int(n_pages), dtype=torch.int32, device=self.k.device)
        refs[:keep] = self.refs[:keep]
        return PagedKV.wrap(k, v, self.table, refs)

    def pages_in_use(self) -> int:
        """Pages that a table entry names (waits for the device)."""
        return int((self.refs > 0).sum())


class PagedBatchDecoder(BatchDecoder):
    """BatchDecoder over a paged cache: up to ``batch`` sequences share ``n_pages`` pages of ``page_size``
    positions.  A sequence at position -1 is idle (its logits and pick mean nothing).

    Each step reserves the pages it writes to, copying those that are shared, before it runs the layers, so
    prompts can be shared: prefill one sequence, fork() it, and let the copies continue."""

    def __init__(self, model, batch: int, n_pages: int, page_size: int = 16, max_seq: int | None = None,
                 kv_dtype=torch.float16, use_graph: bool = True):
        if n_pages < 1 or page_size < 1:
            raise ValueError("a pool needs at least one page of at least one position")
        self._pool = (int(n_pages), int(page_size), kv_dtype)
        super().__init__(model, batch, max_seq, use_graph)

    def _init_cache(self):
        m, B = self.m, self.B
        n_pages, page_size, dtype = self._pool
        self.kv = PagedKV(m.n_layers, n_pages, page_size, m.n_kv_local, m.head_dim, B, -(-self.S // page_size), dtype,
                          m.device)
        self._jobs = {}
        rows = max(B, m.PREFILL_CHUNK)
        self.awork = ops.attention_paged_work(self.kv, rows, m.n_heads_local)
        i32 = dict(dtype=torch.int32, device=m.device)
        self.row_pos = torch.full((m.PREFILL_CHUNK,), -1, **i32)
        self.row_seq, self.row_zero = (torch.zeros(m.PREFILL_CHUNK, **i32) for _ in range(2))
        self.idle = torch.ones(B, dtype=torch.bool, device=m.device)
        self.pos.fill_(-1)
        self._logit_graph = None

    # ------------------------------------------------------------------ the step
    def _layer_jobs(self, key, l, q, k, v, out, pos, row_seq):
        j = self._jobs.get((key, l))
        if j is None:
            m = self.m
            # (positions at max_seq and above have no angle: reported as bad positions)
            j = (ops.paged_append_job(self.kv, l, q, k, v, q, pos, m.rope_cs[:self.S], row_seq),
                 ops.paged_attn_job(self.kv, l, q, out, pos, 1.0 / math.sqrt(m.head_dim), self.awork, row_seq))
            self._jobs[(key, l)] = j
        return j

    def _heads(self, t, n):
        return t.unflatten(-1, (n, self.m.head_dim))

    def _attend(self, l, qp, kp, vp, stride):
        m = self.m
        nh, nkv, hd = m.n_heads_local, m.n_kv_local, m.head_dim
        if stride:  # column ranges of the stacked linear's rows
            q, k, v = self.qkv.split((nh * hd, nkv * hd, nkv * hd), dim=1)
        else:
            q, k, v = self.q, self.k, self.v
        append, attn = self._layer_jobs("step", l, self._heads(q, nh), self._heads(k, nkv), self._heads(v, nkv),
                                        self._heads(self.att, nh), self.pos, None)
        ops.rope_kv_paged(append)
        ops.attention_paged(attn)

    def _run(self, with_pick: bool = True):
        self.kv.reserve(self.pos)
        super()._run(with_pick)
        if with_pick:
            self.pos.masked_fill_(self.idle, -1)  # (the pick moved every position on)

    def set_tokens(self, ids, positions):
        """The next input token and its position, per sequence; position -1: the sequence is idle."""
        positions = [int(p) for p in positions]
        live = [p >= 0 for p in positions]
        if any(p < -1 for p in positions):
            raise ValueError("positions start at 0 (-1: idle)")
        super().set_tokens([int(t) if a else 0 for t, a in zip(ids, live)] if len(ids) == len(live) else ids,
                           [max(p, 0) for p in positions])
        self.idle.copy_(torch.tensor([not a for a in live]))
        self.pos.masked_fill_(self.idle, -1)

    def step_logits(self):
        """The layers and the LM head for the set tokens, without a pick: logits into self.logits; tokens and
        positions stay."""
        if not self.use_graph:
            self._run(with_pick=False)
            return
        if self._logit_graph is None:
            self._run(with_pick=False)  # eager warm-up outside the capture; the replay does the same again
            torch.cuda.synchronize(self.m.device)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                self._run(with_pick=False)
            self._logit_graph = g
        self._logit_graph.replay()

    # ------------------------------------------------------------------ sequences
    def prefill(self, b: int, ids, start_pos: int = 0):
        """Fill sequence b's pages with ``ids`` at positions start_pos.. (chunked tensor-core prefill).  MemoryError
        when the pool runs out (what came before that chunk is stored)."""
        ids = [int(t) for t in ids]
        if not 0 <= b < self.B:
            raise ValueError(f"sequence outside [0, {self.B})")
        if start_pos < 0 or start_pos + len(ids) > self.S:
            raise ValueError("prefill past max_seq")
        m, chunk = self.m, self.m.PREFILL_CHUNK
        self.row_seq.fill_(b)
        table = self.kv.table[b].data_ptr()
        for c in range(0, len(ids), chunk):
            part = ids[c:c + chunk]
            n, p0 = len(part), start_pos + c
            self.row_pos[:n].copy_(torch.arange(p0, p0 + n, dtype=torch.int32))
            self.kv.reserve(self.row_pos[:n], self.row_seq[:n])
            if int(self.kv.counts[1]):
                raise MemoryError("the page pool is exhausted")

            def attend(l, buf):
                append, attn = self._layer_jobs(
                    "prefill", l, self._heads(buf["q"], m.n_heads_local), self._heads(buf["k"], m.n_kv_local),
                    self._heads(buf["v"], m.n_kv_local), self._heads(buf["att"], m.n_heads_local), self.row_pos,
                    self.row_zero)
                for j in (append, attn):  # the sequence alone, as sequence 0: its rows share their tiles
                    j.rows, j.kv.table, j.kv.n_seqs = n, table, 1
                ops.rope_kv_paged(append)
                ops.attention_paged(attn)

            m._prefill_chunk(part, p0, attend=attend)

    def fork(self, parents):
        """Sequence b continues sequence parents[b] (shared pages, and its token, position and output); b
        itself: unchanged, -1: freed and idle.  parents: B ints."""
        parents = [int(p) for p in parents]
        if len(parents) != self.B or any(not -1 <= p < self.B for p in parents):
            raise ValueError(f"one parent in [-1, {self.B}) per sequence")
        par = torch.tensor(parents, dtype=torch.int32, device=self.m.device)
        self.kv.fork(par)
        at, gone = par.clamp_min(0).long(), par < 0
        for t in (self.ids, self.pos, self.out_ids, self.idle):
            t.copy_(t[at])
        self.idle |= gone
        self.pos.masked_fill_(self.idle, -1)

    def free(self, seqs):
        """Give back the pages of the given sequences, which become idle."""
        gone = {int(b) for b in seqs}
        if any(not 0 <= b < self.B for b in gone):
            raise ValueError(f"sequence outside [0, {self.B})")
        self.fork([-1 if b in gone else b for b in range(self.B)])

    def _room(self, lengths):
        """Raise MemoryError unless sequences of the given lengths fit the pool once this decoder's are freed, beside
        the pages that other tables over it hold (waits for the device)."""
        kv = self.kv
        own = kv.table[(kv.table >= 0) & (kv.table < kv.n_pages)].long()
        mine = torch.zeros_like(kv.refs).scatter_add_(0, own, torch.ones_like(own, dtype=kv.refs.dtype))
        need, have = sum(-(-n // kv.page_size) for n in lengths), kv.n_pages - int((kv.refs > mine).sum())
        if need > have:
            raise MemoryError(f"{need} pages needed, {have} free")

    def generate(self, prompts, max_new_tokens: int) -> list[list[int]]:
        """Greedy continuation of every prompt; what the sequences held before is freed (not if the call is refused:
        ValueError, or MemoryError where the pool is too small)."""
        self._check_prompts(prompts, max_new_tokens)
        self._room([len(pr) + max_new_tokens - 1 for pr in prompts])  # (the last token is not stored)
        self.free(range(self.B))
        return super().generate(prompts, max_new_tokens)

    def beam_search(self, prompt, beams: int, max_new_tokens: int, eos_id: int | None = None):
        """The ``beams`` continuations of ``prompt`` with the highest sum of log probabilities that a beam search
        finds: a list of (token ids, sum), best first.  The prompt's pages are shared by all beams; each step
        forks the beams that go on and copies only the pages they write to.  eos_id ends a continuation (it
        counts in the sum and is not returned).  Equal sums: the lower beam, then the lower token."""
        prompt = [int(t) for t in prompt]
        if not prompt or max_new_tokens < 1 or len(prompt) + max_new_tokens > self.S:
            raise ValueError("a prompt of at least one token, and prompt + new tokens within max_seq")
        if not 1 <= beams <= min(self.B, L.MAX_TOP - 1):
            raise ValueError(f"beams outside [1, {min(self.B, L.MAX_TOP - 1)}]")
        if not 0 <= prompt[-1] < self.m.vocab_size:
            raise ValueError("token id outside the vocabulary")
        full = (len(prompt) - 1) // self.kv.page_size
        own = -(-(len(prompt) + max_new_tokens - 1) // self.kv.page_size) - full  # blocks that the beams write to
        self._room([full * self.kv.page_size] + [own * self.kv.page_size] * beams)
        self.free(range(self.B))
        self.prefill(0, prompt[:-1])
        rest = [-1] * (self.B - beams)
        live, done = [([], 0.0)], []
        tokens, at = [prompt[-1]], len(prompt) - 1
        top = min(beams + (eos_id is not None), self.m.vocab_size)
        for step in range(max_new_tokens):
            self.set_tokens(tokens + [0] * (self.B - len(tokens)), [at] * len(tokens) + [-1] * (self.B - len(tokens)))
            self.step_logits()
            lp = self.logprobs([-1] * self.B, top)
            found = sorted((-(live[b][1] + float(lp["top_logprobs"][b, j])), b, int(lp["top_ids"][b, j]))
                           for b in range(len(live)) for j in range(top))
            nxt = []
            for neg, b, tok in found:
                if len(nxt) == beams:
                    break
                if tok == eos_id:
                    done.append((live[b][0], -neg))
                else:
                    nxt.append((b, tok, -neg))
            done = sorted(done, key=lambda d: -d[1])[:beams]
            live = [(live[b][0] + [tok], s) for b, tok, s in nxt]
            if not live or step + 1 == max_new_tokens or (len(done) == beams and done[-1][1] >= live[0][1]):
                break
            parents = [b for b, _, _ in nxt]
            self.fork(parents + [-1] * (beams - len(parents)) + rest)
            tokens, at = [tok for _, tok, _ in nxt], at + 1
        return sorted(done + live, key=lambda d: -d[1])[:beams]

    def compact(self):
        """Move the pages in use to the front of the pool; returns how many there are."""
        self.kv.compact()
        return int(self.kv.counts[1])

    def release(self):
        self._logit_graph = None
        self._jobs = {}
        super().release()
        if hasattr(self, "kv"):
            del self.kv
        torch.cuda.empty_cache()
