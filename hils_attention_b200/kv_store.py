"""Paged K/V store for decode: the page is the chunk.

The reference's cache layer (utils/hils_cache_utils.py:9-76) re-allocates the whole cache with torch.cat on
every step (:61-62) and moves it to host memory beyond a length threshold (:19-23, :45-59); its serving
notes ask the serving engine for a page size of 64 (README.md:255,262), the chunk size.  This store keeps
that granularity: K and V live in one preallocated pool of pages of 64 tokens, a sequence owns a list of
pages (its page table), and growing a sequence by one token never copies anything - every 64 tokens it
takes one page from the free list.  Sequences of different lengths share one decode batch; the kernels
read the page table and the per-sequence lengths from device memory (ops.decode_step_paged).

Because a page is a chunk, the sparse branch reads each selected chunk as ONE page, and the sliding
window (whose left edge is snapped to a chunk boundary) walks whole pages: no kernel gathers rows across
a page boundary.  Inside a page the rows of one head are contiguous, (h_kv, 64, D): the chunk of one head
is a single 16 KB run (D = 128) where the token-major layout has 64 rows h_kv * D apart.  The pooled chunk keys and their prior bias - one row per completed chunk, 1/64 of the
store - are kept dense per sequence slot, since the selection streams all of them on every step.

Full pages are never written again, so several sequences may share them: `fork` gives a second sequence the pages of the
first (a reference count per page, only the unfinished last page is copied), `compact` moves the pages in use to the front of
the pool.  A step over a tree of drafted tokens (`begin_tree` .. `end_tree`) keeps the drafts beside the pages until it is
known which of them are accepted; only those are written.

Host-side bookkeeping (free list, tables, lengths) is plain Python and mirrors what sits on the device;
nothing here reads device memory back, so a decode step issues no synchronisation.
"""
from __future__ import annotations

from collections import Counter
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib, ops


class PagePool:
    """Free list of page ids and the number of sequences that hold each page.  Page 0 is reserved as the scratch page that
    inactive batch rows write to."""

    def __init__(self, num_pages: int):
        if num_pages < 2:
            raise ValueError("a pool needs at least two pages (page 0 is the scratch page)")
        self.num_pages = int(num_pages)
        self._free: List[int] = list(range(self.num_pages - 1, 0, -1))   # pop() hands out 1, 2, 3, ...
        self._refs: List[int] = [0] * self.num_pages

    @property
    def free(self) -> int:
        return len(self._free)

    def shuffle(self, seed: int) -> None:
        """Hand the free pages out in a random order from now on (what a pool looks like after many sequences came
        and went); used to measure with a sequence's pages scattered over the pool."""
        import random
        random.Random(seed).shuffle(self._free)

    def take(self, n: int = 1) -> List[int]:
        if n > len(self._free):
            raise MemoryError(f"paged store: {n} pages wanted, {len(self._free)} free of {self.num_pages - 1}")
        out = [self._free.pop() for _ in range(n)]
        for p in out:
            self._refs[p] = 1
        return out

    def share(self, pages: Sequence[int]) -> None:
        """One more sequence holds each of `pages`."""
        for p in pages:
            if not 0 < p < self.num_pages or self._refs[p] == 0:
                raise ValueError(f"page id {p} is not a page in use")
        for p in pages:
            self._refs[p] += 1

    def shared(self, page: int) -> bool:
        return self._refs[page] > 1

    def give(self, pages: Sequence[int]) -> None:
        """One sequence less holds each of `pages`; those nobody holds any more go back to the free list."""
        pages = list(pages)
        for p, n in Counter(pages).items():
            if not 0 < p < self.num_pages:
                raise ValueError(f"page id {p} is not a pool page")
            if self._refs[p] < n:
                raise ValueError(f"page id {p} is already free")
        for p in reversed(pages):
            self._refs[p] -= 1
            if self._refs[p] == 0:
                self._free.append(p)

    def compact(self) -> Tuple[List[int], List[int]]:
        """Renumber the pages in use to 1 .. n (n pages in use): returns the moved pages' old and new ids and rebuilds the
        free list.  The contents are the caller's to copy."""
        used = [p for p in range(1, self.num_pages) if self._refs[p]]
        n = len(used)
        src = [p for p in used if p > n]
        dst = [p for p in range(1, n + 1) if not self._refs[p]]
        for a, b in zip(src, dst):
            self._refs[a], self._refs[b] = 0, self._refs[a]
        self._free = list(range(self.num_pages - 1, n, -1))
        return src, dst


class PagedKVStore:
    """K/V pages, page tables, lengths and pooled chunk keys of up to `max_seqs` sequences and `num_layers` layers.

    Device tensors (all preallocated):
      k_pages, v_pages (num_layers, num_pages, h_kv, S, D)   the pool; one table serves every layer
      page_table       (max_seqs, max_pages) int32            page of chunk c of the sequence in slot b
      lens             (max_seqs) int32                       tokens the sequence in slot b holds
      lmk_k            (num_layers, max_seqs, max_pages, h_lmk, D)   pooled chunk keys
      prior_b          (num_layers, max_seqs, max_pages, h_q) fp32    prior bias of each chunk
    A decode batch is the slots [0, batch) with batch = 1 + the highest active slot; rows of inactive slots
    hold length 0 and point at the scratch page, so they cost one token of work and touch no sequence's data.
    """

    def __init__(self, num_pages: int, max_seqs: int, max_pages_per_seq: int, h_kv: int, head_dim: int, h_q: int,
                 h_lmk: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, device="cuda", num_layers: int = 1,
                 page_size: int = 64):
        if page_size != 64:
            raise ValueError("the page is the chunk of the decode kernels: 64 tokens")
        self.S = page_size
        self.num_layers, self.max_seqs, self.max_pages = int(num_layers), int(max_seqs), int(max_pages_per_seq)
        self.h_kv, self.h_q, self.D = int(h_kv), int(h_q), int(head_dim)
        self.h_lmk = int(h_lmk if h_lmk is not None else h_q)
        self.pool = PagePool(num_pages)
        dev = torch.device(device)
        self.dtype = dtype
        self.k_pages = torch.zeros((num_layers, num_pages, h_kv, self.S, head_dim), dtype=dtype, device=dev)
        dev = self.device = self.k_pages.device                     # with its index: "cuda" alone means another device later
        self.v_pages = torch.zeros_like(self.k_pages)
        self.page_table = torch.zeros((max_seqs, max_pages_per_seq), dtype=torch.int32, device=dev)   # 0 = scratch page
        self.lens = torch.zeros((max_seqs,), dtype=torch.int32, device=dev)
        self.lmk_k = torch.zeros((num_layers, max_seqs, max_pages_per_seq, self.h_lmk, head_dim), dtype=dtype, device=dev)
        self.prior_b = torch.zeros((num_layers, max_seqs, max_pages_per_seq, h_q), dtype=torch.float32, device=dev)
        self._active_dev = torch.zeros((max_seqs,), dtype=torch.int32, device=dev)
        # host mirrors
        self._tables: List[List[int]] = [[] for _ in range(max_seqs)]
        self._lens: List[int] = [0] * max_seqs
        self._active: List[bool] = [False] * max_seqs
        self._in_step = False
        self._tree = 0                                              # nodes per sequence of the drafted step in progress
        self._drafts: Optional[Tuple[torch.Tensor, ...]] = None     # k, v, lmk_q of the drafted tokens of every layer: views of
        self._draft_room: Optional[Tuple[torch.Tensor, ...]] = None  # room for max_seqs sequences of the widest tree so far
        self._paths: Optional[List[List[int]]] = None               # accepted nodes per slot, between accept_tree and end_tree
        self._scratch: Optional[torch.Tensor] = None                # of a drafted step, one for all layers
        self._captured: List[torch.Tensor] = []                     # what captured steps write to: kept as long as the store

    # ---- bookkeeping ---------------------------------------------------------------------------------
    @property
    def batch(self) -> int:
        """Rows of a decode batch: 1 + the highest active slot."""
        for b in range(self.max_seqs - 1, -1, -1):
            if self._active[b]:
                return b + 1
        return 0

    def active_slots(self) -> List[int]:
        return [b for b in range(self.max_seqs) if self._active[b]]

    def length(self, slot: int) -> int:
        return self._lens[slot]

    def pages_of(self, slot: int) -> List[int]:
        return list(self._tables[slot])

    def _set_table(self, slot: int, first_chunk: int, pages: Sequence[int]) -> None:
        if not pages:
            return
        t = torch.tensor(list(pages), dtype=torch.int32)
        self.page_table[slot, first_chunk:first_chunk + len(pages)].copy_(t, non_blocking=True)

    def allocate(self, n_tokens: int = 0) -> int:
        """Activate the lowest free slot for a sequence that already has `n_tokens` tokens (to be written with
        write_prefill); reserves the pages those tokens need.  Returns the slot."""
        if self._in_step:
            raise RuntimeError("allocate() between begin_step() and end_step()")
        n_pages = (n_tokens + self.S - 1) // self.S
        if n_pages > self.max_pages or n_tokens >= self.max_pages * self.S:
            raise ValueError(f"{n_tokens} tokens do not fit {self.max_pages} pages per sequence")
        try:
            slot = self._active.index(False)
        except ValueError:
            raise MemoryError(f"paged store: all {self.max_seqs} sequence slots are in use") from None
        pages = self.pool.take(n_pages)
        self._tables[slot] = pages
        self._lens[slot] = int(n_tokens)
        self._active[slot] = True
        self._set_table(slot, 0, pages)
        self.lens[slot:slot + 1].fill_(int(n_tokens))
        self._active_dev[slot:slot + 1].fill_(1)
        return slot

    def release(self, slot: int) -> None:
        """Return the sequence's pages to the pool; the slot's row goes back to the scratch page."""
        if self._in_step:
            raise RuntimeError("release() between begin_step() and end_step()")
        if not self._active[slot]:
            raise ValueError(f"slot {slot} is not active")
        n = len(self._tables[slot])
        self.pool.give(self._tables[slot])
        self._tables[slot] = []
        self._lens[slot] = 0
        self._active[slot] = False
        if n:
            self.page_table[slot, :n].zero_()
        self.lens[slot:slot + 1].zero_()
        self._active_dev[slot:slot + 1].zero_()

    def fork(self, slot: int, copies: int = 1) -> List[int]:
        """Start `copies` further sequences with the contents of `slot` (parallel samples, beams, a shared prompt); returns
        their slots.  Full pages are shared, the unfinished last page and the pooled chunk keys are copied."""
        if self._in_step:
            raise RuntimeError("fork() between begin_step() and end_step()")
        if not self._active[slot]:
            raise ValueError(f"slot {slot} is not active")
        if copies < 0:
            raise ValueError(f"{copies} copies")
        free = [b for b in range(self.max_seqs) if not self._active[b]][:copies]
        if len(free) < copies:
            raise MemoryError(f"paged store: {copies} sequence slots wanted, {len(free)} free")
        T = self._lens[slot]
        full, rem = T // self.S, T % self.S
        head = self._tables[slot][:full]
        new = self.pool.take(copies if rem else 0)
        if rem and new:
            self._copy_pages([self._tables[slot][full]] * copies, new)
        for i, b in enumerate(free):
            self.pool.share(head)
            self._tables[b] = head + new[i:i + 1]
            self._lens[b], self._active[b] = T, True
            self._set_table(b, 0, self._tables[b])
            self.lens[b:b + 1].fill_(T)
            self._active_dev[b:b + 1].fill_(1)
            if full:
                self.lmk_k[:, b, :full].copy_(self.lmk_k[:, slot, :full])
                self.prior_b[:, b, :full].copy_(self.prior_b[:, slot, :full])
        return free

    def compact(self) -> int:
        """Move the pages in use to the front of the pool (ids 1 .. pages in use): what lies behind is free, and a snapshot of
        the cache is one slice.  Returns the number of pages moved."""
        if self._in_step:
            raise RuntimeError("compact() between begin_step() and end_step()")
        src, dst = self.pool.compact()
        if src:
            self._copy_pages(src, dst)
            to = dict(zip(src, dst))
            for b in self.active_slots():
                table = [to.get(p, p) for p in self._tables[b]]
                if table != self._tables[b]:
                    self._tables[b] = table
                    self._set_table(b, 0, table)
        return len(src)

    def _copy_pages(self, src: Sequence[int], dst: Sequence[int]) -> None:
        ops.copy_pages(self.k_pages, self.v_pages, src, dst)

    # ---- contents ------------------------------------------------------------------------------------
    def write_prefill(self, slot: int, layer: int, k: torch.Tensor, v: torch.Tensor, lmk_k: Optional[torch.Tensor] = None,
                      prior_b: Optional[torch.Tensor] = None) -> None:
        """Store the prefill of one sequence: k, v (T, h_kv, D) with T = the length given to allocate(); lmk_k
        (T // 64, h_lmk, D) and prior_b (T // 64, h_q) of its complete chunks."""
        T = self._lens[slot]
        if k.shape != (T, self.h_kv, self.D) or v.shape != k.shape:
            raise ValueError(f"write_prefill: expected ({T}, {self.h_kv}, {self.D}), got {tuple(k.shape)} / {tuple(v.shape)}")
        pages = self._tables[slot]
        if any(self.pool.shared(p) for p in pages):
            raise RuntimeError(f"write_prefill: slot {slot} shares pages with another sequence")
        full, rem = T // self.S, T % self.S
        if full:
            ids = torch.tensor(pages[:full], dtype=torch.long, device=self.device)
            def paged(x):   # (full * S, h, D) -> (full, h, S, D)
                return x[:full * self.S].reshape(full, self.S, self.h_kv, self.D).transpose(1, 2).to(self.dtype)
            self.k_pages[layer].index_copy_(0, ids, paged(k))
            self.v_pages[layer].index_copy_(0, ids, paged(v))
        if rem:
            self.k_pages[layer, pages[full], :, :rem].copy_(k[full * self.S:].transpose(0, 1))
            self.v_pages[layer, pages[full], :, :rem].copy_(v[full * self.S:].transpose(0, 1))
        if lmk_k is not None and full:
            if lmk_k.shape[0] != full:
                raise ValueError(f"write_prefill: {full} complete chunks but {lmk_k.shape[0]} chunk keys")
            self.lmk_k[layer, slot, :full].copy_(lmk_k)
            if prior_b is not None:
                self.prior_b[layer, slot, :full].copy_(prior_b)

    def gather(self, slot: int, layer: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """Dense copies (T, h_kv, D) of a sequence's keys and values (tests, chunk-prefill against the history)."""
        T = self._lens[slot]
        n = (T + self.S - 1) // self.S
        ids = torch.tensor(self._tables[slot][:n], dtype=torch.long, device=self.device)
        k = self.k_pages[layer].index_select(0, ids).transpose(1, 2).reshape(n * self.S, self.h_kv, self.D)[:T]
        v = self.v_pages[layer].index_select(0, ids).transpose(1, 2).reshape(n * self.S, self.h_kv, self.D)[:T]
        return k, v

    # ---- the decode step -----------------------------------------------------------------------------
    def begin_step(self) -> int:
        """Make room for one more token in every active sequence (a sequence standing at a multiple of 64 tokens
        takes a page) and return max_len, the host-side bound of the lengths that the step call wants."""
        if self._in_step:
            raise RuntimeError("begin_step() twice without end_step()")
        self._reserve({b: 1 for b in self.active_slots()})
        self._in_step = True
        return max((self._lens[b] for b in range(self.max_seqs) if self._active[b]), default=0)

    def _reserve(self, more) -> None:
        """Take the pages that more[b] further tokens of the sequence in slot b need beyond those its table holds (some may
        already be reserved); all or nothing."""
        need = {b: (self._lens[b] + n + self.S - 1) // self.S for b, n in more.items()}
        for b, c in need.items():
            if c > self.max_pages:
                raise MemoryError(f"paged store: the sequence in slot {b} has reached {self.max_pages} pages")
        want = sum(max(0, c - len(self._tables[b])) for b, c in need.items())
        if want > self.pool.free:
            raise MemoryError(f"paged store: {want} pages wanted, {self.pool.free} free")
        for b, c in need.items():
            have = len(self._tables[b])
            if c > have:
                pg = self.pool.take(c - have)
                self._tables[b].extend(pg)
                self._set_table(b, have, pg)

    def step_args(self, layer: int):
        """(k_pages, v_pages, page_table, lens, lmk_k, prior_b) of one layer for the current batch."""
        n = self.batch
        return (self.k_pages[layer], self.v_pages[layer], self.page_table[:n], self.lens[:n], self.lmk_k[layer, :n],
                self.prior_b[layer, :n])

    def completing(self) -> List[int]:
        """Slots whose chunk is completed by the token of the current step (its pooled key is due after the step)."""
        return [b for b in range(self.max_seqs) if self._active[b] and (self._lens[b] + 1) % self.S == 0]

    def chunk_keys(self, layer: int, slots: Sequence[int]) -> torch.Tensor:
        """(n, 64, h_kv, D): the keys of the last chunk of each of `slots` (a token-major view of the pages)."""
        ids = torch.tensor([self._tables[b][self._lens[b] // self.S] for b in slots], dtype=torch.long, device=self.device)
        return self.k_pages[layer].index_select(0, ids).transpose(1, 2)

    def put_chunk_keys(self, layer: int, slots: Sequence[int], lmk_k: torch.Tensor, prior_b: Optional[torch.Tensor]) -> None:
        """Store the pooled key (n, h_lmk, D) and prior bias (n, h_q) of the chunk each of `slots` is completing."""
        rows = torch.tensor(list(slots), dtype=torch.long, device=self.device)
        cols = torch.tensor([self._lens[b] // self.S for b in slots], dtype=torch.long, device=self.device)
        self.lmk_k[layer].index_put_((rows, cols), lmk_k.to(self.dtype))
        if prior_b is not None:
            self.prior_b[layer].index_put_((rows, cols), prior_b.to(torch.float32))

    def end_step(self) -> None:
        """Every active sequence is one token longer (after all layers ran the step)."""
        if not self._in_step or self._tree:
            raise RuntimeError("end_step() without begin_step()")
        n = self.batch
        self.lens[:n].add_(self._active_dev[:n])
        for b in range(n):
            if self._active[b]:
                self._lens[b] += 1
        self._in_step = False

    # ---- a step over drafted trees -------------------------------------------------------------------
    def begin_tree(self, n: int) -> int:
        """Begin a step over trees of up to `n` drafted tokens per sequence (at most 64) and return max_len.  Every active
        sequence gets the pages for n more tokens; unused ones stay reserved for its next tokens.  The drafts' buffers are kept
        from step to step and only move when a tree is wider than all before it: begin one of the largest n (and end it with
        nothing accepted) before a step is captured into a graph.  A captured step replays a step of the same n and batch."""
        if self._in_step:
            raise RuntimeError("begin_tree() between begin_step() / begin_tree() and its end")
        if not 1 <= n <= 64:
            raise ValueError(f"a tree of {n} nodes (1 to 64)")
        self._reserve({b: n for b in self.active_slots()})
        heads = (self.h_kv, self.h_kv, self.h_q)
        room = self.num_layers * self.max_seqs * n * self.D
        if self._draft_room is None or self._draft_room[0].numel() < room * self.h_kv:
            self._retire(*(self._draft_room or ()))
            self._draft_room = tuple(torch.empty(room * h, dtype=self.dtype, device=self.device) for h in heads)
        shape = (self.num_layers, self.batch, n)
        self._drafts = tuple(t[:shape[0] * shape[1] * n * h * self.D].view(*shape, h, self.D) for t, h in zip(self._draft_room, heads))
        self._in_step, self._tree, self._paths = True, int(n), None
        return max((self._lens[b] for b in self.active_slots()), default=0)

    def draft(self, layer: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The places of the drafted tokens of one layer in the step in progress: k, v (batch, n, h_kv, D) and the landmark
        query (batch, n, h_q, D), which the pooled key of a chunk completed by an accepted token needs."""
        if not self._tree:
            raise RuntimeError("draft() without begin_tree()")
        return tuple(t[layer] for t in self._drafts)

    def step_bound(self, max_len: Optional[int] = None) -> int:
        """The max_len a drafted step is given: no sequence may be longer when it runs.  The longest of the present lengths, or
        the caller's bound; in a step that is being captured, whose replays follow the lengths on the device, all that a page
        table holds."""
        now, most = max((self._lens[b] for b in self.active_slots()), default=0), self.max_pages * self.S
        if max_len is None:
            return most if _lib.capturing(self.device) else now
        if not now <= max_len <= most:
            raise ValueError(f"max_len {max_len}: the longest sequence has {now} tokens and a page table holds {most}")
        return int(max_len)

    @property
    def scratch(self) -> Optional[torch.Tensor]:
        """Scratch of a drafted step.  The layers run one after the other and share it."""
        return self._scratch

    def keep_scratch(self, scratch: torch.Tensor) -> None:
        """The scratch a layer's step used, for the next one.  A captured step goes on writing to its scratch and to the drafts'
        places whenever it is replayed, so these stay allocated when larger ones follow."""
        if scratch is not self._scratch:
            if self._scratch is not None:
                self._retire(self._scratch)
            self._scratch = scratch
        if _lib.capturing(self.device):
            for t in (scratch, *self._draft_room):
                if all(t is not c for c in self._captured):
                    self._captured.append(t)

    @staticmethod
    def _retire(*buffers: torch.Tensor) -> None:
        """Before buffers are let go: steps may have used them on another stream than the one they were allocated on."""
        for t in buffers:
            if t.is_cuda:
                t.record_stream(torch.cuda.current_stream(t.device))

    def accept_tree(self, paths: Sequence[Sequence[int]]) -> None:
        """After all layers ran: the nodes to keep of every row of the batch, from the root of the accepted path on (node ids
        ascend along a path; empty: nothing accepted).  Their keys and values are written into the pages."""
        if not self._tree or self._paths is not None:
            raise RuntimeError("accept_tree() once per begin_tree()")
        paths = [[int(x) for x in p] for p in paths]
        if len(paths) != self.batch:
            raise ValueError(f"accept_tree: {len(paths)} paths for a batch of {self.batch}")
        for b, p in enumerate(paths):
            if any(not 0 <= x < self._tree for x in p) or any(x >= y for x, y in zip(p, p[1:])):
                raise ValueError(f"accept_tree: path {p} of slot {b} is not an ascending list of nodes below {self._tree}")
            if p and not self._active[b]:
                raise ValueError(f"accept_tree: slot {b} is not active")
        width = max((len(p) for p in paths), default=0)
        if width:
            t = torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32).to(self.device, non_blocking=True)
            self._commit_drafts(t)
        self._paths = paths

    def _commit_drafts(self, path: torch.Tensor) -> None:
        n = self.batch
        k, v, _ = self._drafts
        ops.commit_drafts(k, v, self.k_pages, self.v_pages, self.page_table[:n], self.lens[:n], path)

    def completed(self) -> Tuple[List[int], List[int]]:
        """Slots whose chunk the accepted tokens complete, and the node that is the chunk's last token (at most one chunk per
        sequence: a tree has at most 64 nodes)."""
        if self._paths is None:
            raise RuntimeError("completed() before accept_tree()")
        slots = [b for b, p in enumerate(self._paths) if self._lens[b] % self.S + len(p) >= self.S]
        return slots, [self._paths[b][self.S - 1 - self._lens[b] % self.S] for b in slots]

    def end_tree(self) -> None:
        """Every sequence is longer by its accepted path (after the chunks these tokens complete got their pooled keys)."""
        if self._paths is None:
            raise RuntimeError("end_tree() before accept_tree()")
        n = self.batch
        if n:
            self.lens[:n].add_(torch.tensor([len(p) for p in self._paths], dtype=torch.int32).to(self.device, non_blocking=True))
        for b, p in enumerate(self._paths):
            self._lens[b] += len(p)
        self._in_step, self._tree, self._paths = False, 0, None

    def bytes_held(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_pages, self.v_pages, self.lmk_k, self.prior_b,
                                                          self.page_table, self.lens))
