"""A KV cache in pages: sequences of different lengths that fork, share a prefix and are freed.

``KVCache`` (``kv_cache.py``) gives a batch one row range and one cursor, as the
reference does (``models/dreamzero/model.py:35-65``). Here every layer has a pool
``[2, P, R, H, D]`` of ``P`` pages of ``R`` rows, and each of ``batch`` sequences a list
of page numbers and a length of its own:

* ``append(layer, k, v)`` writes one chunk per sequence at its own end and does not
  move it; ``commit(n)`` does, once every layer has appended. Both as ``KVCache``: a
  step is one of the whole batch, ``n`` rows for every sequence. Lengths come to differ
  through ``free`` and ``fork``; ``SelfAttention`` then takes a rotary table per sequence.
* ``fork(src, dst)`` makes sequence ``dst`` a copy of ``src`` by sharing its pages: no
  rows move. The partly filled last page is copied when one of the two next writes
  to it (``kv_page_copy``, one launch for all layers). Row weights, where a cache tracks
  them, are copied at once.
* ``hold_prefix(seq)`` turns the history of one sequence into a prefix of the whole
  batch (several candidate futures of one episode): it is kept once, and attention
  computes it once for all sequences (``shared_prefix_attention``). Until then it
  takes pages in every sequence, for a step writes them all.
* ``free(seq)`` gives a sequence's pages back; ``compact()`` moves what is in use to
  the lowest page numbers.
* ``fp4=True`` holds the rows in 4 bits (``kv_page_append_fp4``): 68 bytes of a head's row
  of 128 where bf16 takes 256. ``dtype`` is then that of the rows written and of attention.
* ``track_weights=True`` has ``attend`` add up the softmax weight that each row of a
  sequence received (``paged_key_weights``; ``weights[layer]`` ``[batch, H, W * R]``), by which
  ``evict(keep, recent)`` brings every longer sequence down to ``keep`` rows: the last
  ``recent`` and the heaviest before them, each layer and head by its own weights. Rows carry
  their positions in their rotated keys: the caller goes on counting positions from where
  the sequence was, not from its new length. A prefix keeps all of its rows. A row receives
  weight from the steps after its own, nothing from the chunk that it was written with: let
  ``recent`` cover the last chunk at least. (After one chunk, all weights are 0, and the
  lowest rows would be kept.) ``weights`` are 4 bytes for each row that a table has room
  for, layer and head: ``max_rows`` bounds them.

Which page is whose is decided on the host, before anything is launched:
``reserve(n)`` finds pages for the next ``n`` rows of every sequence or raises
``RuntimeError("KV cache full: ...")`` with nothing changed. The kernels read page
numbers and lengths from ``block_table`` ``[batch, W]`` and ``cache_lens`` ``[batch]``,
int32 tensors on the device that are changed in place, so a graph captured once
(``runtime.CachedStepGraph``) follows them; a captured step cannot reserve, so pages
are reserved before it is replayed. A ``reserve`` that takes pages sends the whole
table, ``batch`` x ``W`` entries, with a copy that waits for what the stream holds (64 x
256 entries take about a millisecond of the host's time): ``max_rows`` keeps ``W`` small,
and one ``reserve`` of many rows ahead spares the steps after it.
"""

from __future__ import annotations

import heapq
from collections import Counter

import torch

from .. import ops


class PagedKVCache:
    def __init__(self, layers: int, batch: int, pages: int, page_rows: int, heads: int,
                 head_dim: int, device: torch.device | str, dtype: torch.dtype,
                 max_rows: int | None = None, fp4: bool = False,
                 track_weights: bool = False) -> None:
        """``max_rows``: rows a sequence may hold (default: all pages); it sets the width of
        ``block_table``, for which attention launches are planned."""
        if page_rows <= 0 or page_rows % 16 or page_rows > 1024:
            raise ValueError(f"page_rows must be a multiple of 16 up to 1024, got {page_rows}")
        if fp4 and (dtype not in (torch.bfloat16, torch.float16) or head_dim not in (64, 128, 256)):
            raise ValueError(f"a cache in 4 bits serves bf16 and f16 at head dims 64, 128 and 256, got "
                             f"{dtype} at {head_dim}")
        self.fp4, self.dtype, self.head_dim = fp4, dtype, head_dim
        shape = ((2, pages, heads, page_rows * (head_dim // 2 + head_dim // 32)) if fp4 else
                 (2, pages, page_rows, heads, head_dim))
        self.pools = [torch.zeros(shape, device=device, dtype=torch.uint8 if fp4 else dtype)
                      for _ in range(layers)]
        self.pages, self.page_rows, self.batch = pages, page_rows, batch
        self.width = pages if max_rows is None else -(-max_rows // page_rows)
        self.lengths = [0] * batch
        self.tables: list[list[int]] = [[] for _ in range(batch)]
        self.prefix: list[int] = []
        self.prefix_rows = 0
        self._users = Counter()  # page -> sequences (and the prefix) that hold it
        self._free = list(range(pages))  # heap: lowest numbers first
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((batch, self.width), -1, **i32)
        self.cache_lens = torch.zeros(batch, **i32)
        self.prefix_table = torch.full((self.width,), -1, **i32)
        self.prefix_len = torch.zeros(1, **i32)
        self.status = torch.zeros(1, **i32)
        # What the rows received: of every layer, a sequence's tail behind its length is 0.
        self.weights = (torch.zeros(layers, batch, heads, self.width * page_rows, device=device,
                                    dtype=torch.float32) if track_weights else None)

    def _copy_pages(self, src: list[int], dst: list[int]) -> None:
        pools = self.pools
        if self.fp4:  # a page's bytes, as rows of 16-bit elements, one for each head
            pools = [p.view(torch.bfloat16).unsqueeze(3) for p in pools]
        ops.kv_page_copy(pools, src, dst)

    # -- pages ---------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._users[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._users[page] -= 1
        if self._users[page] == 0:
            del self._users[page]
            heapq.heappush(self._free, page)

    def _push_tables(self, tables: list[list[int]] | None = None) -> None:
        """The host's tables (or these) to the device, in place. A list that was never this
        long keeps -1 (no page) behind its end."""
        rows = [t + [-1] * (self.width - len(t)) for t in tables or self.tables]
        self.block_table.copy_(torch.tensor(rows, dtype=torch.int32).view(self.batch, self.width))

    def _push_lengths(self) -> None:
        self.cache_lens.copy_(torch.tensor(self.lengths, dtype=torch.int32))

    def _missing(self, n: int) -> tuple[list[int], int]:
        """Sequences whose last page is shared and would be written by the next ``n`` rows,
        and how many pages those and the new rows need. Raises when there are too few."""
        shared, need = [], 0
        claimed = Counter()
        for b, (table, length) in enumerate(zip(self.tables, self.lengths)):
            if length + n > self.width * self.page_rows:
                raise RuntimeError(f"KV cache full: {length} + {n} > {self.width * self.page_rows}")
            need += max(0, -(-(length + n) // self.page_rows) - len(table))
            if n and length % self.page_rows:
                last = table[length // self.page_rows]
                # The last of a page's sharers to claim it may keep it.
                if self._users[last] - claimed[last] > 1:
                    claimed[last] += 1
                    shared.append(b)
                    need += 1
        if need > len(self._free):
            raise RuntimeError(f"KV cache full: {need} pages needed, {len(self._free)} of "
                               f"{self.pages} free")
        return shared, need

    def _outside_a_capture(self, what: str) -> None:
        """What the host decides a replay would not repeat."""
        if self.block_table.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"PagedKVCache.{what} belongs before a capture, not inside one")

    def reserve(self, n: int) -> None:
        """Pages for the next ``n`` rows of every sequence, none of them shared. Nothing
        changes when they are there already, or (``RuntimeError``) when there are too few."""
        if n < 0:
            raise ValueError(f"cannot reserve {n} rows")
        shared, need = self._missing(n)
        if need == 0:
            return
        self._outside_a_capture(f"reserve({n})")
        # Pages change hands once everything that can fail has been done.
        new = iter(heapq.nsmallest(need, self._free))
        tables = [list(t) for t in self.tables]
        src, dst = [], []
        for b in shared:
            at = self.lengths[b] // self.page_rows
            src.append(tables[b][at])
            tables[b][at] = next(new)
            dst.append(tables[b][at])
        for table, length in zip(tables, self.lengths):
            while len(table) * self.page_rows < length + n:
                table.append(next(new))
        if src:
            self._copy_pages(src, dst)
        self._push_tables(tables)
        for _ in range(need):
            self._take()
        for page in src:
            self._drop(page)  # (no page's last user: the last of its sharers keeps it)
        self.tables = tables

    _check_room = reserve

    # -- writing -------------------------------------------------------------
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Write one chunk's ``k``/``v`` ``[batch, n, H, D]`` for ``layer`` at each sequence's
        end (lengths unchanged)."""
        self.reserve(k.shape[1])
        write = ops.kv_page_append_fp4 if self.fp4 else ops.kv_page_append
        write(self.pools[layer], k, v, self.block_table, self.cache_lens, self.status)

    def commit(self, n: int) -> None:
        """Move every sequence's end once every layer has appended its chunk."""
        if n < 0:
            raise ValueError(f"cannot commit {n} rows")
        for table, length in zip(self.tables, self.lengths):
            if length + n > len(table) * self.page_rows:
                raise RuntimeError(f"commit of {n} rows behind {length}, but only "
                                   f"{len(table) * self.page_rows} are reserved: append first")
        self._advance(n)
        self.cache_lens.add_(n)

    # -- sequences -----------------------------------------------------------
    def fork(self, src: int, dst: int) -> None:
        """Sequence ``dst`` becomes a copy of ``src``, on the same pages."""
        if src == dst:
            return
        self._outside_a_capture("fork")
        table, length = list(self.tables[src]), self.lengths[src]
        table = table[:-(-length // self.page_rows)]  # reserved pages behind the end stay src's
        dropped = self.tables[dst]
        for page in table:
            self._users[page] += 1
        for page in dropped:
            self._drop(page)
        self.tables[dst], self.lengths[dst] = table, length
        self._push_tables()
        self._push_lengths()
        if self.weights is not None:
            self.weights[:, dst] = self.weights[:, src]

    def free(self, seq: int) -> None:
        """Give a sequence's pages back; it starts again from nothing (and the prefix)."""
        self._outside_a_capture("free")
        for page in self.tables[seq]:
            self._drop(page)
        self.tables[seq], self.lengths[seq] = [], 0
        self._push_tables()
        self._push_lengths()
        if self.weights is not None:
            self.weights[:, seq] = 0

    def hold_prefix(self, seq: int) -> None:
        """The history of ``seq`` (behind a prefix held already, whose last page has to be
        full) becomes the prefix of every sequence; the sequences' own rows are freed."""
        self._outside_a_capture("hold_prefix")
        if self.prefix_rows % self.page_rows:
            raise RuntimeError(f"a prefix of {self.prefix_rows} rows ends inside a page: nothing "
                               "can follow it in the prefix")
        length = self.lengths[seq]
        table = self.tables[seq][:-(-length // self.page_rows)]
        if self.prefix_rows + length > self.width * self.page_rows:
            raise RuntimeError(f"KV cache full: {self.prefix_rows} + {length} > "
                               f"{self.width * self.page_rows}")
        for page in table:
            self._users[page] += 1
        self.prefix += table
        self.prefix_rows += length
        for b in range(self.batch):
            for page in self.tables[b]:
                self._drop(page)
            self.tables[b], self.lengths[b] = [], 0
        self._push_prefix()
        self._push_tables()
        self._push_lengths()
        if self.weights is not None:
            self.weights.zero_()

    def evict(self, keep: int, recent: int = 0, seq: int | None = None) -> int:
        """Bring every sequence (or ``seq`` alone) that holds more than ``keep`` rows down to
        ``keep``: its last ``recent`` rows (at most ``keep``) and the heaviest before them, in
        their order, each layer and head by its own weights. Returns how many sequences that
        was. Between steps only: rows that are appended but not committed are nobody's yet, and
        are lost. Rows stay where their pages are the sequence's alone; the others' go to new pages
        (``RuntimeError`` with nothing changed when there are too few: all sequences' new pages
        are found before any old one is free, so on a full pool that sequences share, evict
        them one by one, which frees pages for the next and leaves the last sharer in place)."""
        if self.weights is None:
            raise RuntimeError("evict needs PagedKVCache(track_weights=True)")
        if keep < 0 or recent < 0:
            raise ValueError(f"cannot keep {keep} rows, {recent} of them the last")
        self._outside_a_capture("evict")
        which = range(self.batch) if seq is None else [range(self.batch)[seq]]
        long = [b for b in which if self.lengths[b] > keep]
        if not long:
            return 0
        count = -(-keep // self.page_rows)
        need = sum(self._users[p] > 1 for b in long for p in self.tables[b][:count])
        if need > len(self._free):
            raise RuntimeError(f"KV cache full: {need} pages needed, {len(self._free)} of "
                               f"{self.pages} free")
        new = iter(heapq.nsmallest(need, self._free))
        tables = [list(t) for t in self.tables]
        for b in long:
            tables[b] = [next(new) if self._users[p] > 1 else p for p in tables[b][:count]]
        to = self.block_table
        if need:
            to = torch.tensor([t + [-1] * (self.width - len(t)) for t in tables], dtype=torch.int32)
            to = to.to(self.block_table.device)
        # Every layer's rows are chosen before any layer's move: what can fail comes first.
        at = slice(which[0], which[-1] + 1)
        layers = [weights[at] for weights in self.weights]
        picked = [ops.kv_keep_rows(weights, self.cache_lens[at], keep, recent) for weights in layers]
        for pool, weights, rows in zip(self.pools, layers, picked):
            ops.kv_page_gather(pool, self.block_table[at], rows, to[at], weights, self.head_dim)
        for _ in range(need):
            self._take()
        for b in long:
            kept = set(tables[b])
            for page in self.tables[b]:
                if page not in kept:
                    self._drop(page)
            self.lengths[b] = keep
        self.tables = tables
        self._push_tables()
        self._push_lengths()
        return len(long)

    def _push_prefix(self) -> None:
        row = self.prefix + [-1] * (self.width - len(self.prefix))
        self.prefix_table.copy_(torch.tensor(row, dtype=torch.int32))
        self.prefix_len.copy_(torch.tensor([self.prefix_rows], dtype=torch.int32))

    def compact(self) -> int:
        """Move the pages in use to the lowest numbers, in every layer; returns how many
        moved. What is in use and what is free never overlap, so one pass does it."""
        self._outside_a_capture("compact")
        live = sorted(self._users)
        n = len(live)
        src = [p for p in live if p >= n]
        held = set(live)
        dst = [p for p in range(n) if p not in held]
        if src:
            self._copy_pages(src, dst)
            new = dict(zip(src, dst))
            self.tables = [[new.get(p, p) for p in t] for t in self.tables]
            self.prefix = [new.get(p, p) for p in self.prefix]
            self._users = Counter({new.get(p, p): c for p, c in self._users.items()})
            self._free = list(range(n, self.pages))
            self._push_tables()
            self._push_prefix()
        return len(src)

    def reset(self) -> None:
        self._outside_a_capture("reset")
        self.tables = [[] for _ in range(self.batch)]
        self.lengths = [0] * self.batch
        self.prefix, self.prefix_rows = [], 0
        self._users.clear()
        self._free = list(range(self.pages))
        self._push_tables()
        self._push_lengths()
        self._push_prefix()
        self.status.zero_()
        if self.weights is not None:
            self.weights.zero_()

    # -- attention -----------------------------------------------------------
    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               block_boundaries: torch.Tensor | None = None, softmax_scale: float | None = None,
               causal: bool = False) -> torch.Tensor:
        """Attention of each sequence's ``q`` over the prefix, its cached rows and its ``k``/``v``."""
        kw = dict(pages=self.pools[layer], block_table=self.block_table,
                  cache_lens=self.cache_lens, block_boundaries=block_boundaries,
                  softmax_scale=softmax_scale, causal=causal)
        attention = ops.paged_attention_fp4 if self.fp4 else ops.paged_attention
        if self.prefix:
            attention = ops.shared_prefix_attention_fp4 if self.fp4 else ops.shared_prefix_attention
            kw.update(prefix_table=self.prefix_table, prefix_len=self.prefix_len)
        if self.weights is None:
            return attention(q, k, v, **kw)
        out, lse = attention(q, k, v, return_lse=True, **kw)
        ops.paged_key_weights(q, lse, self.weights[layer], pages=self.pools[layer],
                              block_table=self.block_table, cache_lens=self.cache_lens,
                              softmax_scale=softmax_scale)
        return out

    def overflowed(self) -> bool:
        """Whether a captured append found a row without a page (synchronises)."""
        return bool(int(self.status.item()))

    # -- what runtime.CachedStepGraph keeps of a cache --------------------------
    @property
    def cursor(self) -> torch.Tensor:
        return self.cache_lens

    def _host_state(self):
        return list(self.lengths)

    def _captured_form(self) -> bool:
        return bool(self.prefix)  # which operator attend() calls

    def _restore_host(self, state) -> None:
        self.lengths = list(state)

    def _device_state(self) -> list[torch.Tensor]:
        """What a step changes on the device and a warm-up has to put back."""
        kept = [self.cache_lens, self.status]
        return kept if self.weights is None else [*kept, self.weights]

    def _advance(self, n: int) -> None:
        self.lengths = [length + n for length in self.lengths]
