"""Paged KV pool, request page tables and per-tick batch metadata on the MI355X path.

Drop-in for the reference's src/helios/runtime/qwen3/paged_cache.py: the classes,
methods, arguments, attribute names, metadata tensors (names, dtypes, shapes), page
allocation order and exception types are the ones its decoder uses (layers.py:161-164,
model.py:30-110, decode.py:133-290, prefix_cache.py:227-290), so that decoder runs on
this module unchanged. How they are computed is this module's own design:

* One device allocation holds every layer's K and V pages,
  ``[2, n_layers, num_pages, page_size, n_kv_heads, head_dim]``; ``keys[l]`` and
  ``values[l]`` are contiguous views of it, so a page id names the same page in every
  layer and the pool costs one allocation however many layers it has.
* Free page ids live on a LIFO stack in a numpy array. A page handle gives its id back
  when the last holder (a request, a prefix-cache snapshot) drops it.
* A tick's metadata comes from one kernel launch (``hx_tick_metadata``, the default on a
  ROCm pool) fed three int32 values per sequence, or, with ``device_metadata=False``,
  from vectorised numpy on the host. Every host-built tensor is uploaded only when its
  values change.
* ``attend`` runs the HIP kernels: KV append and paged varlen attention, with one work
  plan per tick reused by every layer. There is no CPU attention branch; on a CPU pool
  only the bookkeeping works.
* Extensions, all off the reference's call path: ``restore_blocks(copy=...,
  private_tail=...)`` (copying restores on the page-copy kernel), ``attend_projected``
  (q/k RMSNorm + RoPE fused with the append), the shared-prefix cascade, and attention
  over selected blocks (``KVPagePool(block_size=...)``, ``BlockSparse``).
"""

from __future__ import annotations

from bisect import bisect_left
from collections.abc import Sequence
from dataclasses import dataclass
from itertools import accumulate

import numpy as np
import torch

from helios_amd import ops
from helios_amd.config import Qwen3Config

_NUMPY_DTYPE = {torch.int32: np.int32, torch.int64: np.int64, torch.float32: np.float32}


def _page_count(tokens: int, page_size: int) -> int:
    """Pages that hold ``tokens`` tokens."""
    return -(-tokens // page_size)


# --------------------------------------------------------------------------- pool
class KVPage:
    """Handle of one pool page (paged_cache.py:14-20).

    Pages are shared by identity: a request's page table and every prefix-cache
    snapshot of it hold the same handle. The id goes back on the pool's free stack when
    the last holder drops the handle."""

    __slots__ = ("__weakref__", "index", "pool")

    def __init__(self, pool: KVPagePool, index: int) -> None:
        self.pool = pool
        self.index = index

    def __del__(self) -> None:
        pool = getattr(self, "pool", None)
        if pool is not None:
            pool._push_free(self.index)

    def __repr__(self) -> str:
        return f"KVPage({self.index})"


@dataclass(frozen=True)
class PagedKVBlockSnapshot:
    """Whole pages of a request, held by a prefix cache (paged_cache.py:23-27)."""

    length: int
    pages: tuple[KVPage, ...]
    memory_bytes: int


class KVPagePool:
    """K and V pages of every layer plus the free-page stack (paged_cache.py:30-86).

    ``keys[l]`` / ``values[l]`` are ``[num_pages, page_size, n_kv_heads, head_dim]``
    contiguous views of ``storage``. On a fresh pool ids are handed out from 0 upwards;
    the id released last is the next one handed out.

    With ``block_size`` (a power of two from 16 to 1024 that divides the page) the pool
    also keeps each block's key bounds, ``bounds[l]`` ``[num_pages, page_size //
    block_size, n_kv_heads, 2, head_dim]`` (2 / block_size of the keys' memory): every append
    of a batch brings them up to date, so that ``BlockSparse`` batches can select by them.
    Keys written into the pool by other means need ``PagedKVCache.refresh_bounds``."""

    def __init__(self, config: Qwen3Config, num_pages: int, *, device: torch.device,
                 page_size: int = 256, block_size: int | None = None) -> None:
        if num_pages < 1:
            raise ValueError(f"a KV page pool needs at least one page, not {num_pages}")
        if page_size < 1 or page_size % 256 != 0:
            raise ValueError(f"page_size must be a positive multiple of 256, not {page_size}")
        if block_size is not None:
            if not 16 <= block_size <= 1024 or block_size & (block_size - 1) or page_size % block_size:
                raise ValueError(
                    f"block_size must be a power of two from 16 to 1024 that divides the page, not {block_size}")
            if config.dtype not in (torch.bfloat16, torch.float16) or config.head_dim % 8 or config.head_dim > 256:
                raise ValueError("key bounds need bfloat16 or float16 heads of a multiple of 8 up to 256 elements")
        self.config = config
        self.num_pages = int(num_pages)
        self.page_size = int(page_size)
        self.device = torch.device(device)
        self.storage = torch.empty(
            (2, config.n_layers, self.num_pages, self.page_size, config.n_kv_heads, config.head_dim),
            dtype=config.dtype, device=self.device,
        )
        self.keys = tuple(self.storage[0].unbind(0))
        self.values = tuple(self.storage[1].unbind(0))
        self.block_size = block_size
        self.bounds: tuple[torch.Tensor, ...] | None = None
        if block_size is not None:
            self.bounds = tuple(torch.zeros(
                (config.n_layers, self.num_pages, self.page_size // block_size, config.n_kv_heads, 2, config.head_dim),
                dtype=config.dtype, device=self.device).unbind(0))
        # _stack[:_top] holds the free ids; _stack[_top - 1] is handed out next. Released
        # ids wait in _released (in release order) until the next acquire or free-page
        # count moves them onto the stack: a release can run inside the garbage
        # collector at any allocation, also in the middle of acquire, so it never
        # touches the stack itself.
        self._stack = np.arange(self.num_pages - 1, -1, -1, dtype=np.int64)
        self._top = self.num_pages
        self._released: list[int] = []

    @property
    def bytes_per_token(self) -> int:
        """K and V bytes of one token over all layers."""
        per_layer_row = self.config.n_kv_heads * self.config.head_dim * self.storage.element_size()
        return 2 * self.config.n_layers * per_layer_row

    @property
    def bytes_per_page(self) -> int:
        return self.page_size * self.bytes_per_token

    @property
    def free_pages(self) -> int:
        self._drain_released()
        return self._top

    def acquire(self, count: int) -> list[KVPage]:
        """``count`` fresh page handles, popped off the free stack."""
        if count < 0:
            raise ValueError(f"cannot acquire a negative number of pages ({count})")
        self._drain_released()
        if count > self._top:
            raise RuntimeError(f"KV page pool exhausted: {count} pages asked for, {self._top} free")
        top = self._top
        ids = self._stack[top - count:top][::-1].tolist()
        self._top = top - count
        return [KVPage(self, i) for i in ids]

    def _push_free(self, index: int) -> None:
        """Release of a page id (from ``KVPage.__del__``, possibly inside the garbage
        collector): queued, never written to the stack directly."""
        self._released.append(index)

    def _drain_released(self) -> None:
        """Move queued releases onto the free stack, oldest first (so the id released
        last is handed out first). Nothing here allocates a collectable object, so no
        release can run in between."""
        released = self._released
        n = len(released)
        while n:
            for k in range(n):
                self._stack[self._top] = released[k]
                self._top += 1
            del released[:n]
            n = len(released)

    def copy_pages(self, src_pages: Sequence[int], dst_pages: Sequence[int]) -> None:
        """Bit-copy pages for every layer, keys, values and any key bounds, on the page-copy
        kernel."""
        ops.kv_copy_pages(self.keys, self.values, src_pages, dst_pages)
        if self.bounds is not None:
            ops.kv_copy_pages(self.bounds, None, src_pages, dst_pages)


# ----------------------------------------------------------------- request cache
class PagedKVCache:
    """One request's page table, committed length and capacity (paged_cache.py:89-174).

    ``pages[i]`` holds tokens ``[i * page_size, (i + 1) * page_size)``. Between a batch's
    ``prepare`` / ``prepare_packed`` and its ``advance`` / ``advance_packed`` an append is
    in flight (``_pending_tokens``): the pages already cover the new tokens, ``length``
    does not count them yet."""

    batch_size = 1

    def __init__(self, pool: KVPagePool, capacity: int) -> None:
        limit = pool.config.context_length
        if not 1 <= capacity <= limit:
            raise ValueError(f"KV-cache capacity {capacity} is outside 1..{limit:,} tokens")
        self.pool, self.capacity = pool, capacity
        self.length = 0
        self.pages: list[KVPage] = []
        self._pending_tokens: int | None = None  # tokens of the append in flight

    @property
    def memory_bytes_per_token(self) -> int:
        """K and V bytes of one token over all layers (the pool's figure)."""
        return self.pool.bytes_per_token

    # A single request has one slot, so its per-slot figure is the same.
    memory_bytes_per_slot_token = memory_bytes_per_token

    @staticmethod
    def _check_slot(slot: int) -> None:
        if slot != 0:
            raise ValueError(f"a single-request paged cache has slot 0 only, not {slot}")

    def slot_length(self, slot: int) -> int:
        self._check_slot(slot)
        return self.length

    def snapshot_block_slot(self, slot: int, start: int, end: int) -> PagedKVBlockSnapshot:
        """The pages of tokens [start, end): whole pages of committed tokens only."""
        self._check_slot(slot)
        size = self.pool.page_size
        whole = start % size == 0 and end % size == 0
        if not (whole and 0 <= start < end <= self.length):
            raise ValueError(
                f"a paged snapshot covers whole pages of the {self.length} committed tokens; "
                f"[{start}, {end}) does not")
        first, stop = start // size, end // size
        pages = tuple(self.pages[first:stop])
        if len(pages) != stop - first:
            raise RuntimeError(f"page table holds {len(self.pages)} pages, the snapshot needs {stop}")
        return PagedKVBlockSnapshot(length=end - start, pages=pages,
                                    memory_bytes=len(pages) * self.pool.bytes_per_page)

    def snapshot_block(self, start: int, end: int) -> PagedKVBlockSnapshot:
        return self.snapshot_block_slot(0, start, end)

    def restore_blocks(
        self, blocks: Sequence[PagedKVBlockSnapshot], *, copy: bool = False,
        private_tail: bool = False,
    ) -> None:
        """Adopt snapshot pages into this empty cache.

        By default the pages are shared, zero-copy (paged_cache.py:142-163). ``copy=True``
        bit-copies them into fresh private pages for every layer, K and V (the copying
        restore of cache.py:131-147, at page granularity). ``private_tail=True`` shares
        every page but the last and copies that one (copy-on-write), so the request may
        ``truncate`` into it and write it again: a prompt the prefix cache covers
        completely then recomputes only its last token for its first logits, where the
        reference drops the whole last block and recomputes it (decode.py:173-174)."""
        if self.pages or self.length or self._pending_tokens is not None:
            raise RuntimeError("restore_blocks needs an empty request cache")
        size = self.pool.page_size
        pages: list[KVPage] = []
        for block in blocks:
            whole = block.length >= 1 and block.length == len(block.pages) * size
            if not whole or any(page.pool is not self.pool for page in block.pages):
                raise ValueError("a restored block must be whole pages of this cache's pool")
            pages.extend(block.pages)
        if len(pages) * size > self.capacity:
            raise ValueError(
                f"restored blocks hold {len(pages) * size} tokens, above the capacity {self.capacity}")
        if pages and copy:
            fresh = self.pool.acquire(len(pages))
            self.pool.copy_pages([p.index for p in pages], [p.index for p in fresh])
            pages = fresh
        elif pages and private_tail:
            tail = self.pool.acquire(1)
            self.pool.copy_pages([pages[-1].index], [tail[0].index])
            pages[-1:] = tail
        self.pages = pages
        self.length = len(pages) * size

    def truncate(self, length: int) -> None:
        """Forget tokens from ``length`` on; pages past the new length are dropped."""
        if self._pending_tokens is not None or not 0 <= length <= self.length:
            raise ValueError(
                f"cannot truncate to {length}: {self.length} tokens committed"
                + (", an append is in flight" if self._pending_tokens is not None else ""))
        del self.pages[_page_count(length, self.pool.page_size):]
        self.length = length

    def refresh_bounds(self) -> None:
        """Key bounds of all committed tokens from the pool's keys, every layer: for keys that
        came into the pool otherwise than by a batch's append."""
        pool = self.pool
        if pool.bounds is None:
            raise RuntimeError("the pool keeps no key bounds; create it with block_size")
        if self._pending_tokens is not None:
            raise RuntimeError("refresh_bounds needs the append in flight to be committed")
        if not self.length:
            return
        table = torch.tensor([[page.index for page in self.pages]], dtype=torch.int32, device=pool.device)
        ends = torch.tensor([0, self.length], dtype=torch.int32, device=pool.device)
        for keys, bounds in zip(pool.keys, pool.bounds):
            ops.kv_block_bounds(keys, bounds, table, ends, ends[1:], max_q=self.length)

    def close(self) -> None:
        self.pages = []
        self.length = 0
        self._pending_tokens = None


# ------------------------------------------------------------- tick metadata
class _HostTick:
    """The metadata of one tick on the host, vectorised over rows (numpy).

    From each sequence's committed length, tokens this tick, logit rows and page ids:
    ``cu_seq_q``, ``cu_seq_k``, ``seqused_k`` (int32), the padded ``block_table``
    (int32), and per packed row its ``positions`` and ``write_slots`` (int64), plus the
    ``logit_indices`` of each sequence's trailing rows."""

    def __init__(self, lengths: list[int], counts: list[int], tails: list[int] | None,
                 tables: list[list[int]], width: int, page_size: int) -> None:
        batch = len(counts)
        start = np.asarray(lengths, dtype=np.int64)
        count = np.asarray(counts, dtype=np.int64)
        end = start + count
        self.block_table = np.zeros((batch, width), dtype=np.int32)
        for b, ids in enumerate(tables):
            self.block_table[b, :len(ids)] = ids
        self.cu_seq_q = np.zeros(batch + 1, dtype=np.int32)
        np.cumsum(count, out=self.cu_seq_q[1:])
        self.cu_seq_k = np.zeros(batch + 1, dtype=np.int32)
        np.cumsum(end, out=self.cu_seq_k[1:])
        self.seqused_k = end.astype(np.int32)
        owner = np.repeat(np.arange(batch), count)               # sequence of every row
        first_row = self.cu_seq_q[:-1].astype(np.int64)[owner]
        self.positions = start[owner] + np.arange(owner.size, dtype=np.int64) - first_row
        page = self.block_table[owner, self.positions // page_size].astype(np.int64)
        self.write_slots = page * page_size + self.positions % page_size
        self.logit_indices = None
        if tails is not None:
            tail = np.asarray(tails, dtype=np.int64)
            holder = np.repeat(np.arange(batch), tail)
            rank = np.arange(holder.size, dtype=np.int64) - np.repeat(np.cumsum(tail) - tail, tail)
            self.logit_indices = self.cu_seq_q[1:].astype(np.int64)[holder] - tail[holder] + rank
        self.max_q = int(count.max())
        self.max_k = int(end.max())
        self.ends = end.tolist()


def _pinned(shape, dtype: torch.dtype) -> tuple[torch.Tensor, np.ndarray]:
    """A zeroed page-locked host tensor from torch's caching host allocator and its numpy
    view. A non-blocking copy from it is recorded on the stream that runs the copy, and the
    allocator hands the block out again only once that copy has run, so the host never
    waits before rewriting staging memory."""
    t = torch.zeros(shape, dtype=dtype, pin_memory=True)
    return t, t.numpy()


class _DeviceTickMetadata:
    """Staging and device buffers for ``ops.tick_metadata``.

    Device buffers are sized for the largest batch and the most rows seen so far; a tick
    gets views of them, so a batch object reused with other request caches (as the
    reference's decoder does, decode.py:235-241) needs no new allocation. Each tick's
    host values go to fresh pinned staging (``_pinned``) and cross with non-blocking
    copies: building a tick never waits for the device."""

    def __init__(self, device: torch.device) -> None:
        self.device = device
        self._cap = 0
        self._rows = 0
        self.block_table: torch.Tensor | None = None
        self.write_slots = self.positions = self.logit_indices = None

    def _ensure(self, batch: int, rows: int) -> None:
        if batch > self._cap:
            cap = max(batch, 2 * self._cap, 8)
            self._seq = torch.empty(3 * cap, dtype=torch.int32, device=self.device)
            self._cu_q = torch.empty(cap + 1, dtype=torch.int32, device=self.device)
            self._cu_k = torch.empty(cap + 1, dtype=torch.int32, device=self.device)
            self._used = torch.empty(cap, dtype=torch.int32, device=self.device)
            self._cap = cap
        if rows > self._rows:
            cap = max(rows, 2 * self._rows, 256)
            self.write_slots = torch.empty(cap, dtype=torch.int64, device=self.device)
            self.positions = torch.empty(cap, dtype=torch.int64, device=self.device)
            self.logit_indices = torch.empty(cap, dtype=torch.int64, device=self.device)
            self._rows = cap

    def upload_block_table(self, tables: list[list[int]], width: int) -> torch.Tensor:
        shape = (len(tables), width)
        if self.block_table is None or tuple(self.block_table.shape) != shape:
            self.block_table = torch.empty(shape, dtype=torch.int32, device=self.device)
        staged, host = _pinned(shape, torch.int32)
        for row, ids in enumerate(tables):
            host[row, :len(ids)] = ids
        self.block_table.copy_(staged, non_blocking=True)
        return self.block_table

    def build(self, lengths: list[int], counts: list[int], tails: list[int] | None,
              page_size: int) -> dict[str, torch.Tensor]:
        """Upload (lengths, counts, logit rows), launch the metadata kernel and return
        views of this tick's tensors."""
        batch = len(counts)
        total = sum(counts)
        n_logits = sum(tails) if tails is not None else 0
        self._ensure(batch, max(total, n_logits, 1))
        staged, host = _pinned(3 * batch, torch.int32)
        host[:batch] = lengths
        host[batch:2 * batch] = counts
        if tails is not None:
            host[2 * batch:3 * batch] = tails
        seq = self._seq[:3 * batch]
        seq.copy_(staged, non_blocking=True)
        views = self.last = {
            "seq": seq,
            "cu_seq_q": self._cu_q[:batch + 1],
            "cu_seq_k": self._cu_k[:batch + 1],
            "seqused_k": self._used[:batch],
            "write_slots": self.write_slots[:total],
            "positions": self.positions[:total],
            "logit_indices": self.logit_indices[:n_logits] if n_logits else None,
        }
        ops.tick_metadata(
            seq, self.block_table, page_size, total_q=total,
            cu_seq_q=views["cu_seq_q"], cu_seq_k=views["cu_seq_k"], seqused_k=views["seqused_k"],
            write_slots=self.write_slots, positions=self.positions,
            logit_indices=self.logit_indices if n_logits else None, n_logits=n_logits,
        )
        return views


# ------------------------------------------------------------ prefix cascade
class _PrefixCascade:
    """Shared-prefix split of one tick's attention.

    Decode rows whose page tables start with the same pages (prefix-cache hits restored
    by ``restore_blocks``) would each stream those pages again. A family of such rows
    shares, row by row, s_r leading pages with a reference row (the one with most pages).
    Its shared range is cut into at most ``MAX_LEVELS`` levels [b_{j-1}, b_j); level j
    holds every member with s_r >= b_j and attends once to those pages as one multi-row
    sequence with no causal limit (virtual batch A: the chunk kernel's MFMA path, split
    over key tiles). A member then attends only to its pages from B_r = the largest
    boundary <= s_r (batch B: the tick's sequences with tables shifted by B_r pages), and
    its results are merged by log-sum-exp (``ops.attn_merge``, one pass over all levels), which
    gives the attention over all of its keys. Attention needs no absolute key position
    (RoPE is already applied), so a shifted table is an ordinary shorter sequence.

    The boundaries minimise a cost in microseconds per layer: pages a member still reads
    itself (s_r - B_r, 1 MiB of K+V each at the decode kernel's rate), the padded MFMA
    work of each level (64-row blocks) and a fixed cost per level (its merge pass).
    """

    MIN_GROUP = 2
    MAX_LEVELS = 4
    US_PER_PAGE_READ = 0.19       # one page of K+V (1 MiB) at about 5.5 TB/s
    US_PER_BLOCK_PAGE = 0.54      # 64 rows x 32 heads x 256 keys x d=128 at about 500 TFLOP/s
    US_PER_LEVEL = 2.0            # one more part per member in the merge pass, level set-up

    def __init__(self, plan_a, plan_b, rows_a, merge, members, bt_a, bt_b):
        self.plan_a, self.plan_b = plan_a, plan_b
        self.rows_a = rows_a  # packed row of every batch-A query row, level by level
        self.merge = merge    # (merged packed rows, part_start, part_idx) for attn_merge
        self.members = members  # (sequence of each merged row, member index of each sequence)
        self.bt_a, self.bt_b = bt_a, bt_b

    @classmethod
    def _boundaries(cls, shared: list[int]) -> list[int]:
        """Level boundaries b_1 < ... < b_k (k <= MAX_LEVELS) for members sharing
        ``shared`` leading pages each, by dynamic programming over the distinct values."""
        cand = sorted({s for s in shared if s > 0})
        if not cand:
            return []
        # Sorted shares with prefix sums: below(x) = #{s < x}, total(x) = sum{s < x}, so
        # every count and page sum below is O(log n) (exact integers, as a direct sum).
        ordered = sorted(shared)
        prefix = [0, *accumulate(ordered)]

        def below(x):
            return bisect_left(ordered, x)

        def count(b):
            return len(ordered) - below(b)

        def extra(lo, hi, b):  # pages read by members with lo <= s < hi beyond boundary b
            i, k = below(lo), below(hi)
            return prefix[k] - prefix[i] - b * (k - i)

        def level_cost(prev, b):
            c = count(b)
            if c < cls.MIN_GROUP:
                return None
            blocks = -(-c // 64)
            return blocks * (b - prev) * cls.US_PER_BLOCK_PAGE + cls.US_PER_LEVEL

        inf = float("inf")
        top = max(shared) + 1
        # best[j][i]: cost of members with s < cand[i] plus levels ending at cand[i], j levels
        best = [[inf] * len(cand) for _ in range(cls.MAX_LEVELS)]
        back = [[-1] * len(cand) for _ in range(cls.MAX_LEVELS)]
        for i, b in enumerate(cand):
            lc = level_cost(0, b)
            if lc is not None:
                best[0][i] = extra(0, b, 0) * cls.US_PER_PAGE_READ + lc
        for j in range(1, cls.MAX_LEVELS):
            for i, b in enumerate(cand):
                for h in range(i):
                    if best[j - 1][h] == inf:
                        continue
                    lc = level_cost(cand[h], b)
                    if lc is None:
                        continue
                    cost = best[j - 1][h] + extra(cand[h], b, cand[h]) * cls.US_PER_PAGE_READ + lc
                    if cost < best[j][i]:
                        best[j][i], back[j][i] = cost, h
        none = extra(0, top, 0) * cls.US_PER_PAGE_READ
        choice, pick = none, None
        for j in range(cls.MAX_LEVELS):
            for i, b in enumerate(cand):
                if best[j][i] == inf:
                    continue
                cost = best[j][i] + extra(b, top, b) * cls.US_PER_PAGE_READ
                if cost < choice:
                    choice, pick = cost, (j, i)
        if pick is None:
            return []
        j, i = pick
        out = []
        while i >= 0 and j >= 0:
            out.append(cand[i])
            i, j = back[j][i], j - 1
        return sorted(out)

    @classmethod
    def levels(cls, batch: "PagedBatchCache", q_lens: list[int]) -> list[tuple[int, int, int, list[int]]]:
        """(reference row, first page, end page, member rows) of every level."""
        ps = batch.pool.page_size
        caches = batch.caches
        by_first: dict[int, list[int]] = {}
        for b, (cache, n) in enumerate(zip(caches, q_lens)):
            if n == 1 and cache.length >= ps and cache.pages:
                by_first.setdefault(id(cache.pages[0]), []).append(b)
        out = []
        for rows in by_first.values():
            if len(rows) < cls.MIN_GROUP:
                continue
            ref = max(rows, key=lambda b: len(caches[b].pages))
            ref_pages, ref_full = caches[ref].pages, caches[ref].length // ps
            shared = []
            for b in rows:
                pages = caches[b].pages
                cap = min(caches[b].length // ps, ref_full, len(pages))
                k = 0
                while k < cap and pages[k] is ref_pages[k]:
                    k += 1
                shared.append(k)
            prev = 0
            for bound in cls._boundaries(shared):
                members = [b for b, k in zip(rows, shared) if k >= bound]
                out.append((ref, prev, bound, sorted(members)))
                prev = bound
        return out

    @classmethod
    def build(cls, batch: "PagedBatchCache", q_lens: list[int], k_lens: list[int]):
        # The merge kernel is built for head_dim 128.
        if batch.pool.device.type != "cuda" or batch.pool.config.head_dim != 128:
            return None
        levels = cls.levels(batch, q_lens)
        if not levels:
            return None
        device, ps = batch.pool.device, batch.pool.page_size
        config = batch.pool.config
        n_seq = len(batch.caches)
        offsets = [0, *accumulate(q_lens)]
        shift = [0] * n_seq
        rows_a, cu_a, used_a, tables_a, spans = [], [0], [], [], []
        for ref, first, end, rows in levels:
            spans.append((len(rows_a), len(rows)))
            for b in rows:
                shift[b] = max(shift[b], end)
                rows_a.append(offsets[b])
            cu_a.append(cu_a[-1] + len(rows))
            used_a.append((end - first) * ps)
            tables_a.append([page.index for page in batch.caches[ref].pages[first:end]])
        width_a = max(len(t) for t in tables_a)
        width_b = batch.block_table.shape[1]
        tables_b = [[page.index for page in cache.pages[shift[b]:]] for b, cache in enumerate(batch.caches)]
        k_lens_b = [k - x * ps for k, x in zip(k_lens, shift)]
        # One merge pass: every member row folds in its levels' results in level order.
        parts: dict[int, list[int]] = {}
        for start, count in spans:
            for j in range(start, start + count):
                parts.setdefault(rows_a[j], []).append(j)
        out_rows = sorted(parts)
        part_start = [0, *accumulate(len(parts[r]) for r in out_rows)]
        part_idx = [j for r in out_rows for j in parts[r]]
        # Members are decode rows, so a packed row names its sequence.
        seq_of_row = {offsets[b]: b for b in range(n_seq) if q_lens[b] == 1}
        member_seq = [seq_of_row[r] for r in out_rows]
        member_of_seq = [-1] * n_seq
        for k, b in enumerate(member_seq):
            member_of_seq[b] = k
        # Every int32 array of the cascade in one pinned host buffer and every int64 array
        # in another: two non-blocking host-to-device copies per tick (the tick never waits
        # for the device); the tensors below are views of their device copies.
        pin32, i32 = _pinned(len(tables_a) * width_a + len(tables_b) * width_b + n_seq
                             + len(cu_a) + len(used_a) + len(part_start) + len(part_idx)
                             + len(member_seq) + n_seq, torch.int32)
        at = 0

        def put(values):
            nonlocal at
            i32[at:at + len(values)] = values
            at += len(values)
            return at - len(values), len(values)

        spans32 = {}
        for j, t in enumerate(tables_a):
            i32[at + j * width_a: at + j * width_a + len(t)] = t
        spans32["bt_a"] = (at, len(tables_a) * width_a)
        at += len(tables_a) * width_a
        for j, t in enumerate(tables_b):
            row = t[:width_b]
            i32[at + j * width_b: at + j * width_b + len(row)] = row
        spans32["bt_b"] = (at, len(tables_b) * width_b)
        at += len(tables_b) * width_b
        spans32["shift"] = put([x * ps for x in shift])
        spans32["cu_a"] = put(cu_a)
        spans32["used_a"] = put(used_a)
        spans32["part_start"] = put(part_start)
        spans32["part_idx"] = put(part_idx)
        spans32["member_seq"] = put(member_seq)
        spans32["member_of_seq"] = put(member_of_seq)
        pin64, i64 = _pinned(len(rows_a) + len(out_rows), torch.int64)
        i64[:] = rows_a + out_rows
        dev32 = torch.empty(pin32.shape, dtype=torch.int32, device=device)
        dev32.copy_(pin32, non_blocking=True)
        dev64 = torch.empty(pin64.shape, dtype=torch.int64, device=device)
        dev64.copy_(pin64, non_blocking=True)

        def view(name):
            o, n = spans32[name]
            return dev32[o:o + n]

        bt_a = view("bt_a").view(len(tables_a), width_a)
        bt_b = view("bt_b").view(len(tables_b), width_b)
        used_b = batch.seqused_k - view("shift")
        heads = dict(n_q_heads=config.n_heads, n_kv_heads=config.n_kv_heads, head_dim=config.head_dim,
                     page_size=ps)
        plan_a = ops.VarlenAttnPlan(
            view("cu_a"), None, view("used_a"),
            total_q=len(rows_a), max_q=max(len(lv[3]) for lv in levels), max_k=max(used_a),
            block_table_stride=width_a, window=(-1, -1),
            q_lens=[len(lv[3]) for lv in levels], k_lens=used_a, **heads)
        plan_b = ops.VarlenAttnPlan(
            batch.cu_seq_q, batch.cu_seq_k, used_b, total_q=offsets[-1], max_q=max(q_lens),
            max_k=max(k_lens_b), block_table_stride=width_b, window=(-1, 0),
            q_lens=q_lens, k_lens=k_lens_b, **heads)
        rows_t = dev64[:len(rows_a)]
        merge = (dev64[len(rows_a):], view("part_start"), view("part_idx"))
        members = (view("member_seq"), view("member_of_seq"))
        return cls(plan_a, plan_b, rows_t, merge, members, bt_a, bt_b)

    def attend(self, queries: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
               side: torch.cuda.Stream | None = None) -> torch.Tensor:
        """Attention of every packed row, the new K/V already in the pool. With ``side``,
        batch A and the chunk rows of batch B (MFMA) run there while the decode rows of
        batch B (HBM) run on the current stream."""
        rows_a, (out_rows, part_start, part_idx) = self.rows_a, self.merge

        def batch_a():  # member rows read in place through the row map (no gather)
            return self.plan_a.run(queries, k_pool, v_pool, self.bt_a, return_lse=True, query_rows=rows_a)

        if side is None:
            member_seq, member_of_seq = self.members
            if self.plan_a.hints[0] == 0:
                # One stream, one call, three launches: batch A's chunk items share batch
                # B's chunk launch, ahead of batch B's decode launch, which also runs
                # batch A's combine records (workgroups after the decode ones); batch B's
                # combine launch does the members' merge.
                pa = self.plan_a
                o_a = torch.empty((pa.total_q, pa.n_q_heads, pa.head_dim), dtype=queries.dtype, device=queries.device)
                lse_a = torch.empty((pa.n_q_heads, pa.total_q), dtype=torch.float32, device=queries.device)
                merge = ops.MergeParts(o_a, lse_a, member_seq, member_of_seq, part_start, part_idx,
                                       level_plan=pa, level_block_table=self.bt_a, level_query_rows=rows_a)
            else:
                # Batch A's decode and chunk launches first, then batch B as above.
                o_a, lse_a = self.plan_a.run(queries, k_pool, v_pool, self.bt_a, return_lse=True,
                                             query_rows=rows_a, phases=("decode", "chunk"))
                merge = ops.MergeParts(o_a, lse_a, member_seq, member_of_seq, part_start, part_idx,
                                       level_plan=self.plan_a)
            out, _ = self.plan_b.run(queries, k_pool, v_pool, self.bt_b, return_lse=True, merge=merge)
            return out
        (out, lse), (o_a, lse_a) = ops.run_overlapped(self.plan_b, queries, k_pool, v_pool, self.bt_b,
                                                      side, return_lse=True, side_first=batch_a)
        ops.attn_merge(out, lse, o_a, lse_a, out_rows, parts=(part_start, part_idx))
        return out


# --------------------------------------------------- attention over selected blocks
@dataclass(frozen=True)
class BlockSparse:
    """How the decode rows of a batch attend to long caches: each row, per KV head, to
    ``budget`` blocks of the pool's ``block_size`` tokens, the first ``sink``, the last
    ``recent`` and otherwise those whose key bounds promise the highest scores
    (``ops.select_blocks``). Rows of at most ``budget`` blocks attend to all of their keys."""

    budget: int
    sink: int = 1
    recent: int = 2

    def __post_init__(self) -> None:
        if self.sink < 0 or self.recent < 1 or self.sink + self.recent > self.budget:
            raise ValueError("a sparse budget must cover its sink (at least 0) and recent (at least 1) blocks")


class _SparseTick:
    """One tick's sparse attention: its decode rows (one new token) over selected blocks, its
    other rows over all of their keys with a plan of their own. ``None`` tensors mean all
    sequences are decode rows, in order."""

    def __init__(self, batch: PagedBatchCache, sparse: BlockSparse, counts: list[int], ends: list[int]) -> None:
        self.sparse, self.batch = sparse, batch
        self.rows = self.row_seq = self.plan = None
        self.keys = batch.seqused_k
        if max(counts) == 1:
            return
        pool, config = batch.pool, batch.pool.config
        starts = [0, *accumulate(counts)]
        decode = [b for b, n in enumerate(counts) if n == 1]
        chunks = [b for b, n in enumerate(counts) if n > 1]
        chunk_counts, chunk_ends = [counts[b] for b in chunks], [ends[b] for b in chunks]
        chunk_rows = [r for b in chunks for r in range(starts[b], starts[b + 1])]
        parts = [decode, [ends[b] for b in decode], [0, *accumulate(chunk_counts)], chunk_ends, chunks]
        pin32, i32 = _pinned(sum(map(len, parts)), torch.int32)
        pin64, i64 = _pinned(len(decode) + len(chunk_rows), torch.int64)
        i32[:] = [x for part in parts for x in part]
        i64[:] = [starts[b] for b in decode] + chunk_rows
        dev32 = torch.empty(pin32.shape, dtype=torch.int32, device=pool.device)
        dev32.copy_(pin32, non_blocking=True)
        dev64 = torch.empty(pin64.shape, dtype=torch.int64, device=pool.device)
        dev64.copy_(pin64, non_blocking=True)
        self.row_seq, self.keys, cu_q, used, ids = dev32.split([len(part) for part in parts])
        self.rows, self.chunk_rows = dev64.split([len(decode), len(chunk_rows)])
        self.table = batch.block_table.index_select(0, ids)
        self.plan = ops.VarlenAttnPlan(
            cu_q, None, used, total_q=len(chunk_rows), max_q=max(chunk_counts), max_k=max(chunk_ends),
            n_q_heads=config.n_heads, n_kv_heads=config.n_kv_heads, head_dim=config.head_dim,
            page_size=pool.page_size, block_table_stride=self.table.shape[1], window=(-1, 0),
            q_lens=chunk_counts, k_lens=chunk_ends)

    def attend(self, rows: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
               bounds: torch.Tensor) -> torch.Tensor:
        """Attention of every packed row, the new K/V and bounds already in the pool."""
        sparse, block, table = self.sparse, self.batch.pool.block_size, self.batch.block_table
        out = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
        blocks = ops.select_blocks(rows, bounds, table, self.keys, sparse.budget, block_size=block, sink=sparse.sink,
                                   recent=sparse.recent, row_seq=self.row_seq, rows=self.rows)
        ops.block_sparse_attn(rows, k_pool, v_pool, blocks, table, self.keys, block_size=block,
                              row_seq=self.row_seq, rows=self.rows, out=out)
        if self.plan is not None:
            chunk_out = self.plan.run(rows, k_pool, v_pool, self.table, query_rows=self.chunk_rows)
            out.index_copy_(0, self.chunk_rows, chunk_out)
        return out


# ------------------------------------------------------------------- batches
class PagedBatchCache:
    """Request caches of one pool stepping together (paged_cache.py:177-345).

    ``prepare(T)`` reserves pages for T new tokens per request and builds the tick's
    metadata; ``attend`` appends each layer's new K/V and runs paged attention;
    ``advance(T)`` commits the tokens. ``caches`` may be reassigned between ticks (the
    reference's decoder reuses one batch object that way).

    ``device_metadata`` (default: the pool is on a ROCm device) builds the metadata with
    the kernel instead of on the host. ``prefix_cascade`` (same default) lets decode rows
    that share leading pages attend to them once per group (``_PrefixCascade``).
    ``overlap=True`` runs chunk rows (MFMA-bound) and the cascade's batch A on a second
    stream while decode rows (HBM-bound) run on the current one. It is off by default: on
    MI355X the decode grid fills every CU and a chunk workgroup cannot share a CU with
    decode workgroups, so the kernels interleave rather than overlap (the full Qwen3-4B
    tick measured 12.5 ms of attention with it, 12.0 ms without). ``sparse`` lets decode rows
    of long caches attend to selected blocks; a tick in which one does runs on one stream
    and without the cascade."""

    def __init__(self, caches: Sequence[PagedKVCache], *, device_metadata: bool | None = None,
                 prefix_cascade: bool | None = None, overlap: bool = False,
                 sparse: BlockSparse | None = None) -> None:
        caches = tuple(caches)
        if not caches:
            raise ValueError("a paged batch needs at least one request cache")
        pool = caches[0].pool
        if any(cache.pool is not pool for cache in caches):
            raise ValueError("every request cache of a paged batch must use one page pool")
        if len({id(cache) for cache in caches}) != len(caches):
            raise ValueError("a request cache appears more than once in the paged batch")
        on_gpu = pool.device.type == "cuda"
        if device_metadata is None:
            device_metadata = on_gpu
        if device_metadata and not on_gpu:
            raise ValueError("device metadata needs a pool on a ROCm device")
        if overlap and not on_gpu:
            raise ValueError("overlapped streams need a pool on a ROCm device")
        if sparse is not None and pool.bounds is None:
            raise ValueError("block-sparse attention needs a pool with key bounds (block_size)")
        if sparse is not None and _page_count(pool.config.context_length, pool.page_size) \
                * (pool.page_size // pool.block_size) > ops.MAX_SELECT_BLOCKS:
            raise ValueError(f"block-sparse attention covers {ops.MAX_SELECT_BLOCKS} blocks of a context; "
                             "use larger ones")
        self.pool = pool
        self.caches = caches
        self._sparse = sparse
        self._sparse_tick: _SparseTick | None = None
        self.batch_size = len(caches)
        self._staged: dict[str, tuple[torch.Tensor, np.ndarray]] = {}
        self._table_key: tuple | None = None
        self._device_meta = _DeviceTickMetadata(pool.device) if device_metadata else None
        self._use_cascade = on_gpu if prefix_cascade is None else bool(prefix_cascade)
        self._overlap = bool(overlap)
        self._side_stream: torch.cuda.Stream | None = None
        self._plan: ops.VarlenAttnPlan | None = None
        self._cascade: _PrefixCascade | None = None
        self._lens: tuple[list[int], list[int]] | None = None
        self._row_positions: torch.Tensor | None = None

    # -- bookkeeping ----------------------------------------------------------
    @property
    def length(self) -> int:
        if len(self.caches) != 1:
            raise RuntimeError("requests of a paged batch have their own lengths; use slot_length")
        return self.caches[0].length

    def slot_ids(self, slots: Sequence[int] | torch.Tensor) -> tuple[int, ...]:
        """The batch's slots, which must be every request in order."""
        if isinstance(slots, torch.Tensor):
            if slots.ndim != 1:
                raise ValueError(f"paged batch slots must be a 1-D tensor, not {slots.ndim}-D")
            slots = slots.tolist()
        rows = tuple(int(s) for s in slots)
        if rows != tuple(range(len(self.caches))):
            raise ValueError(f"paged batch slots must be 0..{len(self.caches) - 1} in order, not {rows}")
        return rows

    def slot_length(self, slot: int) -> int:
        if not 0 <= slot < len(self.caches):
            raise ValueError(f"slot {slot} is outside the batch of {len(self.caches)}")
        return self.caches[slot].length

    def slot_lengths(self, slots: Sequence[int] | torch.Tensor) -> torch.Tensor:
        """Committed lengths of the slots, int64, on the pool's device."""
        rows = self.slot_ids(slots)
        return self.metadata("slot_lengths", [self.caches[r].length for r in rows], torch.long)

    def metadata(self, name: str, values, dtype: torch.dtype) -> torch.Tensor:
        """``values`` (a list, nested lists for 2-D, or an array) as a ``dtype`` tensor on
        the pool's device, kept per ``name``: the same tensor is returned, and uploaded
        again only when the values change."""
        array = np.asarray(values, dtype=_NUMPY_DTYPE.get(dtype))
        staged = self._staged.get(name)
        if staged is not None and staged[0].dtype == dtype and tuple(staged[0].shape) == array.shape:
            tensor, last = staged
            if np.array_equal(last, array):
                return tensor
        else:
            tensor = torch.empty(array.shape, dtype=dtype, device=self.pool.device)
        # A fresh array each call: the copy's source is never rewritten afterwards.
        tensor.copy_(torch.from_numpy(array))
        self._staged[name] = (tensor, array)
        return tensor

    def prepare(self, tokens: int) -> None:
        """Reserve pages for ``tokens`` new tokens of every request and build the tick's
        metadata (paged_cache.py:221-270)."""
        if tokens < 1:
            raise ValueError(f"a paged append needs at least one token, not {tokens}")
        self._begin_tick([tokens] * len(self.caches), None, packed=False)

    def advance(self, tokens: int, *, slots: Sequence[int] | torch.Tensor | None = None) -> None:
        """Commit the ``tokens`` prepared for every request."""
        if slots is not None:
            self.slot_ids(slots)
        if any(cache._pending_tokens != tokens for cache in self.caches):
            raise RuntimeError(f"advance({tokens}) does not match the tokens prepared this tick")
        self._commit([tokens] * len(self.caches))

    def _commit(self, counts: Sequence[int]) -> None:
        """The prepared tokens become part of each request's committed length."""
        for cache, n in zip(self.caches, counts):
            cache.length += n
            cache._pending_tokens = None

    def _begin_tick(self, counts: list[int], tails: list[int] | None, *, packed: bool) -> None:
        """Validate, reserve pages (nothing is taken when any check fails), mark the
        appends pending and build the metadata. A request with an append already in
        flight raises RuntimeError for ``prepare`` and ValueError for ``prepare_packed``,
        the reference's exception types."""
        caches = self.caches
        size = self.pool.page_size
        on_gpu = self.pool.device.type == "cuda"
        short: list[int] = []
        for cache, n in zip(caches, counts):
            if cache._pending_tokens is not None:
                raise (ValueError if packed else RuntimeError)(
                    "a request of the batch already has an append in flight")
            if cache.length + n > cache.capacity:
                raise ValueError(
                    f"appending {n} tokens to {cache.length} exceeds the request capacity {cache.capacity}")
            short.append(max(0, _page_count(cache.length + n, size) - len(cache.pages)))
        if sum(short) > self.pool.free_pages:
            raise RuntimeError(
                f"KV page pool exhausted: the tick needs {sum(short)} pages, {self.pool.free_pages} free")
        for cache, n, extra in zip(caches, counts, short):
            if extra:
                cache.pages.extend(self.pool.acquire(extra))
            cache._pending_tokens = n
        self.batch_size = len(caches)
        self.counts = tuple(counts)
        lengths = [cache.length for cache in caches]
        tables = [[page.index for page in cache.pages] for cache in caches]
        width = max(_page_count(cache.capacity, size) for cache in caches)
        if self._device_meta is not None:
            ends = self._device_tick(lengths, counts, tails, tables, width)
        else:
            ends = self._host_tick(lengths, counts, tails, tables, width)
        self._plan = None
        self._lens = (list(counts), ends)
        self._sparse_tick = self._cascade = None
        if self._sparse is not None and on_gpu and any(
                n == 1 and end > self._sparse.budget * self.pool.block_size for n, end in zip(counts, ends)):
            self._sparse_tick = _SparseTick(self, self._sparse, list(counts), ends)
        elif self._use_cascade:
            self._cascade = _PrefixCascade.build(self, list(counts), ends)

    def _host_tick(self, lengths, counts, tails, tables, width) -> list[int]:
        tick = _HostTick(lengths, counts, tails, tables, width, self.pool.page_size)
        key = (width, tuple(map(tuple, tables)))
        if key != self._table_key:
            self.block_table = self.metadata("block_table", tick.block_table, torch.int32)
            self._table_key = key
        self.cu_seq_q = self.metadata("cu_seq_q", tick.cu_seq_q, torch.int32)
        self.cu_seq_k = self.metadata("cu_seq_k", tick.cu_seq_k, torch.int32)
        self.seqused_k = self.metadata("seqused_k", tick.seqused_k, torch.int32)
        self.write_slots = self.metadata("write_slots", tick.write_slots, torch.long)
        self._host_positions = tick.positions
        self._row_positions = None
        if tails is not None:
            self.positions = self.metadata("positions", tick.positions, torch.long).unsqueeze(0)
            self.logit_indices = self.metadata("logit_indices", tick.logit_indices, torch.long)
        self.max_q, self.max_k = tick.max_q, tick.max_k
        return tick.ends

    def _device_tick(self, lengths, counts, tails, tables, width) -> list[int]:
        """The tick's metadata from the kernel: O(batch) host work, two small copies."""
        meta = self._device_meta
        key = (width, tuple(map(tuple, tables)))
        if key != self._table_key or meta.block_table is None:
            self.block_table = meta.upload_block_table(tables, width)
            self._table_key = key
        views = meta.build(lengths, counts, tails, self.pool.page_size)
        self.cu_seq_q = views["cu_seq_q"]
        self.cu_seq_k = views["cu_seq_k"]
        self.seqused_k = views["seqused_k"]
        self.write_slots = views["write_slots"]
        self._row_positions = views["positions"]
        if tails is not None:
            self.positions = views["positions"].unsqueeze(0)
            self.logit_indices = views["logit_indices"]
        ends = [s + n for s, n in zip(lengths, counts)]
        self.max_q, self.max_k = max(counts), max(ends)
        return ends

    # -- attention ----------------------------------------------------------------
    def _side(self) -> torch.cuda.Stream | None:
        """Second stream (default priority) for chunk rows and the cascade's batch A, which
        then overlap the decode rows; None when overlapping is off."""
        if not self._overlap:
            return None
        if self._side_stream is None:
            self._side_stream = torch.cuda.Stream(device=self.pool.device)
        return self._side_stream

    def _attention_plan(self, total_q: int) -> ops.VarlenAttnPlan:
        """The tick's work plan, built at the first layer and reused by the others."""
        if self._plan is None:
            config = self.pool.config
            q_lens, k_lens = self._lens
            self._plan = ops.VarlenAttnPlan(
                self.cu_seq_q, self.cu_seq_k, self.seqused_k,
                total_q=total_q, max_q=self.max_q, max_k=self.max_k,
                n_q_heads=config.n_heads, n_kv_heads=config.n_kv_heads,
                head_dim=config.head_dim, page_size=self.pool.page_size,
                block_table_stride=self.block_table.shape[1], window=(-1, 0),
                q_lens=q_lens, k_lens=k_lens,
            )
        return self._plan

    def _require_device(self) -> None:
        if self.pool.device.type != "cuda":
            raise RuntimeError(
                "helios_amd paged attention runs on a ROCm device only; this pool is on "
                f"{self.pool.device}. There is no CPU fallback."
            )

    def _require_pending(self) -> None:
        if any(cache._pending_tokens is None for cache in self.caches):
            raise RuntimeError("prepare the tick before paged attention")

    def attend(self, layer: int, queries: torch.Tensor, keys: torch.Tensor,
               values: torch.Tensor) -> torch.Tensor:
        """Append this layer's new K/V and attend (paged_cache.py:301-333): queries
        ``[B, Hq, T, d]``, keys / values ``[B, Hkv, T, d]``; returns ``[B, Hq, T, d]``."""
        tokens = _validate_attention_inputs(self, layer, queries, keys, values)
        if any(cache._pending_tokens != tokens for cache in self.caches):
            raise RuntimeError(f"prepare({tokens}) must precede paged attention over {tokens} tokens")
        self._require_device()
        rows = queries.transpose(1, 2).reshape(-1, queries.shape[1], queries.shape[3])
        out = self._append_and_attend(layer, rows, keys, values)
        return out.view(len(self.caches), tokens, queries.shape[1], queries.shape[3]).transpose(1, 2)

    def attend_projected(self, layer: int, queries: torch.Tensor, keys: torch.Tensor,
                         values: torch.Tensor, q_norm_weight: torch.Tensor,
                         k_norm_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                         eps: float) -> torch.Tensor:
        """``attend`` for raw projections: q_norm/k_norm + RoPE (layers.py:146-160) run
        fused with the KV append, then paged attention.

        ``queries`` ``[B, T, Hq * d]``, ``keys``/``values`` ``[B, T, Hkv * d]`` as the
        projection layers produce them (``[1, sum(counts), ...]`` for a packed tick).
        Returns what ``attend`` returns for the normalised, rotated inputs."""
        config = self.pool.config
        if not 0 <= layer < config.n_layers:
            raise ValueError(f"layer {layer} is outside the model's {config.n_layers} layers")
        self._require_pending()
        rows = queries.shape[0] * queries.shape[1]
        if rows != self.write_slots.shape[0]:
            raise ValueError(f"{rows} projected rows do not match the {self.write_slots.shape[0]} prepared")
        self._require_device()
        k_pool, v_pool = self.pool.keys[layer], self.pool.values[layer]
        q_rot = ops.qk_norm_rope_append_packed(
            queries, keys, values, config.n_heads, q_norm_weight, k_norm_weight, cos, sin, self._positions_for_rows(),
            k_pool, v_pool, self.write_slots, eps)
        if q_rot is not None:
            out = self._attend_rows(q_rot, layer)
            return out.view(1, rows, config.n_heads, config.head_dim).transpose(1, 2)
        q = queries.reshape(rows, config.n_heads, config.head_dim)
        k = keys.reshape(rows, config.n_kv_heads, config.head_dim)
        v = values.reshape(rows, config.n_kv_heads, config.head_dim)
        q_rot = ops.qk_norm_rope_append(q, k, v, q_norm_weight, k_norm_weight, cos, sin,
                                        self._positions_for_rows(), k_pool, v_pool,
                                        self.write_slots, eps)
        out = self._attend_rows(q_rot, layer)
        return out.view(queries.shape[0], queries.shape[1], config.n_heads, config.head_dim).transpose(1, 2)

    def _positions_for_rows(self) -> torch.Tensor:
        """Absolute position of every packed row (int64, on the device)."""
        if self._row_positions is None:
            self._row_positions = self.metadata("row_positions", self._host_positions, torch.long)
        return self._row_positions

    def _update_bounds(self, layer: int) -> None:
        """Key bounds of the blocks this tick's new keys went to, if the pool keeps them."""
        if self.pool.bounds is not None:
            ops.kv_block_bounds(self.pool.keys[layer], self.pool.bounds[layer], self.block_table, self.cu_seq_q,
                                self.seqused_k, max_q=self.max_q)

    def _attend_rows(self, rows: torch.Tensor, layer: int) -> torch.Tensor:
        """Attention of packed query rows whose new K/V is already in the pool."""
        k_pool, v_pool = self.pool.keys[layer], self.pool.values[layer]
        self._update_bounds(layer)
        if self._sparse_tick is not None:
            return self._sparse_tick.attend(rows, k_pool, v_pool, self.pool.bounds[layer])
        if self._cascade is not None:
            return self._cascade.attend(rows, k_pool, v_pool, self._side())
        plan = self._attention_plan(rows.shape[0])
        side = self._side()
        if side is not None:
            return ops.run_overlapped(plan, rows, k_pool, v_pool, self.block_table, side)
        out = plan.attend_rows(rows, k_pool, v_pool, self.block_table)
        return out if out is not None else plan.run(rows, k_pool, v_pool, self.block_table)

    def _write(self, layer: int, keys: torch.Tensor, values: torch.Tensor) -> None:
        """KV append alone (paged_cache.py:335-345): ``[B, Hkv, T, d]`` rows to their
        write slots."""
        k_rows, v_rows = _as_rows(keys), _as_rows(values)
        ops.kv_append(self.pool.keys[layer], self.pool.values[layer], self.write_slots, k_rows, v_rows)

    def _append_and_attend(self, layer: int, rows: torch.Tensor, keys: torch.Tensor,
                           values: torch.Tensor) -> torch.Tensor:
        """``_write`` then paged attention: one fused call when the new rows allow 16-byte
        loads (always, for contiguous projections), else the append kernel first."""
        k_rows, v_rows = _as_rows(keys), _as_rows(values)
        k_pool, v_pool = self.pool.keys[layer], self.pool.values[layer]
        fused = (self._cascade is None and self._sparse_tick is None and self._side() is None
                 and _vector_aligned(k_rows) and _vector_aligned(v_rows))
        if fused:
            plan = self._attention_plan(rows.shape[0])
            out = plan.run(rows, k_pool, v_pool, self.block_table, append=(k_rows, v_rows, self.write_slots))
            self._update_bounds(layer)
            return out
        ops.kv_append(k_pool, v_pool, self.write_slots, k_rows, v_rows)
        return self._attend_rows(rows, layer)


class PackedBatchCache(PagedBatchCache):
    """A tick where request i contributes ``counts[i]`` query tokens, all packed along one
    token dimension (paged_cache.py:417-546): decode rows and prefill chunks together."""

    def prepare_packed(self, counts: Sequence[int], logit_counts: Sequence[int] | None = None) -> None:
        """Reserve pages for each request's ``counts[i]`` tokens and build the packed
        metadata; ``logit_counts[i]`` trailing rows of request i produce logits (1 each
        by default)."""
        counts = [int(n) for n in counts]
        if len(counts) != len(self.caches) or min(counts, default=0) < 1:
            raise ValueError("a packed tick needs one token count of at least 1 per request")
        tails = [1] * len(counts) if logit_counts is None else [int(n) for n in logit_counts]
        if len(tails) != len(counts) or any(not 1 <= t <= n for t, n in zip(tails, counts)):
            raise ValueError("each request's logit rows must number 1 to its token count")
        self._begin_tick(counts, tails, packed=True)

    def advance_packed(self) -> None:
        """Commit every request's prepared tokens."""
        self._commit(self.counts)

    def attend(self, layer, queries, keys, values):
        """Packed ``attend`` (paged_cache.py:501-520): queries ``[1, Hq, sum(counts), d]``,
        keys / values ``[1, Hkv, sum(counts), d]``."""
        if queries.shape[0] != 1 or queries.shape[2] != sum(self.counts):
            raise ValueError(
                f"packed attention takes [1, heads, {sum(self.counts)}, head_dim] queries, "
                f"not {list(queries.shape)}")
        self._require_device()
        if self._cascade is None and self._sparse_tick is None and not self._overlap:
            out = self._attention_plan(queries.shape[2]).append_attend(
                queries, keys, values, self.pool.keys[layer], self.pool.values[layer], self.block_table,
                self.write_slots)
            if out is not None:
                self._update_bounds(layer)
                return out
        out = self._append_and_attend(layer, queries[0].transpose(0, 1), keys, values)
        return out.transpose(0, 1).unsqueeze(0)


def _as_rows(x: torch.Tensor) -> torch.Tensor:
    """``[B, H, T, d]`` -> ``[B * T, H, d]`` in packed-row order (a view when possible)."""
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])


def _vector_aligned(t: torch.Tensor) -> bool:
    return t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0


def _validate_attention_inputs(cache: PagedBatchCache, layer: int, queries: torch.Tensor,
                               keys: torch.Tensor, values: torch.Tensor) -> int:
    """Check a layer index and the ``[B, H, T, d]`` shapes of queries, keys and values
    against the pool's config (ValueError, as paged_cache.py:352-375); returns T."""
    config = cache.pool.config
    if not 0 <= layer < config.n_layers:
        raise ValueError(f"layer {layer} is outside the model's {config.n_layers} layers")
    if queries.ndim != 4 or keys.ndim != 4:
        raise ValueError("paged attention takes 4-D [batch, heads, tokens, head_dim] tensors")
    tokens = keys.shape[2]
    rows = len(cache.caches)
    want_q = (rows, config.n_heads, tokens, config.head_dim)
    want_kv = (rows, config.n_kv_heads, tokens, config.head_dim)
    if tuple(queries.shape) != want_q or tuple(keys.shape) != want_kv or tuple(values.shape) != want_kv:
        raise ValueError(
            f"paged attention expects queries {list(want_q)} and keys/values {list(want_kv)}, got "
            f"{list(queries.shape)}, {list(keys.shape)} and {list(values.shape)}")
    return tokens
