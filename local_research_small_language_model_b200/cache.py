"""Block-major KV cache for the B200 path (replaces model/attention/base.py:11-32).

Storage per layer:
  k_store, v_store  [B, H, Tcap, D]  activation dtype; one (head, block) tile of
                    block_size x D is contiguous (8 KB at 64 x 64 bf16), so the
                    decode kernel stages a block with one bulk copy;
  proto_sum         [B, H, NBcap, D] fp32 running block sums of K, so the
                    compressor (model/forecast.py:57-78) is never re-run over
                    the whole cache: prototype = proto_sum / block_size;
  len_dev           int32 on the device, tokens cached so far (read by the
                    fused decode kernel, which makes CUDA-graph replay possible).
Tcap is max_seq_len rounded up to a whole block.  ``k`` and ``v`` return views
in the reference's [B, T, H, D] layout.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import ops


class B200KVCache:
    def __init__(self, max_batch_size: int, max_seq_len: int, n_kv_head: int, head_dim: int,
                 device: torch.device, dtype: torch.dtype, block_size: int = 64,
                 len_dev: Optional[torch.Tensor] = None):
        self.block_size = block_size
        self.max_batch_size = max_batch_size
        self.max_seq_len = max_seq_len
        self.n_kv_head = n_kv_head
        self.head_dim = head_dim
        self.tcap = ops.num_blocks(max_seq_len, block_size) * block_size
        self.nbcap = self.tcap // block_size
        self.k_store = torch.zeros(max_batch_size, n_kv_head, self.tcap, head_dim, device=device, dtype=dtype)
        self.v_store = torch.zeros_like(self.k_store)
        self.proto_sum = torch.zeros(max_batch_size, n_kv_head, self.nbcap, head_dim, device=device,
                                     dtype=torch.float32)
        self.len_dev = len_dev if len_dev is not None else torch.zeros(1, dtype=torch.int32, device=device)
        self.current_len = 0

    @property
    def k(self) -> torch.Tensor:
        return self.k_store.permute(0, 2, 1, 3)

    @property
    def v(self) -> torch.Tensor:
        return self.v_store.permute(0, 2, 1, 3)

    def update(self, xk: torch.Tensor, xv: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Appends xk, xv [B,T,H,D]; returns the cached [B,current_len,H,D] views
        (KVCache.update, model/attention/base.py:19-29)."""
        t = xk.shape[1]
        if self.current_len + t > self.tcap:
            raise ValueError(f"cache overflow: {self.current_len} + {t} > {self.tcap}")
        ops.kv_append(xk, xv, self.k_store, self.v_store, self.proto_sum, self.current_len, self.block_size)
        self.advance(t)
        return self.k[:, :self.current_len], self.v[:, :self.current_len]

    def advance(self, t: int, device: bool = True) -> None:
        """Bumps the host length and, unless the caller bumps a shared length
        array itself, the device length."""
        self.current_len += t
        if device:
            self.len_dev.add_(t)

    def prototypes(self) -> torch.Tensor:
        """Block prototypes [B, N_b, H, D] fp32 of the cached tokens."""
        nb = ops.num_blocks(self.current_len, self.block_size)
        return (self.proto_sum[:, :, :nb] / self.block_size).permute(0, 2, 1, 3)

    def reset(self) -> None:
        self.current_len = 0
        self.len_dev.zero_()


class PageTable:
    """Which pages of a pool hold each sequence, shared by the layers' caches.

      table  int32 [max_seqs, width] on the device: position t of sequence b
             lies in page table[b, t // page_size]; -1 where none is held;
      lens   int32 [max_seqs] on the device, tokens cached so far;
      active int32 [max_seqs] on the device: 0 for a released sequence, which
             takes no part in decode steps until a prompt takes its place, else 1
             (absent: 0 where active is 1, else ops.LEN_ABSENT).

    The host keeps the same lengths (``held``), each sequence's pages, the
    released sequences and the free pages; ``reserve`` before a forward,
    ``advance`` after it."""

    def __init__(self, max_seqs: int, max_seq_len: int, num_pages: int, device: torch.device, page_size: int = 64):
        if min(max_seqs, max_seq_len, num_pages, page_size) < 1:
            raise ValueError("max_seqs, max_seq_len, num_pages and page_size must be positive")
        self.max_seqs, self.num_pages, self.page_size = max_seqs, num_pages, page_size
        self.width = ops.num_blocks(max_seq_len, page_size)
        self.capacity = self.width * page_size
        self.table = torch.full((max_seqs, self.width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.active = torch.ones(max_seqs, dtype=torch.int32, device=device)
        self.absent = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.reset_host()

    def reset_host(self) -> None:
        self.held: List[int] = [0] * self.max_seqs
        self.owned: List[List[int]] = [[] for _ in range(self.max_seqs)]
        self.free: List[int] = list(range(self.num_pages - 1, -1, -1))
        self.released: List[bool] = [False] * self.max_seqs

    def _counts(self, counts) -> List[int]:
        if isinstance(counts, int):
            counts = [min(counts, 0) if out else counts for out in self.released]
        else:
            counts = [int(c) for c in counts]
        if len(counts) != self.max_seqs or min(counts) < 0:
            raise ValueError(f"need {self.max_seqs} non-negative token counts, got {counts}")
        return counts

    def reserve(self, counts) -> None:
        """Pages for counts[b] more tokens of every sequence b, or the same
        number for all but the released ones.  A list's tokens for a released
        sequence take its place up again.  Raises, with nothing changed, when a
        sequence would pass its longest or the pool has too few pages."""
        counts = self._counts(counts)
        need = []
        for b, c in enumerate(counts):
            if self.held[b] + c > self.capacity:
                raise ValueError(f"cache overflow: sequence {b} would hold {self.held[b] + c} of {self.capacity}")
            need.append(max(0, ops.num_blocks(self.held[b] + c, self.page_size) - len(self.owned[b])))
        if sum(need) > len(self.free):
            raise ValueError(f"out of pages: {sum(need)} needed, {len(self.free)} free")
        rows, cols, pages = [], [], []
        for b, n in enumerate(need):
            for _ in range(n):
                rows.append(b)
                cols.append(len(self.owned[b]))
                self.owned[b].append(self.free.pop())
                pages.append(self.owned[b][-1])
        if pages:
            where = torch.tensor([rows, cols, pages], dtype=torch.int64).to(self.table.device)
            self.table[where[0], where[1]] = where[2].to(torch.int32)
        for b, c in enumerate(counts):
            if c and self.released[b]:
                self._take_part(b, True)

    def _take_part(self, seq: int, yes: bool) -> None:
        self.released[seq] = not yes
        self.active[seq] = int(yes)
        self.absent[seq] = 0 if yes else ops.LEN_ABSENT

    def fills(self, lengths) -> bool:
        """Whether prompts of these lengths (None: unknown) would reach a
        sequence that holds tokens."""
        if lengths is None:
            return any(self.held)
        return any(n and h for n, h in zip(lengths, self.held))

    def advance(self, counts, device: bool = True) -> None:
        """Counts the tokens of a finished forward (counts as in reserve): on
        the host and, unless a captured step does that itself, on the device."""
        same = counts if isinstance(counts, int) else None
        counts = self._counts(counts)
        for b, c in enumerate(counts):
            if self.held[b] + c > len(self.owned[b]) * self.page_size:
                raise ValueError(f"sequence {b} has no pages for {self.held[b] + c} tokens: reserve them first")
        for b, c in enumerate(counts):
            self.held[b] += c
        if device:
            if same is not None:  # a captured step follows later releases
                self.lens.add_(self.active, alpha=same)
            elif len(set(counts)) == 1:
                self.lens.add_(counts[0])
            else:
                self.lens.add_(torch.tensor(counts, dtype=torch.int32).to(self.lens.device))

    def release(self, seq: int) -> None:
        """Frees a finished sequence's pages.  It takes no part in the steps
        that follow (its row of their results is that of no context); a prompt
        may take its place."""
        if not 0 <= seq < self.max_seqs:
            raise ValueError(f"no sequence {seq} of {self.max_seqs}")
        self.free.extend(reversed(self.owned[seq]))
        self.owned[seq], self.held[seq] = [], 0
        self.table[seq].fill_(-1)
        self.lens[seq] = 0
        self._take_part(seq, False)

    def reset(self) -> None:
        self.reset_host()
        self.table.fill_(-1)
        self.lens.zero_()
        self.active.fill_(1)
        self.absent.zero_()


class B200PagedKVCache:
    """One layer's pool of pages, k_pages and v_pages [num_pages, H, page, D]
    (head-major: a head's page is one contiguous run), under a PageTable that
    all layers share.  Sequences grow page by page, so a batch of ragged lengths
    holds what it needs and not batch x longest (KVCache.update,
    model/attention/base.py:11-32, reserves the longest for all)."""

    def __init__(self, pages: PageTable, n_kv_head: int, head_dim: int, device: torch.device, dtype: torch.dtype):
        self.pages = pages
        shape = (pages.num_pages, n_kv_head, pages.page_size, head_dim)
        self.k_pages = torch.zeros(shape, device=device, dtype=dtype)
        self.v_pages = torch.zeros(shape, device=device, dtype=dtype)

    def append(self, xk: torch.Tensor, xv: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
               lens: Optional[torch.Tensor] = None) -> None:
        """Writes rows xk, xv [N,H,D] behind the cached tokens of their
        sequences (one row each, or packed by cu_seqlens; ``lens`` in place of
        the PageTable's, ops.LEN_ABSENT for a sequence whose row is not
        written, as for the released ones without it); lengths are advanced on
        the PageTable, once for all layers."""
        pages = self.pages
        if lens is None:
            lens = pages.lens + pages.absent if any(pages.released) else pages.lens
        ops.paged_append(xk.to(self.k_pages.dtype), xv.to(self.v_pages.dtype), self.k_pages, self.v_pages, pages.table,
                         lens, cu_seqlens)
