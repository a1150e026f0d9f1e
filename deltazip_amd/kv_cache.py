"""A paged key/value cache: which pages belong to which sequence, and the tensors that a step needs of that.

The pages of all layers are held in one tensor, [2 layers, pages, kv_heads, page_size, head_dim]; a page number
means the same page in each.  Sequences that were forked share pages: a page is copied when a sequence is
about to write to one that others still read.  What the reference's serving engine (serving/vllm) divides between its scheduler
and its workers is here one class; the scheduling itself stays the caller's.

All bookkeeping is on the host and known when a call returns; what the device does follows in the order of the
current stream.  A cache serves one stream at a time: a page that was freed may be given away while kernels in
front of that still read it.
"""
from __future__ import annotations

import heapq
from typing import Dict, Hashable, Iterable, List, NamedTuple, Optional, Sequence, Tuple

import numpy as np
import torch


from .paged import MAX_DIM, copy_pages


class OutOfPages(RuntimeError):
    """The pool has too few free pages for the call; nothing was changed."""


class PagedBatch(NamedTuple):
    """What a step of one new token per row needs of the cache, on the device: the newest token's position and slot
    (int64 [rows]), the tables (int32 [rows, pages]) and lengths (int32 [rows], the new token counted); and, on the host, whether
    most of its rows' pages are another of its rows', too (for `paged_attention`, which takes no notice of it for one row; of
    one row: whether sharing spares the cache most of as many pages).  A captured step keeps what it was captured with."""
    positions: torch.Tensor
    slots: torch.Tensor
    block_tables: torch.Tensor
    lengths: torch.Tensor
    shared: bool = False


class _Sequence:
    __slots__ = ("row", "length", "pages")

    def __init__(self, row: int, length: int, pages: List[int]) -> None:
        self.row, self.length, self.pages = row, length, pages


class PagedKVCache:
    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, max_tokens: int,
                 dtype: torch.dtype = torch.float16, device="cuda") -> None:
        """max_tokens: of one sequence (how wide tables can get)."""
        if min(num_layers, num_pages, num_kv_heads, max_tokens) < 1:
            raise ValueError("layers, pages, heads and tokens must be positive")
        if page_size < 8 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError("a page must hold a power of two of tokens, from 8 to 1024")
        if head_dim < 8 or head_dim > MAX_DIM or head_dim % 8:
            raise ValueError(f"head_dim must be a multiple of 8 up to {MAX_DIM}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("keys and values are float16 or bfloat16")
        self.page_size, self.num_pages, self.num_layers = page_size, num_pages, num_layers
        self.max_pages = -(-max_tokens // page_size)
        self.pool = torch.empty((2 * num_layers, num_pages, num_kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self.keys: Sequence[torch.Tensor] = self.pool[:num_layers].unbind(0)       # per layer, [pages, kv_heads, page_size, dim]
        self.values: Sequence[torch.Tensor] = self.pool[num_layers:].unbind(0)
        self._free = list(range(num_pages))         # a heap: low pages first
        self._users = [0] * num_pages               # sequences that hold a page
        self._spared = 0                            # pages that sharing has spared: holders beyond the first
        self._seqs: Dict[Hashable, _Sequence] = {}
        self._rows = np.zeros((8, self.max_pages), dtype=np.int32)                 # tables, a row per sequence
        self._free_rows = list(range(8))[::-1]

    # -- what there is ---------------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def __contains__(self, seq: Hashable) -> bool:
        return seq in self._seqs

    def __len__(self) -> int:
        return len(self._seqs)

    def length(self, seq: Hashable) -> int:
        return self._get(seq).length

    def pages(self, seq: Hashable) -> Tuple[int, ...]:
        return tuple(self._get(seq).pages)

    def _get(self, seq: Hashable) -> _Sequence:
        s = self._seqs.get(seq)
        if s is None:
            raise ValueError(f"no sequence {seq!r} in the cache")
        return s

    # -- sequences that come, grow, fork and go ----------------------------------------------
    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._users[page] = 1
        return page

    def _new_row(self) -> int:
        if not self._free_rows:
            n = len(self._rows)
            self._rows = np.concatenate((self._rows, np.zeros_like(self._rows)))
            self._free_rows = list(range(n, 2 * n))[::-1]
        return self._free_rows.pop()

    def add(self, seq: Hashable, tokens: int = 0) -> None:
        """A new sequence with room for its first tokens (a prompt, say; they are stored by the caller at `slots`)."""
        if seq in self._seqs:
            raise ValueError(f"sequence {seq!r} is in the cache")
        need = self._pages_for(tokens)
        if need > len(self._free):
            raise OutOfPages(f"{need} pages wanted, {len(self._free)} free")
        pages = [self._take() for _ in range(need)]
        s = self._seqs[seq] = _Sequence(self._new_row(), tokens, pages)
        self._rows[s.row, :need] = pages

    def _pages_for(self, tokens: int) -> int:
        n = -(-tokens // self.page_size)
        if tokens < 0 or n > self.max_pages:
            raise ValueError(f"a sequence of {tokens} tokens (at most {self.max_pages * self.page_size})")
        return n

    def extend(self, seqs: Iterable[Hashable], tokens: int = 1) -> None:
        """Room for that many more tokens at the end of every sequence.  A page that the new tokens begin in and that other
        sequences hold too is copied first, in all layers (one launch for all of the call's)."""
        if tokens < 0:
            raise ValueError("tokens must not be negative")
        seqs = list(seqs)
        if len(set(seqs)) < len(seqs):
            raise ValueError("a sequence is named twice")
        if tokens == 0:
            return
        found = [self._get(x) for x in seqs]
        # (a page that all of its holders write to is copied for all but the last of them)
        left: Dict[int, int] = {}
        need, copied = 0, []
        for s in found:
            need += self._pages_for(s.length + tokens) - len(s.pages)
            own = True
            if s.length % self.page_size:
                page = s.pages[s.length // self.page_size]
                users = left.get(page, self._users[page])
                own = users == 1
                if not own:
                    left[page] = users - 1
                    need += 1
            copied.append(not own)
        if need > len(self._free):
            raise OutOfPages(f"{need} pages wanted, {len(self._free)} free")
        # copies first: where they fail nothing has changed
        pairs = [(s.pages[s.length // self.page_size], self._take()) for s, copy in zip(found, copied) if copy]
        if pairs:
            try:
                copy_pages(self.pool, pairs)
            except BaseException:
                for _, page in pairs:
                    self._users[page] = 0
                    heapq.heappush(self._free, page)
                raise
        made = iter(pairs)
        for s, copy in zip(found, copied):
            if copy:
                at = s.length // self.page_size
                old, new = next(made)
                self._users[old] -= 1
                self._spared -= 1
                s.pages[at] = self._rows[s.row, at] = new
            for at in range(len(s.pages), self._pages_for(s.length + tokens)):
                page = self._take()
                s.pages.append(page)
                self._rows[s.row, at] = page
            s.length += tokens

    def fork(self, parent: Hashable, child: Hashable) -> None:
        """`child` begins as `parent` is now and shares its pages."""
        p = self._get(parent)
        if child in self._seqs:
            raise ValueError(f"sequence {child!r} is in the cache")
        for page in p.pages:
            self._users[page] += 1
        self._spared += len(p.pages)
        s = self._seqs[child] = _Sequence(self._new_row(), p.length, list(p.pages))
        self._rows[s.row, :len(p.pages)] = p.pages

    def free(self, seq: Hashable) -> None:
        """Forgets a sequence; pages that no other holds are free again."""
        s = self._get(seq)
        del self._seqs[seq]
        self._free_rows.append(s.row)
        for page in s.pages:
            self._release(page)

    def _release(self, page: int) -> None:
        self._users[page] -= 1
        if self._users[page]:
            self._spared -= 1
        else:
            heapq.heappush(self._free, page)

    def truncate(self, seq: Hashable, length: int) -> None:
        """Takes tokens back from a sequence's end (drafted ones that were not accepted)."""
        s = self._get(seq)
        if not 0 <= length <= s.length:
            raise ValueError(f"a sequence of {s.length} tokens cut to {length}")
        keep = self._pages_for(length)
        for page in s.pages[keep:]:
            self._release(page)
        del s.pages[keep:]
        s.length = length

    def compact(self) -> int:
        """Moves the pages in use to the front of the pool, in all layers, and returns how many there are: every page from
        that number on is free, so pool[:, :n] is all there is to save or swap out."""
        used = [p for p in range(self.num_pages) if self._users[p]]
        n = len(used)
        holes = [p for p in range(n) if not self._users[p]]
        moves = dict(zip([p for p in used if p >= n], holes))
        if moves:
            copy_pages(self.pool, list(moves.items()))
            for s in self._seqs.values():
                if any(p in moves for p in s.pages):
                    s.pages[:] = [moves.get(p, p) for p in s.pages]
                    self._rows[s.row, :len(s.pages)] = s.pages
            for old, new in moves.items():
                self._users[new], self._users[old] = self._users[old], 0
            self._free = list(range(n, self.num_pages))
        return n

    # -- what the operators are given --------------------------------------------------------
    def slots(self, seq: Hashable, first: int = 0, last: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(positions, slots) of a sequence's tokens first .. last - 1, int64 on the device: what `append_kv` stores a prompt
        with.  They must not lie in pages that are shared (a fork's tokens are its parent's, too)."""
        s = self._get(seq)
        last = s.length if last is None else last
        if not 0 <= first <= last <= s.length:
            raise ValueError(f"tokens {first} to {last} of a sequence of {s.length}")
        t = np.arange(first, last, dtype=np.int64)
        pages = self._rows[s.row][t // self.page_size]
        for page in set(pages.tolist()):
            if self._users[page] > 1:
                raise ValueError("tokens in a page that other sequences hold too")
        both = torch.from_numpy(np.stack((t, pages.astype(np.int64) * self.page_size + t % self.page_size))).to(self.pool.device)
        return both[0], both[1]

    def batch(self, seqs: Sequence[Optional[Hashable]], width: Optional[int] = None, out: Optional[PagedBatch] = None) -> PagedBatch:
        """The step's tensors for these sequences, one row each, whose newest token is the one `extend` made room for.  None
        is a padded row: it stores nothing and its attention is zero.  width: pages of a table's row (default: as many
        as the longest needs).  out: a batch of as many rows to write over (a captured step reads it; width is its tables');
        what is returned has the tensors of `out` and `shared` of these rows."""
        rows = len(seqs)
        named = [x for x in seqs if x is not None]
        if len(set(named)) < len(named):
            raise ValueError("a sequence is named twice: its new token has one slot")
        found = [None if x is None else self._get(x) for x in seqs]
        if any(s is not None and not s.length for s in found):
            raise ValueError("a sequence without tokens has no newest one")
        need = max([len(s.pages) for s in found if s is not None], default=0)
        if out is not None:
            if out.lengths.shape[0] != rows:
                raise ValueError(f"out holds {out.lengths.shape[0]} rows, the batch has {rows}")
            width = out.block_tables.shape[1]
        width = max(need, 1) if width is None else width
        if width < need:
            raise ValueError(f"tables of {width} pages for a sequence that has {need}")
        host = np.zeros(16 * rows + 4 * rows * (width + 1), dtype=np.uint8)          # one transfer for all four
        place, slot = (host[8 * rows * i:8 * rows * (i + 1)].view(np.int64) for i in range(2))
        lengths = host[16 * rows:20 * rows].view(np.int32)
        tables = host[20 * rows:].view(np.int32).reshape(rows, width)
        at = np.fromiter((0 if s is None else s.row for s in found), np.int64, rows)
        length = np.fromiter((0 if s is None else s.length for s in found), np.int64, rows)
        real, last = length > 0, np.maximum(length - 1, 0)
        page = self._rows[at, last // self.page_size]
        if any(self._users[p] > 1 for p in page[real].tolist()):
            raise ValueError("a row's newest token lies in a page that other sequences hold too: extend makes it its own")
        place[:], lengths[:] = last, length
        slot[:] = np.where(real, page.astype(np.int64) * self.page_size + last % self.page_size, -1)
        columns = np.arange(min(width, self.max_pages))
        inside = columns < -(-length // self.page_size)[:, None]
        tables[:, :len(columns)] = np.where(inside, self._rows[at, :len(columns)], 0)
        held = sum([len(s.pages) for s in found if s is not None])
        shared = 2 * self._spared > held             # (no more than the whole cache's can be this batch's)
        if shared and rows > 1:
            distinct = np.zeros(self.num_pages, dtype=bool)
            distinct[tables[:, :len(columns)][inside]] = True
            shared = 2 * (held - int(distinct.sum())) > held
        dev = torch.from_numpy(host).to(self.pool.device)
        made = PagedBatch(dev[:8 * rows].view(torch.int64), dev[8 * rows:16 * rows].view(torch.int64),
                          dev[20 * rows:].view(torch.int32).view(rows, width), dev[16 * rows:20 * rows].view(torch.int32),
                          shared)
        if out is None:
            return made
        for to, t in zip(out[:4], made):
            to.copy_(t)
        return out._replace(shared=made.shared)
