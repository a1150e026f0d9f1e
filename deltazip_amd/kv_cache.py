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
from itertools import accumulate
from typing import Dict, Hashable, Iterable, List, NamedTuple, Optional, Sequence, Tuple

import numpy as np
import torch


from .paged import MAX_DIM, MAX_GROUPS, TableStep, copy_pages, extend_tables


class OutOfPages(RuntimeError):
    """The pool has too few free pages for the call; nothing was changed."""


class _Batch(NamedTuple):
    positions: torch.Tensor
    slots: torch.Tensor
    block_tables: torch.Tensor
    lengths: torch.Tensor
    shared: bool = False


class PagedBatch(_Batch):
    """What a step of one new token per row needs of the cache, on the device: the newest token's position and slot
    (int64 [rows]), the tables (int32 [rows, pages]) and lengths (int32 [rows], the new token counted); and, on the host, whether
    most of its rows' pages are another of its rows', too (for `paged_attention`, which takes no notice of it for one row; of
    one row: whether sharing spares the cache most of as many pages).  A captured step keeps what it was captured with.

    With several new tokens of a row, `starts` (int32 [rows + 1]) says where each row's begin among positions and slots; with prefixes that
    neighbouring rows share, `groups` (int32 [n + 1]) and `prefixes` (int32 [n]) say which: both as `prefix_attention` takes them.  (These three are
    no items of the tuple.)"""
    starts: Optional[torch.Tensor] = None
    groups: Optional[torch.Tensor] = None
    prefixes: Optional[torch.Tensor] = None

    def __new__(cls, positions, slots, block_tables, lengths, shared=False, starts=None, groups=None, prefixes=None):
        batch = super().__new__(cls, positions, slots, block_tables, lengths, shared)
        batch.starts, batch.groups, batch.prefixes = starts, groups, prefixes
        return batch

    def _replace(self, **changes) -> "PagedBatch":
        return PagedBatch(**{**self._asdict(), "starts": self.starts, "groups": self.groups, "prefixes": self.prefixes, **changes})


class _Sequence:
    __slots__ = ("row", "length", "pages", "running")

    def __init__(self, row: int, length: int, pages: List[int]) -> None:
        self.row, self.length, self.pages, self.running = row, length, pages, False


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
        self._runs: List["PagedRun"] = []           # not finished

    # -- what there is ---------------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def runs(self) -> Tuple["PagedRun", ...]:
        """Runs that are not finished, those among them that the caller has lost: their sequences come back with `finish`."""
        return tuple(self._runs)

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
        if s.running:
            raise ValueError(f"sequence {seq!r} is in a run: what it holds is known when that (one of `runs`) is finished")
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
        if any(s.running for s in self._seqs.values()):
            raise ValueError("a run holds pages of the cache: it has to be finished first")
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

    def batch(self, seqs: Sequence[Optional[Hashable]], width: Optional[int] = None, out: Optional[PagedBatch] = None,
              tokens: Optional[Sequence[int]] = None, prefix: bool = False) -> PagedBatch:
        """The step's tensors for these sequences, one row each, whose newest token is the one `extend` made room for.  None
        is a padded row: it stores nothing and its attention is zero.  width: pages of a table's row (default: as many
        as the longest needs).  out: a batch of as many rows to write over (a captured step reads it; width is its tables');
        what is returned has the tensors of `out` and `shared` of these rows.

        tokens: how many of each sequence's newest tokens are new (a prompt's, drafted ones; 0 of a padded row), of which the
        positions and slots follow each other.  prefix: neighbouring rows that hold the same pages at their beginning are told as groups
        (as many as there are rows, the last ones empty, so that `out` has the same shape)."""
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
            if tokens is not None or out.starts is not None:
                raise ValueError("out takes one new token of each row")
            if (out.groups is not None) != bool(prefix):
                raise ValueError("out must have been made with prefixes, or without, as the batch is")
            width = out.block_tables.shape[1]
        width = max(need, 1) if width is None else width
        if width < need:
            raise ValueError(f"tables of {width} pages for a sequence that has {need}")
        at = np.fromiter((0 if s is None else s.row for s in found), np.int64, rows)
        length = np.fromiter((0 if s is None else s.length for s in found), np.int64, rows)
        real = length > 0
        if tokens is None:
            n, position = rows, np.maximum(length - 1, 0)
        else:
            new = np.asarray(list(tokens), dtype=np.int64)
            if new.shape != (rows,) or (new < 0).any() or (new > length).any():
                raise ValueError("tokens must say of every row how many of its tokens are new, at most as many as it has")
            begin = np.concatenate((np.zeros(1, np.int64), np.cumsum(new)))
            n, row = int(begin[-1]), np.repeat(np.arange(rows), new)
            position = (length - new - begin[:-1])[row] + np.arange(n)
        groups = min(rows, MAX_GROUPS) if prefix else 0
        parts = [2 * n, 2 * n, rows, rows * width] + ([rows + 1] if tokens is not None else []) + ([groups + 1, groups] if prefix else [])     # words
        ends = list(accumulate(parts))
        host = np.zeros(ends[-1], dtype=np.int32)                                    # one transfer for all of it
        pieces = [host[e - p:e] for e, p in zip(ends, parts)]
        place, slot = pieces[0].view(np.int64), pieces[1].view(np.int64)
        lengths, tables = pieces[2], pieces[3].reshape(rows, width)
        page = self._rows[at if tokens is None else at[row], position // self.page_size]
        if any([self._users[p] > 1 for p in (page[real].tolist() if tokens is None else set(page.tolist()))]):
            raise ValueError("a row's newest token lies in a page that other sequences hold too: extend makes it its own")
        place[:], lengths[:] = position, length
        slot[:] = page.astype(np.int64) * self.page_size + position % self.page_size
        if tokens is None:
            slot[~real] = -1
        columns = np.arange(min(width, self.max_pages))
        inside = columns < -(-length // self.page_size)[:, None]
        tables[:, :len(columns)] = np.where(inside, self._rows[at, :len(columns)], 0)
        held = sum([len(s.pages) for s in found if s is not None])
        shared = 2 * self._spared > held             # (no more than the whole cache's can be this batch's)
        if shared and rows > 1:
            distinct = np.zeros(self.num_pages, dtype=bool)
            distinct[tables[:, :len(columns)][inside]] = True
            shared = 2 * (held - int(distinct.sum())) > held
        if tokens is not None:
            pieces[4][:] = begin
        if prefix:
            bounds, sizes = self._groups_of(tables[:, :len(columns)], inside.sum(1))
            pieces[-2][:] = rows
            pieces[-2][:len(bounds[:groups + 1])], pieces[-1][:len(sizes[:groups])] = bounds[:groups + 1], sizes[:groups]
        dev = torch.from_numpy(host).to(self.pool.device)
        made = [dev[e - p:e] for e, p in zip(ends, parts)]
        made = PagedBatch(made[0].view(torch.int64), made[1].view(torch.int64), made[3].view(rows, width), made[2], shared,
                          made[4] if tokens is not None else None, made[-2] if prefix else None, made[-1] if prefix else None)
        if out is None:
            return made
        for to, t in zip((*out[:4], out.groups, out.prefixes), (*made[:4], made.groups, made.prefixes)):
            if t is not None:
                to.copy_(t)
        return PagedBatch(*out[:4], made.shared, None, out.groups, out.prefixes)

    def _groups_of(self, tables: np.ndarray, used: np.ndarray) -> Tuple[List[int], List[int]]:
        """(rows where groups of neighbours begin and the last one ends, tokens that each group's rows have in common).  A row joins the group in front of
        it where that spares as many pages as the group spared without it; rows without pages between two of a group are among it."""
        alive = np.flatnonzero(used)
        columns = np.arange(tables.shape[1])
        rows, pages = tables[alive], used[alive]
        same = (rows[1:] == rows[:-1]) & (columns < np.minimum(pages[1:], pages[:-1])[:, None])
        common = np.where(same.all(1), len(columns), same.argmin(1)).tolist() if len(alive) > 1 else []        # pages, with the one in front
        bounds, sizes, first = [0], [], 0

        def close(end: int, pages: int) -> None:
            if end == bounds[-1]:
                return
            if pages == 0 and sizes and sizes[-1] == 0:
                bounds[-1] = end
            else:
                sizes.append(pages * self.page_size)
                bounds.append(end)

        while first < len(alive):
            last, cut = first + 1, 0
            while last < len(alive):
                c = min(cut, common[last - 1]) if cut else common[last - 1]
                if not c or c * (last - first) < cut * (last - first - 1):
                    break
                last, cut = last + 1, c
            close(int(alive[first]), 0)
            close(int(alive[last - 1]) + 1, cut)
            first = last
        close(len(used), 0)
        return bounds, sizes

    # -- steps that the device goes by itself ---------------------------------------------------
    def run(self, seqs: Sequence[Optional[Hashable]], steps: int, prefix: bool = False) -> "PagedRun":
        """Up to `steps` steps of one token per row without the host: the pages that they may need are set aside (`OutOfPages`: too few), and
        tables, lengths, positions and slots go on on the device.  Until it is finished these sequences are the run's.
        None is a padded row.  prefix as for `batch`."""
        if steps < 1:
            raise ValueError("steps must be positive")
        named = [x for x in seqs if x is not None]
        found = [self._get(x) for x in named]
        before = [s.length for s in found]
        if len(set(named)) < len(named):
            raise ValueError("a sequence is named twice")
        self.extend(named, steps)                       # (pages that others hold too are copied)
        free: List[int] = []
        for s, n in zip(found, before):
            keep = -(-n // self.page_size)
            free += s.pages[keep:]
            del s.pages[keep:]
            s.length = n
        try:
            return PagedRun(self, list(seqs), steps, free, prefix)
        except BaseException:
            for page in free:
                self._release(page)
            raise


class PagedRun:
    """Steps of a batch whose tables, lengths and free pages stay on the device (`PagedKVCache.run`):

        with cache.run(seqs, steps=64) as run:                         # (finished at its end, whatever happens in it)
            for _ in range(64):
                logits = model.paged_step(tokens, cache, run.step())   # or captured once and replayed

    `step` makes room for each row's next token and returns the batch of it, the same tensors every time; `counts` (int32 [rows]: 1, or 0
    of a row that gets no more tokens) may be written between steps.  A step that needs more pages than were set aside stores
    nothing, of any row, and is reported through the status word.  A captured step is not replayed once the run is finished: the pages that it writes to may be
    others'."""

    def __init__(self, cache: PagedKVCache, seqs: List[Optional[Hashable]], steps: int, free: List[int], prefix: bool) -> None:
        self.cache, self._seqs = cache, seqs
        found = [None if x is None else cache._get(x) for x in seqs]
        rows = len(seqs)
        lengths = np.fromiter((0 if s is None else s.length for s in found), np.int32, rows)
        width = max([-(-int(n) // cache.page_size) for n in lengths + steps * (lengths >= 0)], default=1) if rows else 1
        width = min(max(width, 1), cache.max_pages)
        tables = np.zeros((rows, width), dtype=np.int32)
        for r, s in enumerate(found):
            if s is not None:
                tables[r, :len(s.pages)] = s.pages
        used = -(-lengths.astype(np.int64) // cache.page_size)
        real = np.fromiter((s is not None for s in found), np.int32, rows)
        host = np.concatenate((lengths, real, np.zeros(1, np.int32), np.asarray(free, dtype=np.int32), tables.ravel()))
        dev = torch.from_numpy(host).to(cache.pool.device)
        self._lengths, self.counts, self._taken = dev[:rows], dev[rows:2 * rows], dev[2 * rows:2 * rows + 1]
        self._free, self._tables = dev[2 * rows + 1:2 * rows + 1 + len(free)], dev[2 * rows + 1 + len(free):].view(rows, width)
        self._out = TableStep(self._lengths, self._taken, torch.empty(rows + 1, dtype=torch.int32, device=dev.device),
                              *torch.empty((2, rows), dtype=torch.int64, device=dev.device))
        self._pages, self._finished = free, False
        groups = prefixes = None
        shared = False
        if rows:
            # (the page that a row's tokens go on in is its own: no group has it)
            bounds, sizes = cache._groups_of(tables, used)
            holders = [int(np.count_nonzero(used[a:b])) for a, b in zip(bounds, bounds[1:])]
            shared = 2 * sum(n // cache.page_size * (h - 1) for h, n in zip(holders, sizes) if n) > int(used.sum())
            if prefix:
                n = min(len(sizes), MAX_GROUPS)
                both = torch.from_numpy(np.asarray(bounds[:n + 1] + sizes[:n], dtype=np.int32)).to(cache.pool.device)
                groups, prefixes = both[:n + 1], both[n + 1:]
        self._batch = PagedBatch(self._out.positions, self._out.slots, self._tables, self._lengths, shared, None, groups, prefixes)
        for s in found:
            if s is not None:
                s.running = True
        cache._runs.append(self)

    def __enter__(self) -> "PagedRun":
        return self

    def __exit__(self, *error) -> None:
        self.finish()

    def step(self) -> PagedBatch:
        if self._finished:
            raise ValueError("the run is finished")
        extend_tables(self._tables, self._lengths, self.counts, self._free, self._taken, self.cache.page_size, out=self._out)
        return self._batch

    def finish(self) -> None:
        """Gives the cache its sequences back, as long as they have become, and the pages that were not needed.  Waits for the device: for steps and
        replays on every stream."""
        if self._finished:
            return
        if self.cache.pool.is_cuda:
            torch.cuda.synchronize(self.cache.pool.device)
        lengths, tables = self._lengths.cpu().numpy(), self._tables.cpu().numpy()
        cache, taken = self.cache, set()
        for r, x in enumerate(self._seqs):
            if x is None:
                continue
            s = cache._seqs[x]
            s.length = int(lengths[r])
            s.pages[:] = tables[r, :-(-s.length // cache.page_size)].tolist()
            cache._rows[s.row, :len(s.pages)] = s.pages
            taken.update(s.pages)
            s.running = False
        for page in self._pages:
            if page not in taken:
                cache._release(page)
        cache._runs.remove(self)
        self._finished = True
