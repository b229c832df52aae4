"""A paged key-value cache: pools on the device, bookkeeping of its pages on the host.

    cache = PagedCache(layers=32, pages=8192, page_size=16, kv_heads=8, head_dim=128, max_sequences=64)
    row = cache.open()
    rows, positions = cache.extend([row], [prompt.shape[0]])          # pages for the prompt
    for layer in range(32):
        q = cache.append(layer, k, v, rows, positions, frequencies=w, q=q)
    ...
    rows, positions = cache.extend([row], [1])                        # one decode step
    q = cache.append(layer, k, v, rows, positions, frequencies=w, q=q)
    out = cache.attend(layer, q, scale, rows=rows)

`PageBook` counts references: a fork shares its parent's pages, and the one page that both would write is copied when one of
them is extended. The bookkeeping is host arithmetic; the device sees one small copy of numbers and, where pages move, one
launch of `ops.copy_pages` over all layers. Nothing waits for the device. Calls of one cache belong on one stream, and those
that change the book outside captures; `append` and `attend` may be captured.
"""
from __future__ import annotations

import heapq
import operator

import numpy as np
import torch

from . import native, ops


class PagesExhausted(RuntimeError):
    """There are not enough free pages; nothing was changed."""


def _whole(value, label: str) -> int:
    try:
        return operator.index(value)
    except TypeError:
        raise ValueError(f'{label} must be an integer, got {value!r}') from None


class PageBook:
    """Which sequence owns which pages: tables, lengths, reference counts and free pages, all on the host.

    Methods that move or hand out pages return `(copies, updates)`: pairs (source page, destination page) to be copied
    before anything is written, and entries (row, column, page) of the tables that changed; those that take pages away return
    `updates`. An entry that a sequence does not hold is NO_PAGE, a number outside every pool: the operators store nothing there
    and report it.
    """

    NO_PAGE = -1

    def __init__(self, pages: int, page_size: int, max_sequences: int, max_pages_per_sequence: int):
        for label, value in (('pages', pages), ('page_size', page_size), ('max_sequences', max_sequences),
                             ('max_pages_per_sequence', max_pages_per_sequence)):
            if type(value) is not int or value < 1:
                raise ValueError(f'{label} must be a positive integer, got {value!r}')
        if max_pages_per_sequence * page_size >= 1 << 31 or max_sequences * max_pages_per_sequence >= 1 << 31:
            raise ValueError('a sequence holds fewer than 2^31 tokens, the tables fewer than 2^31 entries')
        self.page_size = page_size
        self.tables = np.full((max_sequences, max_pages_per_sequence), self.NO_PAGE, dtype=np.int32)
        self.lengths = np.zeros(max_sequences, dtype=np.int32)
        self.references = np.zeros(pages, dtype=np.int32)
        self._free_pages = list(range(pages))             # heaps: the lowest number first
        self._free_rows = list(range(max_sequences))
        self._open = np.zeros(max_sequences, dtype=bool)

    @property
    def free_pages(self) -> int:
        return len(self._free_pages)

    def _row(self, row: int) -> int:
        row = _whole(row, 'a row')
        if not 0 <= row < len(self._open) or not self._open[row]:
            raise ValueError(f'row {row!r} is not an open sequence')
        return row

    def _held(self, row: int) -> int:
        return -(-int(self.lengths[row]) // self.page_size)

    def _release(self, row: int, kept: int) -> list[tuple[int, int, int]]:
        """Takes the pages from column `kept` on away from a row: updates."""
        held = self._held(row)
        for page in self.tables[row, kept:held].tolist():
            self.references[page] -= 1
            if self.references[page] == 0:
                heapq.heappush(self._free_pages, page)
        self.tables[row, kept:held] = self.NO_PAGE
        return [(row, column, self.NO_PAGE) for column in range(kept, held)]

    def open(self) -> int:
        """A row for a new, empty sequence."""
        if not self._free_rows:
            raise PagesExhausted('every row is in use')
        row = heapq.heappop(self._free_rows)
        self._open[row] = True
        return row

    def close(self, row: int) -> list[tuple[int, int, int]]:
        """Frees a sequence: its row, and the pages that no fork shares: updates."""
        row = self._row(row)
        updates = self._release(row, 0)
        self.lengths[row] = 0
        self._open[row] = False
        heapq.heappush(self._free_rows, row)
        return updates

    def fork(self, row: int) -> tuple[int, list[tuple[int, int, int]]]:
        """A new sequence with the tokens of `row`, sharing its pages: (new row, updates)."""
        row = self._row(row)
        new = self.open()
        held = self._held(row)
        self.tables[new, :held] = self.tables[row, :held]
        self.references[self.tables[row, :held]] += 1     # a row holds a page once: no index twice
        self.lengths[new] = self.lengths[row]
        return new, [(new, column, int(self.tables[row, column])) for column in range(held)]

    def extend(self, rows, counts) -> tuple[list[tuple[int, int]], list[tuple[int, int, int]]]:
        """Makes room for counts[i] more tokens of rows[i] (each row once) and counts them in: (copies, updates)."""
        rows, counts = [self._row(row) for row in rows], [_whole(count, 'a count') for count in counts]
        if len(rows) != len(counts) or len(set(rows)) != len(rows) or any(count < 0 for count in counts):
            raise ValueError('extend takes one non-negative count for each of different rows')
        capacity = self.tables.shape[1] * self.page_size
        needed, shared = 0, {}
        for row, count in zip(rows, counts):
            length = int(self.lengths[row])
            if length + count > capacity:
                raise ValueError(f'row {row} would hold {length + count} tokens, the tables cover {capacity}')
            needed += -(-(length + count) // self.page_size) - self._held(row)
            if count and length % self.page_size:         # its last page is written again: by one owner only
                page = int(self.tables[row, length // self.page_size])
                shared[page] = shared.get(page, 0) + 1
        # of a page's owners all but the last that is left copy it
        needed += sum(min(writers, int(self.references[page]) - 1) for page, writers in shared.items())
        if needed > len(self._free_pages):
            raise PagesExhausted(f'{needed} pages needed, {len(self._free_pages)} free')
        copies, updates = [], []
        for row, count in zip(rows, counts):
            length = int(self.lengths[row])
            if count and length % self.page_size:
                column = length // self.page_size
                page = int(self.tables[row, column])
                if self.references[page] > 1:
                    own = self._take()
                    self.references[page] -= 1
                    copies.append((page, own))
                    self.tables[row, column] = own
                    updates.append((row, column, own))
            for column in range(self._held(row), -(-(length + count) // self.page_size)):
                self.tables[row, column] = page = self._take()
                updates.append((row, column, page))
            self.lengths[row] = length + count
        return copies, updates

    def _take(self) -> int:
        page = heapq.heappop(self._free_pages)
        self.references[page] = 1
        return page

    def truncate(self, row: int, length: int) -> list[tuple[int, int, int]]:
        """Forgets the tokens of `row` from `length` on (drafts that were not accepted): updates."""
        row, length = self._row(row), _whole(length, 'a length')
        if not 0 <= length <= self.lengths[row]:
            raise ValueError(f'row {row} holds {self.lengths[row]} tokens, cannot keep {length!r}')
        updates = self._release(row, -(-length // self.page_size))
        self.lengths[row] = length
        return updates

    def compact(self) -> tuple[list[tuple[int, int]], list[tuple[int, int, int]]]:
        """Moves the pages in use to the lowest numbers: (copies, updates). Sources and destinations are disjoint."""
        used = np.flatnonzero(self.references)
        sources, destinations = used[used >= len(used)], np.flatnonzero(self.references[:len(used)] == 0)
        if len(sources) == 0:
            return [], []
        moved = np.arange(len(self.references), dtype=np.int32)
        moved[sources] = destinations
        updates = []
        for row in np.flatnonzero(self._open).tolist():
            held = self._held(row)
            new = moved[self.tables[row, :held]]
            updates += [(row, int(column), int(new[column])) for column in np.flatnonzero(new != self.tables[row, :held])]
            self.tables[row, :held] = new
        self.references[destinations] = self.references[sources]
        self.references[sources] = 0
        self._free_pages = list(range(len(used), len(self.references)))
        return list(zip(sources.tolist(), destinations.tolist())), updates


class PagedCache:
    """Keys and values of all layers in pages, with the operators of `ops` on them.

    `pool` is [layers, 2, pages, kv_heads, page_size, head_dim]; `tables` and `lengths` are the device's copies of the book's,
    changed in place, so a captured step keeps reading the current ones. Entries of `tables` that no sequence holds are negative: an
    append to a closed row, or to a page that was not extended to or was given back, stores nothing and is reported. Within the pages
    that a row holds the positions of `extend` are the caller's to keep: a page may be shared with a fork.
    """

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, max_sequences: int,
                 max_pages_per_sequence: int | None = None, dtype: torch.dtype = torch.float16, device: torch.device | str | None = None):
        if dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise ValueError(f'dtype must be float32, float16 or bfloat16, got {dtype}')
        for label, value in (('layers', layers), ('kv_heads', kv_heads), ('head_dim', head_dim)):
            if type(value) is not int or value < 1:
                raise ValueError(f'{label} must be a positive integer, got {value!r}')
        if head_dim * dtype.itemsize % 16 or head_dim > 256:
            raise ValueError('a head has a multiple of 16 bytes and at most 256 elements')
        self.book = PageBook(pages, page_size, max_sequences, pages if max_pages_per_sequence is None else max_pages_per_sequence)
        device = torch.device('cuda' if device is None else device)
        with torch.inference_mode(False):   # tensors made under it could not be changed outside it
            self.pool = torch.empty((layers, 2, pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
            self.tables = torch.full(self.book.tables.shape, PageBook.NO_PAGE, dtype=torch.int32, device=device)
            self.lengths = torch.zeros(max_sequences, dtype=torch.int32, device=device)
        if self.pool.is_cuda:
            with torch.cuda.device(self.pool.device):
                native.call('dtn_device_status_prepare', torch.cuda.current_stream().cuda_stream)   # the word that reports go to exists before any capture

    def keys(self, layer: int) -> torch.Tensor:
        return self.pool[layer, 0]

    def values(self, layer: int) -> torch.Tensor:
        return self.pool[layer, 1]

    def _apply(self, copies, updates, rows, tokens=()) -> tuple[torch.Tensor, ...]:
        """Brings the device up to date: copies pages, then table entries and the lengths of `rows`. Returns `tokens` (integer
        arrays) on the device; everything travels in one copy."""
        width = self.tables.shape[1]
        lists = [np.array([c[0] for c in copies]), np.array([c[1] for c in copies]), np.array([u[0] * width + u[1] for u in updates]),
                 np.array([u[2] for u in updates]), np.asarray(rows, dtype=np.int32), self.book.lengths[rows], *tokens]
        sizes = [len(part) for part in lists]
        numbers = torch.from_numpy(np.concatenate([np.asarray(part, dtype=np.int32) for part in lists])).to(self.pool.device, non_blocking=True)   # pageable memory is staged before the call returns
        sources, destinations, places, pages, changed, lengths, *tokens = numbers.split(sizes)
        if copies:
            with torch.cuda.device_of(self.pool):   # the book has changed already: also where another device is current
                ops.copy_pages(self.pool, sources, destinations)
        if updates:
            self.tables.view(-1).index_copy_(0, places.long(), pages)
        if len(rows):
            self.lengths.index_copy_(0, changed.long(), lengths)
        return tuple(tokens)

    def _outside_captures(self) -> None:
        """The book would change once, its copy to the device be repeated by every replay."""
        if self.pool.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError('a cache is closed, forked, extended, truncated and compacted outside captures; append and attend may be captured')

    def open(self) -> int:
        """A row for a new, empty sequence."""
        return self.book.open()

    def close(self, row: int) -> None:
        """Frees a sequence: its row, and the pages that no fork shares."""
        self._outside_captures()
        self._apply([], self.book.close(row), [row])

    def fork(self, row: int) -> int:
        """A new sequence with the tokens of `row`. Its pages are shared until one of the two writes."""
        self._outside_captures()
        new, updates = self.book.fork(row)
        self._apply([], updates, [new])
        return new

    def extend(self, rows, counts) -> tuple[torch.Tensor, torch.Tensor]:
        """Makes room for counts[i] more tokens of rows[i] (each row once) and counts them in; raises PagesExhausted, and changes
        nothing, where pages are missing. Returns rows and positions of the new tokens (int32, in that order) for `append`.
        A shared page that would be written is copied first."""
        self._outside_captures()
        rows, counts = list(rows), list(counts)
        copies, updates = self.book.extend(rows, counts)
        rows, lengths = np.array(rows, dtype=np.int32), self.book.lengths[rows]
        if counts.count(1) == len(counts):                # a decode step
            return self._apply(copies, updates, rows, (rows, lengths - 1))
        counts = np.array(counts, dtype=np.int64)
        token_rows = np.repeat(rows, counts)
        positions = np.arange(len(token_rows)) + np.repeat(lengths - np.cumsum(counts), counts)   # the last token's is its row's length - 1
        return self._apply(copies, updates, rows, (token_rows, positions))

    def truncate(self, row: int, length: int) -> None:
        """Forgets the tokens of `row` from `length` on."""
        self._outside_captures()
        self._apply([], self.book.truncate(row, length), [row])

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers, in one launch; returns how many moved."""
        self._outside_captures()
        copies, updates = self.book.compact()
        if copies:
            self._apply(copies, updates, [])
        return len(copies)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, rows: torch.Tensor, positions: torch.Tensor, **rotation) -> torch.Tensor | None:
        """`ops.paged_append` into this layer: rows and positions from `extend`, frequencies, layout, amplitude, q, q_out as there."""
        return ops.paged_append(k, v, self.pool[layer, 0], self.pool[layer, 1], self.tables, rows, positions, **rotation)

    def attend(self, layer: int, q: torch.Tensor, scale: float, rows: torch.Tensor | None = None, window: int = 0,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """`ops.paged_attention` of one new token per sequence over this layer; q[i] belongs to sequence rows[i]."""
        return ops.paged_attention(q, self.pool[layer, 0], self.pool[layer, 1], self.tables, self.lengths, scale, rows=rows, window=window, out=out)
