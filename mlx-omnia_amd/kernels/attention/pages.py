"""A KV cache of pages, shared by the sequences that have rows in common.

Beside the one-sequence caches (cache.py, after core/cache/kv.py): the rows of all sequences
and layers lie in one pool of pages,

    keys, values [layers, pages, kv_heads, page_rows, head_dim]

and a sequence is a row of page ids, the same ids in every layer: `fork` gives the children
the parent's full pages to share and copies only the page that is still being filled, `free`
hands back the pages that nobody else holds, `compact` moves what is in use to the front of
the pool. Which page is whose is decided on the host, which holds the counts; `tables` and
`lengths` say the same on the device, where the kernels read them, and change in the order of
the current stream with what the kernels do. The host's arrays change once the device's part
has been launched: a call that is refused, or whose launch fails, leaves them as they were (a
compaction of many pages keeps what it has moved by then).

    cache = PagedKVCache.empty(layers, pages, page_rows, kv_heads, head_dim, sequences=64, rows=32768)
    prompt = cache.open()
    one = cache.batch([prompt], tokens=900)       # a step of 900 tokens of one sequence
    ...each layer's BatchAttentionStep with `one`...
    cache.advance(one)
    answers = cache.fork(prompt, 16)
    step = cache.batch(answers)                   # steps of one token each
    ...each layer..., cache.advance(step), and again
    cache.free(answers)

A page id that is handed out is the lowest one free, so the same calls give the same tables.
One thread at a time calls a cache, and the steps over it; the kernels of its calls run on
streams that are ordered among themselves, as with any tensor that is written.
"""

from __future__ import annotations

from array import array
from collections.abc import Sequence

import numpy as np
import torch

from ...runtime import ops
from .._device import hip_device

PAGE_ROWS = (16, 32, 64, 128, 256)
TILE_ROWS = 128   # query rows of one piece at most (`omnia_attention_batch`'s tiles)


def _capturing(device: torch.device) -> bool:
    return device.type == "cuda" and torch.cuda.is_current_stream_capturing()


class PagedBatch:
    """The sequences of a step and how many new tokens each has, as the kernels read them.

    Made by `PagedKVCache.batch` and kept as long as the same sequences step on: `advance`
    moves it along. Token t of the step's packed rows is the `token_map[t, 1]`-th new one of
    sequence `token_map[t, 0]`; a sequence's tokens lie together, in the order of
    `sequences`. The first `prefix` rows are the same pages for all of them."""

    def __init__(self, cache: "PagedKVCache", sequences: list[int], tokens: list[int], prefix: int) -> None:
        self.cache = cache
        self.sequences, self.tokens = tuple(sequences), tuple(tokens)
        self.total = sum(tokens)
        self.prefix = prefix
        self.index = np.asarray(sequences, dtype=np.int64)
        self.counts = np.asarray(tokens, dtype=np.int64)
        self.ends = np.cumsum(self.counts)
        self.generation = cache._generation[self.index].copy()
        self.clock = -1               # the cache's, at which the step's pages were made sure of
        self.reach = 0                # the most rows that captured steps were prepared for
        device = cache.keys.device
        whose = np.repeat(self.index, self.counts)
        which = np.arange(self.total) - np.repeat(self.ends - self.counts, self.counts)
        upload = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(device)  # noqa: E731
        self.token_map = upload(np.stack([whose, which], axis=1))
        self.chosen, self.rows = upload(self.index), upload(self.counts)
        self.epoch = cache._epoch     # at which its sequences were last seen to be the same
        self.last = 0                 # the most rows a sequence has in the step at hand
        self.plans: dict = {}         # what a layer's binding laid out for the batch
        self.captured: list = []      # of those, the ones that graphs read
        self.now = None               # and each of them
        self._tiles: dict[int, torch.Tensor] = {}
        self._totals: dict[int, tuple[int, int]] = {}

    def tiles(self, group: int) -> torch.Tensor:
        """Runs of at most TILE_ROWS query rows of one sequence, with `group` rows a token: (first
        row, past the last, sequence, which of its new tokens the first row is of)."""
        held = self._tiles.get(group)
        if held is None:
            if _capturing(self.cache.keys.device):
                raise ValueError("a batch's first step cannot be captured: call prepare_capture first")
            runs = []
            for s, end, count in zip(self.sequences, self.ends * group, self.counts * group):
                first = np.arange(end - count, end, TILE_ROWS)
                runs.append(np.stack([first, np.minimum(first + TILE_ROWS, end), np.full_like(first, s),
                                      (first - (end - count)) // group], axis=1))
            flat = np.ascontiguousarray(np.concatenate(runs), dtype=np.int32)
            held = self._tiles[group] = torch.from_numpy(flat).to(self.cache.keys.device)
        return held


    def own_total(self, group: int) -> int:
        """The rows past the shared ones of every tile's sequence, in the step at hand."""
        held = self._totals.get(group)
        if held is None or held[0] != self.clock:
            tiles = -(-self.counts * group // TILE_ROWS)
            held = self._totals[group] = self.clock, int(((self.now - self.prefix) * tiles).sum())
        return held[1]


class PagedKVCache:
    def __init__(self, keys: torch.Tensor, values: torch.Tensor, *, sequences: int | None = None,
                 rows: int | None = None, tables: np.ndarray | None = None, lengths: np.ndarray | None = None,
                 opened: Sequence[int] | None = None) -> None:
        """A cache over the pool `keys`, `values`. Either empty, for at most `sequences` open
        at once of at most `rows` rows each, or as it was left: `tables` [sequences, width]
        (-1 for no page), `lengths` [sequences], and the sequences that are `opened`."""
        if keys.dim() != 5 or keys.shape != values.shape or keys.dtype != values.dtype:
            raise ValueError("PagedKVCache: keys and values must both be [layers, pages, kv_heads, page_rows, head_dim]")
        if keys.device != values.device or not (keys.is_contiguous() and values.is_contiguous()):
            raise ValueError("PagedKVCache: keys and values must be contiguous, on one device")
        layers, pages, kv_heads, page_rows, head_dim = keys.shape
        if page_rows not in PAGE_ROWS or head_dim % 8 or min(layers, pages, kv_heads, head_dim) < 1:
            raise ValueError(f"PagedKVCache: pages of {PAGE_ROWS} rows, heads of a multiple of 8, not {tuple(keys.shape)}")
        if (tables is None) == (sequences is None or rows is None):
            raise ValueError("PagedKVCache: give sequences and rows, or tables, lengths and opened")
        if tables is None:
            if lengths is not None or opened is not None or sequences < 1 or rows < 1:
                raise ValueError("PagedKVCache: sequences and rows must be positive, without lengths or opened")
            tables = np.full((sequences, -(-rows // page_rows)), -1, dtype=np.int32)
            lengths, opened = np.zeros(sequences, dtype=np.int32), ()
        elif lengths is None or opened is None:
            raise ValueError("PagedKVCache: tables need lengths and opened")
        self.keys, self.values = keys, values
        self._tables = np.array(tables, dtype=np.int32, order="C")
        self._rows = np.array(lengths, dtype=np.int64)
        slots = range(len(self._tables))
        if len(set(opened)) != len(opened) or any(s not in slots for s in opened):
            raise ValueError("PagedKVCache: opened names other sequences than the tables, or one twice")
        self._open = np.zeros(len(self._tables), dtype=np.uint8)
        self._open[list(opened)] = 1
        self._held = (self._tables >= 0).sum(axis=1)
        self._check_tables()
        self._refs = np.zeros(pages, dtype=np.int64)
        np.add.at(self._refs, self._tables[self._tables >= 0], 1)
        spare = (np.arange(self._tables.shape[1]) >= -(-self._rows[:, None] // page_rows)) & (self._tables >= 0)
        if (self._refs[self._tables[spare]] > 1).any():
            raise ValueError("PagedKVCache: a page past a sequence's rows is another sequence's as well")
        self._generation = np.zeros(len(self._tables), dtype=np.int64)   # of a slot: whose it is
        self._epoch = 0                                                  # of them all
        self._clock = 0                                                  # turns as sequences grow
        self.tables = torch.from_numpy(self._tables.copy()).to(keys.device)
        self.lengths = torch.from_numpy(self._rows.astype(np.int32)).to(keys.device)
        self._bind()

    def _bind(self) -> None:
        """The library's view of the pool, the tables and the host's arrays: on a HIP device."""
        pool = None
        if hip_device(self.keys):
            pool = ops.PagePool(self.keys, self.values, self.tables, self.lengths)
            pool.keep(self._tables, self._rows, self._held, self._refs, self._generation, self._open)
        self._pool, self._kind = pool, (self.keys.shape, self.keys.dtype)

    def _library(self) -> None:
        """The same again where a tensor lies elsewhere by now: its identity does not say so
        (`.data`, as a module that is moved sets it)."""
        if self._kind != (self.keys.shape, self.keys.dtype):
            raise ValueError("PagedKVCache: the pool is of another shape or kind than it was (resize changes it)")
        tensors = self.keys, self.values, self.tables, self.lengths
        if self._pool.addresses != [t.data_ptr() for t in tensors]:
            if not hip_device(*tensors):
                raise ValueError("PagedKVCache: the pool and its tables have left their device")
            self._bind()

    def _check_tables(self) -> None:
        tables, width = self._tables, self._tables.shape[1] if self._tables.ndim == 2 else 0
        if tables.ndim != 2 or width < 1 or self._rows.shape != (len(tables),):
            raise ValueError("PagedKVCache: tables must be [sequences, width] and lengths [sequences]")
        if width * self.page_rows >= 1 << 30:
            raise ValueError("PagedKVCache: a sequence holds fewer than 2^30 rows")
        if tables.max() >= self.pages or tables.min() < -1:
            raise ValueError("PagedKVCache: a table names a page outside the pool")
        first = np.arange(width)[None] < self._held[:, None]
        if not (first == (tables >= 0)).all():
            raise ValueError("PagedKVCache: a table's pages must come first, without gaps")
        if (self._rows < 0).any() or (self._rows > self._held * self.page_rows).any():
            raise ValueError("PagedKVCache: a length outside its sequence's pages")
        if (self._held[self._open == 0] > 0).any():
            raise ValueError("PagedKVCache: a sequence that is not open holds pages")
        for row in tables:
            if len(np.unique(row[row >= 0])) != (row >= 0).sum():
                raise ValueError("PagedKVCache: a sequence names one page twice")

    @classmethod
    def empty(cls, layers: int, pages: int, page_rows: int, kv_heads: int, head_dim: int, *, sequences: int,
              rows: int, dtype=torch.bfloat16, device=None) -> "PagedKVCache":
        shape = (layers, pages, kv_heads, page_rows, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                   sequences=sequences, rows=rows)

    @property
    def pages(self) -> int:
        return self.keys.shape[1]

    @property
    def page_rows(self) -> int:
        return self.keys.shape[3]

    @property
    def free_pages(self) -> int:
        return int((self._refs == 0).sum())

    def rows(self, sequence: int) -> int:
        """Rows that the sequence holds."""
        self._known([sequence])
        return int(self._rows[sequence])

    def pages_of(self, sequence: int) -> list[int]:
        """The pages that the sequence lies on, the reserved ones included."""
        self._known([sequence])
        return self._tables[sequence, : self._held[sequence]].tolist()

    # What the device is told ---------------------------------------------------------------

    def _refuse_capture(self, what: str) -> None:
        if _capturing(self.keys.device):
            raise ValueError(f"PagedKVCache: {what} cannot be captured (a replay would not repeat the host's part)")
        if self._pool is not None:
            self._library()
            self._pool.stream()   # raises where another device is current, ahead of any change

    def _edit(self, edits: list[int]) -> None:
        """Edits (kind, sequence, a, b), one after the other."""
        if not edits:
            return
        if self._pool is not None:
            self._pool.edit(array("i", edits))
            return
        for kind, s, a, b in zip(*(edits[i::4] for i in range(4))):
            if kind == ops.PAGES_ENTRY:
                self.tables[s, a] = b
            elif kind == ops.PAGES_LENGTH:
                self.lengths[s] = a
            else:
                self.tables[s], self.lengths[s] = -1, 0

    @staticmethod
    def _entries(sequence: int, first: int, pages) -> list[int]:
        """The edits that make `pages` a sequence's entries from `first` on."""
        return [n for i, page in enumerate(pages, first) for n in (ops.PAGES_ENTRY, sequence, i, page)]

    def _copy(self, moves: list[tuple[int, int, int]]) -> None:
        if not moves:
            return
        if self._pool is not None:
            self._pool.copy(moves)
            return
        for pool in (self.keys, self.values):
            for source, target, rows in moves:
                pool[:, target, :, :rows] = pool[:, source, :, :rows]

    # Pages --------------------------------------------------------------------------------

    def _known(self, sequences: Sequence[int]) -> None:
        for s in sequences:
            if not 0 <= s < len(self._open) or not self._open[s]:
                raise ValueError(f"PagedKVCache: sequence {s} is not open")

    def _renew(self, sequences) -> None:
        """The sequences are others now: batches of the ones before are refused."""
        self._generation[sequences] += 1
        self._epoch += 1

    def _take(self, count: int) -> np.ndarray:
        """The lowest `count` free pages, still free."""
        found = (self._refs == 0).nonzero()[0][:count]
        if len(found) < count:
            raise ValueError(f"PagedKVCache: {count} more pages are needed, {len(found)} of {self.pages} are free")
        return found

    def _slots(self, count: int) -> list[int]:
        """The lowest `count` sequences that are not open, still not."""
        closed = (self._open == 0).nonzero()[0]
        if len(closed) < count:
            raise ValueError(f"PagedKVCache: {count} more sequences are asked for, {len(closed)} of "
                             f"{len(self._open)} are not open")
        return closed[:count].tolist()

    def _begin(self, slots: list[int]) -> None:
        self._open[slots] = 1
        self._renew(slots)

    def _pages_for(self, rows: int) -> int:
        pages = -(-int(rows) // self.page_rows)
        if pages > self._tables.shape[1]:
            raise ValueError(f"PagedKVCache: a sequence holds at most {self._tables.shape[1] * self.page_rows} rows, "
                             f"not {rows}")
        return pages

    def open(self, rows: int = 0) -> int:
        """A new sequence, empty or of `rows` rows that the caller writes into the pool itself."""
        self._refuse_capture("opening a sequence")
        if rows < 0:
            raise ValueError("PagedKVCache: a sequence of fewer than no rows")
        if self._pool is not None:   # the same, beside the launch
            s = self._pool.open(int(rows))
            self._epoch += 1
            return s
        pages = self._pages_for(rows)
        slots = self._slots(1)
        s, fresh = slots[0], self._take(pages)
        self._begin(slots)
        self._refs[fresh] = 1
        self._tables[s, :pages] = fresh
        self._held[s], self._rows[s] = pages, rows
        self._edit(self._entries(s, 0, fresh.tolist()) + ([ops.PAGES_LENGTH, s, rows, 0] if rows else []))
        return s

    def _reserve(self, index: np.ndarray, rows: np.ndarray) -> None:
        """Pages for `rows` rows of each sequence, and one of its own where it writes next."""
        size = self.page_rows
        need = -(-rows // size)
        if (need > self._tables.shape[1]).any():
            self._pages_for(int(rows.max()))   # raises
        now = self._rows[index]
        more = np.maximum(need - self._held[index], 0)
        # A partly filled page that another sequence holds as well is copied before it is written.
        at = now // size
        cut = np.flatnonzero((now % size > 0) & (rows > now))
        shared = [i for i in cut if self._refs[self._tables[index[i], at[i]]] > 1]
        if not shared and not more.any():
            return
        self._refuse_capture("reserving pages")
        # Of the holders of one such page the last in turn keeps it.
        holders = {}
        for i in shared:
            holders.setdefault(int(self._tables[index[i], at[i]]), []).append(i)
        copied = [i for page, who in holders.items() for i in (who[:-1] if len(who) == self._refs[page] else who)]
        fresh = self._take(len(copied) + int(more.sum()))
        entries, moves = [], []
        for i, page in zip(copied, fresh.tolist()):
            s, old = int(index[i]), int(self._tables[index[i], at[i]])
            moves.append((old, page, int(now[i] % size)))
            entries.append((s, int(at[i]), page))
        rest = iter(fresh[len(copied):].tolist())
        for i in np.flatnonzero(more):
            s = int(index[i])
            entries += [(s, entry, next(rest)) for entry in range(self._held[s], self._held[s] + int(more[i]))]
        self._copy(moves)
        self._edit([n for entry in entries for n in (ops.PAGES_ENTRY, *entry)])
        for old, _, _ in moves:
            self._refs[old] -= 1
        self._refs[fresh] = 1
        for s, entry, page in entries:
            self._tables[s, entry] = page
        self._held[index] += more

    def reserve(self, sequence: int, rows: int) -> None:
        """Pages for the sequence up to `rows` rows, ahead of the steps that fill them."""
        self._known([sequence])
        self._pages_for(rows)
        self._reserve(np.asarray([sequence]), np.asarray([rows]))

    def fork(self, sequence: int, count: int = 1, *, share: bool = True) -> list[int]:
        """`count` new sequences with the rows of this one, as many as the host has counted: its
        full pages shared, the last, partly filled one copied for each; with `share=False` every
        page copied."""
        self._refuse_capture("forking")
        self._known([sequence])
        if count < 0:
            raise ValueError("PagedKVCache: fewer than no forks")
        if count > len(self._open):
            self._slots(count)   # raises
        if share and self._pool is not None:   # the same, beside the launch: 26 us a fork and a free here
            kids = self._pool.begin(int(sequence), int(count))
            self._epoch += 1
            return kids
        size, rows = self.page_rows, int(self._rows[sequence])
        full, rest = divmod(rows, size)
        if not share:
            full, rest = 0, rows
        each = -(-rest // size)
        kids, fresh = self._slots(count), self._take(each * count)
        if not count:
            return kids
        parent = self._tables[sequence].tolist()
        lines = fresh.reshape(count, each).tolist()
        used = [size] * (each - 1) + [rest - size * (each - 1)]
        self._copy([(page, to, n) for line in lines for page, to, n in zip(parent[full:], line, used)])
        self._edit([n for kid, line in zip(kids, lines) for n in self._entries(kid, 0, parent[:full] + line)
                    + [ops.PAGES_LENGTH, kid, rows, 0]])
        self._refs[fresh] = 1
        self._refs[parent[:full]] += count
        self._begin(kids)
        for kid, line in zip(kids, lines):
            self._tables[kid, : full + each] = parent[:full] + line
        self._held[kids] = full + each
        self._rows[kids] = rows
        return kids

    def free(self, sequences: Sequence[int] | int) -> None:
        """Close sequences; the pages that no other one holds are free again."""
        self._refuse_capture("freeing")
        gone = [int(s) for s in ([sequences] if isinstance(sequences, (int, np.integer)) else sequences)]
        if len(set(gone)) != len(gone):
            raise ValueError("PagedKVCache: a sequence to free is named twice")
        self._known(gone)
        if not gone:
            return
        if self._pool is not None:
            self._pool.end(gone)
            self._epoch += 1
            return
        held = self._tables[gone]
        self._refs -= np.bincount(held[held >= 0], minlength=len(self._refs))
        self._tables[gone] = -1
        self._open[gone] = 0
        self._held[gone] = 0
        self._rows[gone] = 0
        self._renew(gone)
        self._edit([n for s in gone for n in (ops.PAGES_CLEAR, s, 0, 0)])

    def truncate(self, sequence: int, rows: int) -> None:
        """Drop the sequence's rows from `rows` on (a rejected guess), and the pages past them."""
        self._refuse_capture("truncating")
        self._known([sequence])
        if not 0 <= rows <= self._rows[sequence]:
            raise ValueError(f"PagedKVCache: sequence {sequence} holds {self._rows[sequence]} rows, not {rows}")
        keep = self._pages_for(rows)
        gone = int(self._held[sequence]) - keep
        self._edit(self._entries(sequence, keep, [-1] * gone) + [ops.PAGES_LENGTH, sequence, rows, 0])
        self._refs[self._tables[sequence, keep : self._held[sequence]]] -= 1
        self._tables[sequence, keep:] = -1
        self._held[sequence], self._rows[sequence] = keep, rows
        self._renew(sequence)

    def compact(self) -> int:
        """Move the pages in use to the front of the pool, each that lies behind them to the
        lowest free one in turn; how many are in use. Sequences and batches stay what they
        are."""
        self._refuse_capture("compacting")
        if self._pool is not None:
            return self._pool.compact()
        used = np.flatnonzero(self._refs > 0)
        live = len(used)
        source, target = used[used >= live], np.flatnonzero(self._refs[:live] == 0)
        if len(source):
            names = np.arange(self.pages + 1, dtype=np.int32)   # the last for -1
            names[-1], names[source] = -1, target
            self._copy([(a, b, self.page_rows) for a, b in zip(source.tolist(), target.tolist())])
            self._tables[:] = names[self._tables]
            self._refs[target], self._refs[source] = self._refs[source], 0
            self.tables.copy_(torch.from_numpy(self._tables))
        return live

    def resize(self, pages: int) -> None:
        """A pool of `pages` pages, the first ones' contents kept: larger, or smaller by pages
        that are free (`compact` first). The tensors are new ones: a captured step has to be
        captured again."""
        self._refuse_capture("resizing")
        used = np.flatnonzero(self._refs > 0)
        if pages < 1 or (len(used) and used[-1] >= pages):
            raise ValueError(f"PagedKVCache: page {used[-1] if len(used) else 0} is in use, {pages} pages are too few")
        kept = min(pages, self.pages)
        pools = []
        for old in (self.keys, self.values):
            pool = old.new_zeros((old.shape[0], pages, *old.shape[2:]))
            pool[:, :kept] = old[:, :kept]
            pools.append(pool)
        refs = np.zeros(pages, dtype=np.int64)
        refs[:kept] = self._refs[:kept]
        (self.keys, self.values), self._refs = pools, refs
        self._bind()

    # Steps --------------------------------------------------------------------------------

    def batch(self, sequences: Sequence[int], tokens: int | Sequence[int] = 1) -> PagedBatch:
        """The steps of these sequences with so many new tokens each (or each its own number).
        The rows that all of them share are found here, from the tables; what only some of them
        share each reads for itself, so groups that share nothing step as batches of their own."""
        self._refuse_capture("making a batch")
        chosen = [int(s) for s in sequences]
        if not chosen or len(set(chosen)) != len(chosen):
            raise ValueError("PagedKVCache: a batch names at least one sequence, each once")
        self._known(chosen)
        counts = [int(tokens)] * len(chosen) if isinstance(tokens, (int, np.integer)) else [int(n) for n in tokens]
        if len(counts) != len(chosen) or min(counts) < 1:
            raise ValueError("PagedKVCache: every sequence of a batch has at least one new token")
        shared = 0
        if len(chosen) > 1:
            full = int(self._rows[chosen].min()) // self.page_rows
            same = (self._tables[chosen, :full] == self._tables[chosen[0], :full]).all(axis=0)
            shared = full if same.all() else int(np.argmin(same))
        return PagedBatch(self, chosen, counts, shared * self.page_rows)

    def _current(self, batch: PagedBatch) -> None:
        if batch.cache is not self:
            raise ValueError("PagedKVCache: the batch belongs to another cache")
        if batch.epoch != self._epoch:
            if not np.array_equal(self._generation[batch.index], batch.generation):
                raise ValueError("PagedKVCache: a sequence of the batch was freed or truncated; make a new batch")
            batch.epoch = self._epoch

    def ready(self, batch: PagedBatch) -> int:
        """Make sure of the pages of the batch's step; the most rows any of its sequences has
        then, or may have in the replays that were prepared for, if it is being captured."""
        self._current(batch)
        if batch.clock != self._clock:
            rows = self._rows[batch.index] + batch.counts
            self._reserve(batch.index, rows)
            batch.clock, batch.last, batch.now = self._clock, int(rows.max()), rows
        if self._pool is None or not torch.cuda.is_current_stream_capturing():
            return batch.last
        if batch.reach < batch.last:
            raise ValueError("a batch's step is captured after prepare_capture has reserved what its replays reach")
        return batch.reach

    def prepare_capture(self, batch: PagedBatch, steps: int) -> int:
        """Reserve the pages of the batch's next `steps` steps, before a step and its `advance`
        are captured; the most rows a sequence has after them. Replays past that are outside
        the contract (their rows are not stored, nor those past the reach attended). The batch
        holds what the graph reads and lives as long."""
        self._current(batch)
        if steps < 1:
            raise ValueError("PagedKVCache: a captured step is replayed at least once")
        rows = self._rows[batch.index] + steps * batch.counts
        self._reserve(batch.index, rows)
        batch.reach = int(rows.max())
        self.ready(batch)
        return batch.reach

    def advance(self, batch: PagedBatch) -> None:
        """The step's tokens are rows of their sequences now: once a step, after every layer.
        Captured, it moves the device's lengths at each replay, and `account` the host's."""
        self._current(batch)
        counted = not _capturing(self.keys.device)
        if counted:
            self._grown(batch, 1)   # raises where the pages do not hold them
        if self._pool is not None:
            ops.pages_advance(self.lengths, batch.chosen, batch.rows)
        else:
            self.lengths[batch.chosen.long()] += batch.rows
        if counted:
            self.account(batch, 1)

    def account(self, batch: PagedBatch, steps: int) -> None:
        """Count `steps` steps of the batch that the device has taken in replays: before the next
        call that names its sequences, since the host goes by what it has counted (a fork made
        ahead of it has the rows of before the replays)."""
        self._current(batch)
        self._rows[batch.index] = self._grown(batch, steps)
        self._clock += 1

    def _grown(self, batch: PagedBatch, steps: int) -> np.ndarray:
        """The rows of the batch's sequences `steps` steps on."""
        rows = self._rows[batch.index] + steps * batch.counts
        if steps < 0 or (rows > self._held[batch.index] * self.page_rows).any():
            raise ValueError("PagedKVCache: more steps than the pages hold")
        return rows
