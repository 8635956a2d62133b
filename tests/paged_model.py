"""What a cache of pages must hold after any calls: a plain list of rows a sequence, and random
calls made of both."""

from __future__ import annotations

import numpy as np
import torch


class PagedModel:
    """Rows are numbers, each written once: sequence -> its numbers, in order."""

    def __init__(self) -> None:
        self.rows: dict[int, list[int]] = {}
        self.next = 1

    def fresh(self, count: int) -> list[int]:
        numbers = list(range(self.next, self.next + count))
        self.next += count
        return numbers


def _write(cache, sequence: int, first: int, numbers: list[int]) -> None:
    """Put the numbers into rows first .. of the sequence: keys hold it, values its negative."""
    if not numbers:
        return
    at = torch.arange(first, first + len(numbers))
    table = torch.tensor(cache.pages_of(sequence))
    page = table[at // cache.page_rows].to(cache.keys.device)
    row = (at % cache.page_rows).to(cache.keys.device)
    value = torch.tensor(numbers, dtype=torch.float32, device=cache.keys.device)
    # Small whole numbers: exact in bf16 as two digits to the base of 200.
    for pool, sign in ((cache.keys, 1.0), (cache.values, -1.0)):
        for layer in range(pool.shape[0]):
            pool[layer, page, :, row, 0] = (sign * (value % 200)).to(pool.dtype)[:, None]
            pool[layer, page, :, row, -1] = (sign * (value // 200)).to(pool.dtype)[:, None]


def check_against(cache, model: PagedModel) -> None:
    size = cache.page_rows
    tables, lengths = cache.tables.cpu(), cache.lengths.cpu()
    keys, values = cache.keys.float().cpu(), cache.values.float().cpu()
    held = np.zeros(cache.pages, dtype=int)
    for s in range(len(lengths)):
        numbers = model.rows.get(s)
        if numbers is None:
            assert lengths[s] == 0 and (tables[s] == -1).all()
            continue
        assert lengths[s] == len(numbers) == cache.rows(s)
        pages = cache.pages_of(s)
        assert tables[s].tolist() == pages + [-1] * (tables.shape[1] - len(pages))
        assert len(set(pages)) == len(pages) >= -(-len(numbers) // size)
        for page in pages:
            held[page] += 1
        at = torch.arange(len(numbers))
        page, row = torch.tensor(pages, dtype=torch.long)[at // size], at % size
        want = torch.tensor(numbers)
        for layer in range(keys.shape[0]):
            for pool, sign in ((keys, 1), (values, -1)):
                got = pool[layer, page, :, row, -1] * 200 + pool[layer, page, :, row, 0]
                assert torch.equal(got, (sign * want).float()[:, None].expand_as(got))
    assert cache.free_pages == int((held == 0).sum())


def random_calls(cache, model: PagedModel, rng: np.random.Generator, count: int, check_every: int = 1) -> None:
    """`count` random calls; the ones a full pool refuses have to leave everything as it was."""
    for turn in range(count):
        open_ones = sorted(model.rows)
        kind = rng.choice(["open", "step", "step", "step", "fork", "free", "truncate", "compact", "reserve"])
        some = [int(s) for s in rng.permutation(open_ones)[: rng.integers(1, 4)]] if open_ones else []
        try:
            if kind == "open":
                rows = int(rng.integers(0, 45))
                s = cache.open(rows)
                model.rows[s] = model.fresh(rows)
                _write(cache, s, 0, model.rows[s])
            elif kind == "step" and some:
                tokens = [int(n) for n in rng.integers(1, 20, len(some))]
                batch = cache.batch(some, tokens=tokens)
                cache.ready(batch)
                for s, n in zip(some, tokens):
                    numbers = model.fresh(n)
                    _write(cache, s, len(model.rows[s]), numbers)
                    model.rows[s] += numbers
                cache.advance(batch)
            elif kind == "fork" and some:
                share = bool(rng.random() < 0.7)
                for kid in cache.fork(some[0], int(rng.integers(1, 3)), share=share):
                    model.rows[kid] = list(model.rows[some[0]])
            elif kind == "free" and some:
                cache.free(some)
                for s in some:
                    del model.rows[s]
            elif kind == "truncate" and some:
                keep = int(rng.integers(0, len(model.rows[some[0]]) + 1))
                cache.truncate(some[0], keep)
                model.rows[some[0]] = model.rows[some[0]][:keep]
            elif kind == "compact":
                live = cache.compact()
                assert live == cache.pages - cache.free_pages
                assert all(p < live for s in model.rows for p in cache.pages_of(s))
            elif kind == "reserve" and some:
                cache.reserve(some[0], len(model.rows[some[0]]) + int(rng.integers(0, 40)))
        except ValueError as refused:
            assert "needed" in str(refused) or "asked for" in str(refused) or "at most" in str(refused), refused
        if turn % check_every == 0 or turn == count - 1:
            check_against(cache, model)
