"""Calls of the paged cache that go wrong on the host's side; no GPU."""
import pytest
import torch

from deuteron_b200 import ops
from deuteron_b200.paged import PageBook, PagedCache


def a_cache(**changed):
    return PagedCache(**{**dict(layers=1, pages=8, page_size=4, kv_heads=1, head_dim=16, max_sequences=4, max_pages_per_sequence=5, device='cpu'), **changed})


def unheld(cache):
    """Entries of the device's tables that no open sequence holds, and that the book agrees with the device."""
    assert torch.equal(cache.tables, torch.from_numpy(cache.book.tables))
    held = -(-torch.from_numpy(cache.book.lengths).long() // cache.book.page_size)
    return cache.tables[torch.arange(cache.tables.shape[1])[None, :] >= held[:, None]]


def test_entries_that_no_sequence_holds_name_no_page(monkeypatch):
    monkeypatch.setattr(ops, 'copy_pages', lambda pool, sources, destinations: None)
    cache = a_cache()
    assert bool((cache.tables < 0).all()) and bool((unheld(cache) < 0).all())
    a, b = cache.open(), cache.open()
    cache.extend([a, b], [9, 5])
    assert bool((unheld(cache) < 0).all()) and unheld(cache).numel() == 20 - 5
    c = cache.fork(a)
    cache.truncate(a, 4)
    assert bool((unheld(cache) < 0).all()) and cache.tables[c].tolist()[:3] == cache.book.tables[c].tolist()[:3] and min(cache.tables[c].tolist()[:3]) >= 0
    cache.extend([a], [6])
    cache.close(b)
    assert bool((unheld(cache) < 0).all())
    cache.compact()
    cache.truncate(c, 0)
    cache.close(a)
    assert bool((unheld(cache) < 0).all()) and bool((cache.tables < 0).all())
    d = cache.open()
    cache.extend([d], [20])
    assert sorted(cache.tables[d].tolist()) == [0, 1, 2, 3, 4] and bool((unheld(cache) < 0).all())


def test_the_book_names_what_it_takes_away():
    book = PageBook(pages=4, page_size=2, max_sequences=2, max_pages_per_sequence=4)
    row = book.open()
    book.extend([row], [7])
    assert book.truncate(row, 5) == [(row, 3, -1)] and book.truncate(row, 5) == []
    assert book.close(row) == [(row, 0, -1), (row, 1, -1), (row, 2, -1)] and book.free_pages == 4
