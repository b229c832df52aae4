"""Calls of the paged cache that go wrong on the host's side; no GPU."""
import ctypes
import random
import threading

import numpy as np
import pytest
import torch

from deuteron_b200 import native, ops
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


def test_threads_that_call_first_on_one_stream_share_its_workspace(monkeypatch):
    # both threads are held inside the creation until the other is there
    meeting = threading.Barrier(2)

    def call(name, size):
        assert name == 'dtn_paged_attention_workspace_bytes'
        size._obj.value = 8192
        meeting.wait(10)

    monkeypatch.setattr(native, 'call', call)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    monkeypatch.setattr(ops, '_paged_workspaces', {})
    results = []
    threads = [threading.Thread(target=lambda: results.append(ops._paged_workspace(torch.zeros(1), 7))) for _ in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert len(results) == 2 and results[0][-2:] == results[1][-2:]
    kept, = ops._paged_workspaces.values()
    assert kept[0].data_ptr() == results[0][-2] and not kept[0][:4096].any()


def test_a_captured_call_holds_its_workspace(monkeypatch):
    monkeypatch.setattr(native, 'call', lambda name, size: setattr(size._obj, 'value', 8192))
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    monkeypatch.setattr(ops, '_paged_workspaces', {})
    first, second = (ops._paged_workspace(torch.zeros(1), 7) for _ in range(2))
    assert isinstance(first[0], torch.Tensor) and first[0].data_ptr() == first[1] != second[1] and not ops._paged_workspaces


def test_the_kernels_own_division_of_positions_is_exact():
    generator = random.Random(5)
    most = 2 ** 31 - 1
    sizes = [1, 2, 3, 5, 7, 8, 16, 24, 50, 64, 1000, 2 ** 16, 2 ** 16 + 1, 2 ** 20 - 1, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, most - 1, most]
    for size in sizes + [generator.randint(1, most) for _ in range(300)] + [generator.randint(1, 4096) for _ in range(300)]:
        near = [generator.randint(0, most // size) * size + step for _ in range(60) for step in (-1, 0, 1)]   # around multiples
        ends = [most // size * size + step for step in (-1, 0, 1)] + [most - i for i in range(20)] + [size - 1, size, size + 1]
        positions = [n for n in near + ends + [0, 1] + [generator.randint(0, most) for _ in range(50)] if 0 <= n <= most]
        found = (ctypes.c_int * len(positions))()
        native.call('dtn_paged_attention_pages', (ctypes.c_int * len(positions))(*positions), len(positions), size, found)
        assert list(found) == [n // size for n in positions], size
    one = (ctypes.c_int * 1)(-1)
    for arguments in ((one, 1, 8, one), (one, 1, 0, one), (one, 1, 2 ** 31, one), (one, -1, 8, one), (None, 1, 8, one), (one, 1, 8, None)):
        assert native.lib().dtn_paged_attention_pages(*arguments) == native.ERR_INVALID


def test_rows_counts_and_lengths_are_whole_numbers():
    cache = a_cache()
    a, b = cache.open(), cache.open()
    cache.extend([np.int64(a), torch.tensor(b)], [np.int32(3), torch.tensor(2)])
    state = cache.tables.clone(), cache.lengths.tolist(), cache.book.lengths.tolist(), cache.book.free_pages
    for call in (lambda: cache.extend([a], [1.5]), lambda: cache.extend([a], [2.0]), lambda: cache.extend([float(a)], [1]), lambda: cache.extend(['0'], [1]),
                 lambda: cache.truncate(a, 1.5), lambda: cache.close(0.0), lambda: cache.fork(None), lambda: cache.extend([a, b], [1, '1'])):
        with pytest.raises(ValueError, match='integer'):
            call()
        assert torch.equal(cache.tables, state[0]) and (cache.lengths.tolist(), cache.book.lengths.tolist(), cache.book.free_pages) == state[1:]
    rows, positions = cache.extend([a, b], [2, 1])
    assert rows.tolist() == [a, a, b] and positions.tolist() == [3, 4, 2]


def test_rotary_refuses_gradients_that_it_cannot_record():
    x, at, w = torch.zeros(3, 2, 16, requires_grad=True), torch.zeros(3, dtype=torch.int32), torch.zeros(8, dtype=torch.float64)
    for call in (ops.rotary, ops.rotary_backward):
        with pytest.raises(ValueError, match='no_grad'):
            call(x, at, w, out=torch.zeros(3, 2, 16))
        with pytest.raises(ValueError, match='frequencies have no gradient'):
            call(x.detach(), at, w.clone().requires_grad_())
        with torch.no_grad(), pytest.raises(ValueError, match='CUDA'):
            call(x, at, w.clone().requires_grad_(), out=torch.zeros(3, 2, 16))


def test_copies_of_too_many_planes_are_refused():
    one = 1 << 20
    for planes, pairs in ((2 ** 62, 4), (2 ** 33, 2 ** 30), (2 ** 31, 1), (2, 2 ** 30)):
        assert native.lib().dtn_copy_pages(one, planes, 64, 4, 64, 64, one, one, pairs, None) == native.ERR_UNSUPPORTED, (planes, pairs)


def test_attention_refuses_an_out_that_lies_on_q_otherwise():
    pool, tables, lens = torch.zeros(4, 2, 8, 16), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for dtype in (torch.float16, torch.float32):
        memory = torch.zeros(3 * 4 * 16, dtype=torch.float32)
        q = memory.view(dtype)[:3 * 4 * 16].view(3, 4, 16)
        outs = [q.reshape(4, 3, 16).transpose(0, 1)] + ([memory.view(3, 4, 16)] if dtype == torch.float16 else [])
        for out in outs:
            with pytest.raises(ValueError, match='lie elsewhere'):
                ops.paged_attention(q, pool.to(dtype), pool.to(dtype), tables, lens, 1.0, out=out)
        with pytest.raises(ValueError, match='CUDA'):
            ops.paged_attention(q, pool.to(dtype), pool.to(dtype), tables, lens, 1.0, out=q)


@pytest.mark.parametrize('made', [False, True])
@pytest.mark.parametrize('used', [False, True])
def test_a_cache_serves_inside_and_outside_inference_mode(made, used):
    with torch.inference_mode(made):
        cache = a_cache()
        row = cache.open()
    with torch.inference_mode(used):
        rows, positions = cache.extend([row], [5])
        fork = cache.fork(row)
    cache.truncate(fork, 2)
    assert positions.tolist() == [0, 1, 2, 3, 4] and cache.lengths.tolist() == [5, 2, 0, 0]
    assert torch.equal(cache.tables, torch.from_numpy(cache.book.tables))
