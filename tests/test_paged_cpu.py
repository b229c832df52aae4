"""Refusals and host-side parts of the rotary and paged-cache operators; no GPU."""
import ctypes
import math
import random

import pytest
import torch

from deuteron_b200 import native, ops
from deuteron_b200.paged import PageBook, PagedCache, PagesExhausted


def cache(dtype=torch.float16, pages=4, heads=2, size=8, dim=16):
    pool = torch.zeros(2, pages, heads, size, dim, dtype=dtype)
    return pool[0], pool[1], torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)


def test_frequencies_follow_their_formulas():
    w, amplitude = ops.rotary_frequencies(64, device='cpu')
    assert w.dtype == torch.float64 and amplitude == 1.0
    assert torch.allclose(w, torch.tensor([10000.0 ** (-i / 32) for i in range(32)], dtype=torch.float64), rtol=1e-15)
    linear, amplitude = ops.rotary_frequencies(64, scaling='linear', factor=4.0, device='cpu')
    assert torch.equal(linear, w / 4) and amplitude == 1.0
    stretched, _ = ops.rotary_frequencies(64, scaling='ntk', factor=4.0, device='cpu')
    assert stretched[0] == 1.0 and math.isclose(stretched[-1], w[-1] / 4, rel_tol=1e-12) and bool((stretched[1:] < w[1:]).all())
    yarn, amplitude = ops.rotary_frequencies(64, scaling='yarn', factor=8.0, original_length=4096, device='cpu')
    turns = 4096 * w / (2 * math.pi)
    assert torch.equal(yarn[turns >= 32], w[turns >= 32]) and torch.equal(yarn[turns <= 1], w[turns <= 1] / 8)
    between = (turns > 1) & (turns < 32)
    assert bool(between.any()) and bool(((yarn < w) & (yarn > w / 8))[between].all())
    assert math.isclose(amplitude, 0.1 * math.log(8) + 1)
    assert ops.rotary_frequencies(64, scaling='yarn', factor=1.0, original_length=4096, device='cpu')[1] == 1.0
    assert ops.rotary_frequencies(0, device='cpu')[0].shape == (0,)
    for arguments in (dict(rotary_dim=7), dict(rotary_dim=-2), dict(rotary_dim=8.0), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, base=math.inf),
                      dict(rotary_dim=8, factor=2.0), dict(rotary_dim=8, scaling='cubic'), dict(rotary_dim=8, scaling='yarn', factor=2.0),
                      dict(rotary_dim=2, scaling='ntk', factor=2.0), dict(rotary_dim=8, scaling='linear', factor=0.0), dict(rotary_dim=8, scaling='linear', factor=math.nan),
                      dict(rotary_dim=8, scaling='yarn', factor=2.0, original_length=10, fast=1.0, slow=1.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(**arguments, device='cpu')


def test_rotary_refuses():
    x, at, w = torch.zeros(3, 2, 16), torch.zeros(3, dtype=torch.int32), torch.zeros(8, dtype=torch.float64)
    for arguments, message in (
            ((x.int(), at, w), 'dtype'), ((x.double(), at, w), 'dtype'), ((x[0], at, w), 'heads'), ((x.transpose(1, 2), at, w), 'dense'), ((x, at[:2], w), 'entries'),
            ((x, at.float(), w), 'int32 or int64'), ((x, at.expand(3, 3)[0][::2], w), '1-D'), ((x, at, w.float()), 'float64'),
            ((x, at, torch.zeros(9, dtype=torch.float64)), 'a head has 16'), ((x, at, torch.zeros(16, dtype=torch.float64)[::2]), 'contiguous'),
            (([1.0], at, w), 'tensor'), ((x, 5, w), 'tensor'), ((x, at, None), 'tensor'), ((x, at, w), 'CUDA')):
        for call in (ops.rotary, ops.rotary_backward):
            with pytest.raises(ValueError, match=message):
                call(*arguments)
    with pytest.raises(ValueError, match='layout'):
        ops.rotary(x, at, w, layout='pairs')
    for out, message in ((x.half(), 'shape and dtype'), (torch.zeros(3, 2, 18), 'shape and dtype'), (torch.zeros(1, 2, 16).expand(3, 2, 16), 'expanded'),
                         (torch.zeros(3, 1, 16).expand(3, 2, 16), 'expanded')):
        with pytest.raises(ValueError, match=message):
            ops.rotary(x, at, w, out=out)
    with pytest.raises(ValueError, match='lie elsewhere'):
        ops.rotary(x, at, w, out=x.reshape(2, 3, 16).transpose(0, 1))


def test_append_refuses():
    k_pages, v_pages, tables, _ = cache()
    k, rows, at, w = torch.zeros(3, 2, 16, dtype=torch.float16), torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int64), torch.zeros(8, dtype=torch.float64)
    good = dict(k=k, v=k, k_pages=k_pages, v_pages=v_pages, tables=tables, rows=rows, positions=at, frequencies=w, q=k)
    for changed, message in (
            (dict(v=k[:2]), 'shape'), (dict(v=k.float()), 'dtype'), (dict(k_pages=k_pages.float(), v_pages=v_pages.float()), 'dtype'), (dict(k=k.double()), 'dtype'),
            (dict(k=k[:, :1], v=k[:, :1]), 'shape'), (dict(k_pages=k_pages[0]), 'k_pages must be'), (dict(v_pages=v_pages[:2]), 'one shape'), (dict(v_pages=v_pages.float()), 'one shape'),
            (dict(k_pages=k_pages.transpose(1, 2).contiguous().transpose(1, 2)), 'dense'), (dict(v_pages=v_pages[:1].expand(4, 2, 8, 16)), 'same strides'),
            (dict(k_pages=k_pages[:1].expand(4, 2, 8, 16), v_pages=v_pages[:1].expand(4, 2, 8, 16)), 'expanded'),
            (dict(tables=tables.long()), 'tables'), (dict(tables=tables[0]), 'tables'), (dict(tables=tables.t()), 'tables'), (dict(rows=rows.long()), 'int32'), (dict(rows=rows[:2]), 'entries'),
            (dict(positions=at[:1]), 'entries'), (dict(frequencies=torch.zeros(9, dtype=torch.float64)), 'a head has'), (dict(layout='none'), 'layout'),
            (dict(q=k.float()), 'q must be'), (dict(q=k[:2]), 'q must be'), (dict(q=None, q_out=k), 'without q'), (dict(q_out=k.float()), 'q_out'),
            (dict(q_out=k[:, :1].expand(3, 2, 16)), 'expanded'), (dict(rows=None), 'tensor'), (dict(), 'CUDA')):
        with pytest.raises(ValueError, match=message):
            ops.paged_append(**{**good, **changed})


def test_attention_refuses():
    k_pages, v_pages, tables, lens = cache()
    q = torch.zeros(3, 4, 16, dtype=torch.float16)
    good = dict(q=q, k_pages=k_pages, v_pages=v_pages, tables=tables, lengths=lens, scale=0.25)
    for changed, message in (
            (dict(q=q.float()), 'dtype'), (dict(q=q.double()), 'dtype'), (dict(q=q[..., :8]), 'head size'), (dict(q=q[:, :3]), 'multiple'), (dict(q=q[0]), 'heads'),
            (dict(q=torch.zeros(4, 4, 16, dtype=torch.float16)), '3 sequences'), (dict(lengths=lens.long()), 'int32'), (dict(lengths=lens[:2]), 'entries'),
            (dict(rows=lens.long()), 'int32'), (dict(rows=lens[:2]), 'entries'), (dict(rows=[0, 1, 2]), 'tensor'), (dict(window=-1), 'window'),
            (dict(k_pages=k_pages[:, :0], v_pages=v_pages[:, :0]), 'multiple'), (dict(k_pages=k_pages[:, :, :0], v_pages=v_pages[:, :, :0]), 'at least one'),
            (dict(out=q.bfloat16()), 'out'), (dict(out=q.float()[:2]), 'out'), (dict(out=torch.zeros(3, 1, 16).expand(3, 4, 16)), 'expanded'), (dict(), 'CUDA')):
        with pytest.raises(ValueError, match=message):
            ops.paged_attention(**{**good, **changed})


def test_copies_refuse():
    pool, pair = torch.zeros(2, 3, 2, 8, 16), torch.zeros(1, dtype=torch.int32)
    for arguments, message in (
            ((pool[0, 0, 0], pair, pair), 'pages must be'), ((pool[None, None], pair, pair), 'pages must be'), ((pool.transpose(2, 3), pair, pair), 'dense'),
            ((pool[:, :, :, :4], pair, pair), 'dense'), ((pool[..., :8], pair, pair), 'dense'), ((pool[:, :1].expand(2, 3, 2, 8, 16), pair, pair), 'expanded'),
            ((pool[:1].expand(2, 3, 2, 8, 16), pair, pair), 'expanded'), ((pool[:, None].expand(2, 2, 3, 2, 8, 16), pair, pair), 'evenly|expanded'),
            ((pool, pair.long(), pair), 'int32'), ((pool, pair, pair.repeat(2)), 'entries'), ((pool, [0], [1]), 'tensor'), ((pool, pair, pair), 'CUDA')):
        with pytest.raises(ValueError, match=message):
            ops.copy_pages(*arguments)


ONE = 1 << 20
# pointers and integers in the order of the header's structures, then the double
ROTARY = [ONE] * 4 + [0, 1, 1, 8, 4, 8, 8, 8, 8, 0, 0, 0, 1.0]
APPEND = [ONE] * 10 + [0, 1, 1, 8, 8, 8, 8, 8, 4, 8, 64, 64, 1, 1, 1, 4, 0, 1, 8, 8, 8, 8, 0, 1.0]
ATTENTION = [ONE] * 8 + [1 << 30, 1, 2, 1, 8, 16, 8, 16, 8, 4, 8, 64, 64, 1, 1, 1, 0, 0, 1, 1.0]


def status_of(name, good, changes):
    arguments = list(good)
    for place, value in changes.items():
        arguments[place] = value
    library = native.lib()
    if name == 'dtn_copy_pages':
        return library.dtn_copy_pages(*arguments)
    packer = {'dtn_rotary': native.ROTARY_ARGS, 'dtn_paged_append': native.PAGED_APPEND_ARGS, 'dtn_paged_attention': native.PAGED_ATTENTION_ARGS}[name]
    return getattr(library, name)(packer.pack(*arguments), None)


def test_the_structures_are_those_of_the_header():
    header = (native.LIBRARY_PATH.parent.parent / 'include' / 'deuteron_b200.h').read_text()
    for name, packer in (('dtn_rotary_args', native.ROTARY_ARGS), ('dtn_paged_append_args', native.PAGED_APPEND_ARGS), ('dtn_paged_attention_args', native.PAGED_ATTENTION_ARGS)):
        body = header[:header.index('} ' + name)].rsplit('typedef struct {', 1)[1]
        declarations = [line.strip() for line in body.split(';') if line.strip()]
        fields = sum(len(line.split(',')) for line in declarations)
        assert packer.size == 8 * fields and declarations[-1].startswith('double') and len(declarations[-1].split(',')) == 1
        assert all('*' in line or line.startswith('int64_t') for line in declarations[:-1])


def test_the_c_entries_check_before_any_cuda_call():
    copies = [ONE, 1, 64, 4, 64, 64, ONE, ONE, 1, None]
    for name in ('dtn_rotary', 'dtn_paged_append', 'dtn_paged_attention'):
        assert getattr(native.lib(), name)(None, None) == native.ERR_INVALID
    for name, good, bad in (
            ('dtn_rotary', ROTARY, {0: 0, 1: 0, 2: 0, 3: 0, 5: -1, 6: -1, 7: -1, 8: 5, 15: 3}),
            ('dtn_paged_append', APPEND, {0: 0, 1: 0, 2: 0, 3: 0, 4: 0, 5: 0, 6: 0, 7: 0, 8: 0, 9: 0, 11: -1, 12: -1, 13: -1, 18: -1, 19: 0, 22: -1, 23: -1,
                                          25: 5, 27: -1, 32: -1}),
            ('dtn_paged_attention', ATTENTION, {0: 0, 1: 0, 2: 0, 3: 0, 4: 0, 6: 0, 9: -1, 10: 3, 11: 0, 17: -1, 18: 0, 21: -1, 22: -1, 24: -1, 25: 5}),
            ('dtn_copy_pages', copies, {0: None, 1: -1, 3: -1, 5: -1, 6: None, 7: None, 8: -1})):
        for place, value in bad.items():
            changes = {place: value}
            if name == 'dtn_paged_attention' and place == 10:
                changes[11] = 2                                   # three query heads over two kv heads
            assert status_of(name, good, changes) == native.ERR_INVALID, (name, place)
            assert native.last_error()
    for name, good, changes in (('dtn_rotary', ROTARY, {7: 1025}), ('dtn_rotary', ROTARY, {5: 2 ** 31}), ('dtn_paged_append', APPEND, {13: 1025}),
                                ('dtn_paged_append', APPEND, {23: 2 ** 31}), ('dtn_paged_attention', ATTENTION, {12: 264}), ('dtn_copy_pages', copies, {8: 2 ** 31})):
        assert status_of(name, good, changes) == native.ERR_UNSUPPORTED, (name, changes)
    # nothing to do is no error, and needs no pointer and no device
    for name, good, changes in (('dtn_rotary', ROTARY, {0: 0, 5: 0}), ('dtn_rotary', ROTARY, {1: 0, 6: 0}), ('dtn_paged_append', APPEND, {0: 0, 11: 0}),
                                ('dtn_paged_attention', ATTENTION, {0: 0, 9: 0}), ('dtn_copy_pages', copies, {0: None, 8: 0})):
        assert status_of(name, good, changes) == native.OK, (name, changes)


def test_attention_entry_refuses_alignment_and_workspace():
    size = ctypes.c_size_t(0)
    native.call('dtn_paged_attention_workspace_bytes', ctypes.byref(size))
    assert 4096 < size.value < 16 << 20
    for place, value, status, text in ((1, ONE + 8, native.ERR_INVALID, '16-byte'), (2, ONE + 2, native.ERR_INVALID, '16-byte'), (12, 12, native.ERR_INVALID, '16-byte'),
                                       (19, 60, native.ERR_INVALID, '16-byte'), (20, 4, native.ERR_INVALID, '16-byte'), (7, 0, native.ERR_WORKSPACE, 'workspace'),
                                       (8, size.value - 1, native.ERR_WORKSPACE, 'needed'), (8, -1, native.ERR_WORKSPACE, 'needed'), (7, ONE + 4, native.ERR_WORKSPACE, 'aligned')):
        good = list(ATTENTION)
        good[25] = 1
        assert status_of('dtn_paged_attention', good, {place: value}) == status and text in native.last_error(), (place, native.last_error())


def test_the_plan_covers_every_unit_once_and_names_its_owners():
    generator = random.Random(3)
    cases = [([1], 1, 1, 1), ([1], 8, 2, 296), ([1000], 1, 2, 296), ([1, 0, 1], 1, 1, 2), ([2 ** 27], 8, 2, 296), ([5, 1, 700, 0, 33], 4, 2, 148), ([0, 0], 3, 4, 9)]
    cases += [([generator.randint(0, 60) for _ in range(generator.randint(1, 40))], generator.randint(1, 9), generator.randint(1, 4), generator.randint(1, 300)) for _ in range(60)]
    for tiles, heads, least, grid in cases:
        items = len(tiles) * heads
        begin, first, last, workers = ((ctypes.c_int64 * n)() for n in (grid + 1, items, items, 1))
        native.call('dtn_paged_attention_plan', (ctypes.c_int64 * len(tiles))(*tiles), len(tiles), heads, least, grid, begin, first, last, workers)
        count, units = workers[0], sum(n + 3 for n in tiles if n) * heads
        if not units:
            assert count == 0 and set(first) == set(last) == {-1}
            continue
        shares = [begin[c + 1] - begin[c] for c in range(count)]
        assert 1 <= count <= grid and begin[0] == 0 and begin[count] == units and max(shares) - min(shares) <= 1
        assert min(shares) >= least or count == 1
        at, started = 0, []
        for item in range(items):
            if tiles[item // heads] == 0:
                assert first[item] == last[item] == -1
                continue
            end = at + tiles[item // heads]
            owners = [c for c in range(count) if begin[c] < end and begin[c + 1] > at]
            assert (first[item], last[item]) == (owners[0], owners[-1]) and owners == list(range(owners[0], owners[-1] + 1))
            if len(owners) > 1:
                started.append(first[item])
            at = end + 3
        assert len(set(started)) == len(started)          # one counter per block is enough: no two split items start in one block
    assert native.lib().dtn_paged_attention_plan((ctypes.c_int64 * 1)(-1), 1, 1, 1, 1, None, None, None, None) == native.ERR_INVALID


def test_positions_are_divided_by_a_multiplication():
    # the multiplier and shift that the kernel is given: floor(2^(31 + s) / d) + 1 and 31 + s with 2^s >= d
    generator = random.Random(5)
    for d in [2, 3, 5, 7, 8, 16, 24, 50, 64, 1000, 2 ** 20 - 1, 2 ** 30 + 1, 2 ** 31 - 1] + [generator.randint(2, 2 ** 31 - 1) for _ in range(200)]:
        s = 1
        while 1 << s < d:
            s += 1
        multiplier = (1 << (31 + s)) // d + 1
        assert multiplier < 2 ** 32
        for n in [0, 1, d - 1, d, d + 1, 2 ** 31 - 1, (2 ** 31 - 1) // d * d, (2 ** 31 - 1) // d * d - 1] + [generator.randint(0, 2 ** 31 - 1) for _ in range(50)]:
            if 0 <= n < 2 ** 31:
                assert n * multiplier >> (31 + s) == n // d and n * multiplier < 2 ** 64


def test_page_reports_have_their_own_error(monkeypatch):
    for word, text in ((0x6103, 'paged attention'), (0x6200, 'paged append'), (0x63ff, 'copy of pages')):
        monkeypatch.setattr(native, 'device_status', lambda stream=0, word=word: word)
        with pytest.raises(native.PageError, match=text):
            native.raise_on_device_status(0)
    monkeypatch.setattr(native, 'device_status', lambda stream=0: 0x7100)
    with pytest.raises(native.DeviceWaitError, match='self-test'):
        native.raise_on_device_status(0)


def check_book(book):
    """Counts of references are what the tables say; a page is free or held; rows are free or open."""
    held = [book.tables[row, :-(-int(book.lengths[row]) // book.page_size)].tolist() for row in range(len(book.lengths)) if book._open[row]]
    counted = [0] * len(book.references)
    for pages in held:
        assert len(set(pages)) == len(pages)
        for page in pages:
            counted[page] += 1
    assert counted == book.references.tolist()
    assert sorted(book._free_pages) == [page for page, n in enumerate(counted) if n == 0] and book.free_pages == len(book._free_pages)
    assert sorted(book._free_rows) == [row for row, is_open in enumerate(book._open) if not is_open]


@pytest.mark.parametrize('seed', range(6))
def test_the_book_keeps_every_sequence_whole(seed):
    # a model: every sequence's tokens as a list, the pool as one; random calls, the copies applied as the device would
    generator = random.Random(seed)
    size = generator.choice([1, 3, 4, 16])
    book = PageBook(pages=24, page_size=size, max_sequences=7, max_pages_per_sequence=9)
    pool, tables, tokens, next_token = [[None] * size for _ in range(24)], [[0] * 9 for _ in range(7)], {}, 0
    for _ in range(400):
        call = generator.choice(['open', 'close', 'fork', 'extend', 'extend', 'extend', 'truncate', 'compact'])
        copies, updates, written = [], [], []
        state = (book.tables.copy(), book.lengths.copy(), book.references.copy(), sorted(book._free_pages))
        try:
            if call == 'open':
                tokens[book.open()] = []
            elif call == 'compact':
                copies, updates = book.compact()
                used = int((book.references > 0).sum())
                assert not book.references[used:].any()
            elif not tokens:
                continue
            elif call == 'close':
                row = generator.choice(sorted(tokens))
                book.close(row)
                del tokens[row]
            elif call == 'fork':
                row = generator.choice(sorted(tokens))
                new, updates = book.fork(row)
                tokens[new] = list(tokens[row])
            elif call == 'truncate':
                row = generator.choice(sorted(tokens))
                kept = generator.randint(0, len(tokens[row]))
                book.truncate(row, kept)
                del tokens[row][kept:]
            else:
                rows = generator.sample(sorted(tokens), generator.randint(1, len(tokens)))
                counts = [generator.choice([0, 1, 1, 2, size, 2 * size + 1]) for _ in rows]
                copies, updates = book.extend(rows, counts)
                for row, count in zip(rows, counts):
                    for _ in range(count):
                        written.append((row, len(tokens[row]), next_token))
                        tokens[row].append(next_token)
                        next_token += 1
        except (PagesExhausted, ValueError):
            after = (book.tables.copy(), book.lengths.copy(), book.references.copy(), sorted(book._free_pages))
            assert all((a == b).all() for a, b in zip(state[:3], after[:3])) and state[3] == after[3]
            continue
        destinations = [to for _, to in copies]
        assert len(set(destinations)) == len(destinations) and not set(destinations) & {source for source, _ in copies}
        for source, to in copies:
            pool[to] = list(pool[source])
        assert len({(row, column) for row, column, _ in updates}) == len(updates)
        for row, column, page in updates:
            tables[row][column] = page
        for row, position, value in written:
            pool[tables[row][position // size]][position % size] = value
        check_book(book)
        for row, expected in tokens.items():
            assert int(book.lengths[row]) == len(expected)
            assert [pool[tables[row][i // size]][i % size] for i in range(len(expected))] == expected, call
            assert tables[row][:-(-len(expected) // size)] == book.tables[row, :-(-len(expected) // size)].tolist()


def test_the_book_refuses():
    for arguments in ((0, 4, 1, 1), (1, 0, 1, 1), (1, 4, 0, 1), (1, 4, 1, 0), (1, 4.0, 1, 1), (1, 2 ** 20, 1, 2 ** 11), (1, 1, 2 ** 20, 2 ** 11)):
        with pytest.raises(ValueError):
            PageBook(*arguments)
    book = PageBook(pages=3, page_size=4, max_sequences=2, max_pages_per_sequence=3)
    row = book.open()
    for call in (lambda: book.close(1), lambda: book.fork(-1), lambda: book.extend([row, row], [1, 1]), lambda: book.extend([row], [-1]),
                 lambda: book.extend([row], [1, 2]), lambda: book.extend([row], [13]), lambda: book.truncate(row, 1), lambda: book.truncate(row, -1)):
        with pytest.raises(ValueError):
            call()
    book.extend([row], [6])
    other, _ = book.fork(row)
    with pytest.raises(PagesExhausted):
        book.open()
    with pytest.raises(PagesExhausted):
        book.extend([row, other], [2, 3])     # a copy of the shared page is the last free one; a third page is missing
    copies, _ = book.extend([row, other], [2, 2])
    assert copies == [(1, 2)] and book.free_pages == 0
    book.close(other)
    with pytest.raises(ValueError):
        book.close(other)
    check_book(book)


def test_the_cache_brings_the_device_up_to_date():
    cache = PagedCache(layers=2, pages=6, page_size=4, kv_heads=2, head_dim=16, max_sequences=3, max_pages_per_sequence=4, device='cpu')
    a, b = cache.open(), cache.open()
    rows, positions = cache.extend([a, b], [5, 3])
    assert rows.tolist() == [a] * 5 + [b] * 3 and positions.tolist() == [0, 1, 2, 3, 4, 0, 1, 2] and rows.dtype == positions.dtype == torch.int32
    rows, positions = cache.extend([b, a], [0, 1])
    assert rows.tolist() == [a] and positions.tolist() == [5]
    assert [t.numel() for t in cache.extend([], [])] == [0, 0]
    c = cache.fork(a)
    cache.truncate(c, 4)
    assert cache.lengths.tolist() == [6, 3, 4] and torch.equal(cache.tables, torch.from_numpy(cache.book.tables))
    cache.close(b)
    assert cache.lengths.tolist() == [6, 0, 4]
    assert cache.keys(1).data_ptr() == cache.pool[1, 0].data_ptr() and cache.values(0).shape == (6, 2, 4, 16)
    for changed in (dict(dtype=torch.float64), dict(head_dim=12), dict(head_dim=264), dict(layers=0), dict(kv_heads=-1)):
        with pytest.raises(ValueError):
            PagedCache(**{**dict(layers=2, pages=6, page_size=4, kv_heads=2, head_dim=16, max_sequences=3, device='cpu'), **changed})
    with pytest.raises(ValueError, match='CUDA'):
        cache.attend(0, torch.zeros(3, 2, 16, dtype=torch.float16), 1.0)
