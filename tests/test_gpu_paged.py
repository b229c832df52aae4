"""Rotary positions, the paged cache's writer, its attention of one new token and its page copies, against 64-bit forms."""
import math

import pytest
import torch

import paged_math as M
from deuteron_b200 import native, ops
from deuteron_b200.paged import PagedCache, PagesExhausted

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.fixture(autouse=True)
def clean_status(cuda):
    native.device_status(0)
    yield
    ops.check_device_status()


def normal(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def within(actual, exact, bound):
    off = (actual.double() - exact).abs()
    worst = (off - bound).max().item() if off.numel() else 0.0
    assert not torch.isnan(off).any() and worst <= 0, f'{worst} beyond the bound; largest error {off.max().item()}'


# -- rotary positions ----------------------------------------------------------------------------

ROTARY = [   # tokens, heads, dim, pairs
    (1, 40, 128, 64), (3, 1, 16, 8), (5, 3, 64, 16), (7, 2, 96, 48), (2, 5, 80, 37), (33, 4, 40, 20), (4, 2, 256, 128), (65, 9, 72, 4),
    (3, 2, 10, 5), (2, 3, 7, 2), (6, 2, 128, 0), (300, 8, 64, 32), (1, 1, 2, 1), (9, 70, 24, 12), (2, 3, 1024, 512),
]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('shape', ROTARY)
def test_rotary_and_its_gradient(cuda, shape, layout, dtype):
    tokens, heads, dim, pairs = shape
    x = normal((tokens, heads, dim), dtype)
    positions = torch.randint(0, 200_000, (tokens,), generator=torch.Generator().manual_seed(1)).cuda()
    w, _ = ops.rotary_frequencies(2 * pairs)
    for call, sign in ((ops.rotary, 1.0), (ops.rotary_backward, -1.0)):
        exact = M.rotate(x, positions, w, layout, 1.25, sign)
        y = call(x, positions, w, layout=layout, amplitude=1.25)
        assert y.dtype == dtype and y.shape == x.shape
        within(y, exact, M.rotation_bound(x, exact, positions, w, layout, 1.25))
        assert torch.equal(call(x, positions.int(), w, layout=layout, amplitude=1.25), y)
        z = x.clone()
        assert call(z, positions, w, layout=layout, amplitude=1.25, out=z) is z and torch.equal(z, y)


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_rotary_gradient_against_differences_and_the_adjoint(cuda, layout):
    x, g = normal((5, 3, 48), torch.float32, 1), normal((5, 3, 48), torch.float32, 2)
    positions = torch.tensor([0, 1, 17, 4000, 99_999]).cuda()
    w, amplitude = ops.rotary_frequencies(32, scaling='yarn', factor=4.0, original_length=2048)
    gradient = ops.rotary_backward(g, positions, w, layout=layout, amplitude=amplitude)
    # the map is linear: a central difference of <g, rotary(x)> along one element is exact but for rounding. Each of the two
    # products sums over 720 values of FP32 results (each off by 2^-21 (|a| + |b|) at most) and the step is 1
    step = torch.zeros_like(x)
    for place in ((0, 0, 0), (2, 1, 5), (3, 2, 16), (4, 0, 31), (1, 1, 40), (4, 2, 47)):
        step.zero_()
        step[place] = 1.0
        up, down = (ops.rotary(x + s * step, positions, w, layout=layout, amplitude=amplitude).double() for s in (1, -1))
        difference = ((up - down) * g.double()).sum().item() / 2
        touched = 2 ** -20 * amplitude * 4 * (x.abs().max().item() + 1) * g.abs().max().item()
        assert abs(difference - gradient[place].item()) <= touched
    leaf = x.double().requires_grad_()
    M_out = torch.empty(0)
    angle = positions.double()[:, None] * w
    c, s = (angle.cos() * amplitude)[:, None], (angle.sin() * amplitude)[:, None]
    if layout == 'half':
        a, b = leaf[..., :16], leaf[..., 16:32]
        M_out = torch.cat([a * c - b * s, b * c + a * s, leaf[..., 32:]], -1)
    else:
        a, b = leaf[..., 0:32:2], leaf[..., 1:32:2]
        M_out = torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), leaf[..., 32:]], -1)
    (M_out * g.double()).sum().backward()
    within(gradient, leaf.grad, M.rotation_bound(g, leaf.grad, positions, w, layout, amplitude))


@pytest.mark.parametrize('dtype', TYPES)
def test_rotary_of_strided_heads_and_far_positions(cuda, dtype):
    w, _ = ops.rotary_frequencies(64)
    projected = normal((19, 12, 96), dtype)
    positions = torch.tensor([2 ** 30 - i * 7919 for i in range(19)], dtype=torch.int64).cuda()
    by_head = projected.transpose(0, 1).contiguous().transpose(0, 1)   # heads outermost in memory
    padded = normal((19, 12, 101), dtype)[:, :, 3:99]                  # rows that start off 16-byte boundaries
    for x in (projected[:, 2:9], by_head[:, 1:4], projected[::3], padded, projected[:, :, :64], projected[:, :1].expand(19, 5, 96)):
        at = positions[:x.shape[0]].contiguous()
        for layout in ('half', 'interleaved'):
            exact = M.rotate(x, at, w, layout, 1.0)
            bound = M.rotation_bound(x, exact, at, w, layout, 1.0)
            within(ops.rotary(x, at, w, layout=layout), exact, bound)
            target = torch.full((x.shape[0], x.shape[1] + 2, x.shape[2] + 5), 7.0, dtype=dtype, device='cuda')
            view = target[:, 1:-1, 3:3 + x.shape[2]]
            ops.rotary(x, at, w, layout=layout, out=view)
            within(view, exact, bound)
            rim = target.clone()
            rim[:, 1:-1, 3:3 + x.shape[2]] = 7.0
            assert torch.equal(rim, torch.full_like(rim, 7.0))         # nothing beside the view was written


def test_rotary_passes_infinities_and_empty_calls(cuda):
    w, _ = ops.rotary_frequencies(8)
    x = torch.zeros(2, 1, 16, device='cuda')
    x[0, 0, 9], x[1, 0, 15] = float('inf'), float('nan')               # copied elements
    y = ops.rotary(x, torch.tensor([5, 6]).cuda(), w)
    assert torch.equal(torch.nan_to_num(y, 3.0), torch.nan_to_num(x, 3.0))
    for shape in ((0, 4, 16), (3, 0, 16), (3, 4, 0)):
        empty = torch.empty(shape, device='cuda')
        none = w if shape[2] else w[:0]
        assert ops.rotary(empty, torch.zeros(shape[0], dtype=torch.int32, device='cuda'), none).shape == shape


# -- append --------------------------------------------------------------------------------------

APPEND = [   # tokens per sequence, q_heads, kv_heads, dim, pairs, page size, start
    ((1, 1, 1), 8, 2, 128, 64, 16, 31), ((5,), 3, 1, 64, 16, 1, 0), ((17, 2, 40), 4, 4, 96, 48, 24, 7), ((3, 0, 1), 5, 5, 40, 11, 8, 100),
    ((33, 65), 0, 2, 80, 0, 50, 0), ((9,), 6, 3, 256, 128, 64, 60), ((4, 4), 2, 1, 6, 3, 5, 2), ((200,), 32, 8, 128, 64, 16, 0),
]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('case', APPEND)
def test_append_rotates_stores_and_leaves_the_rest(cuda, case, layout, dtype):
    counts, q_heads, kv_heads, dim, pairs, size, start = case
    k_pages, v_pages, tables, _ = M.a_cache([start + n for n in counts], kv_heads, dim, dtype, size, 'cuda', seed=3)
    rows = [r for r, n in enumerate(counts) for _ in range(n)] + [-1, -5]
    places = [start + i for n in counts for i in range(n)] + [0, 2 ** 31 - 1]
    order = torch.randperm(len(rows), generator=torch.Generator().manual_seed(4)).tolist()
    rows, places = [rows[i] for i in order], [places[i] for i in order]
    projected = normal((len(rows), q_heads + 2 * kv_heads, dim), dtype, 5)
    q, k, v = projected.split([q_heads, kv_heads, kv_heads], dim=1)
    w = ops.rotary_frequencies(2 * pairs)[0] if pairs else None
    positions = torch.tensor(places, dtype=torch.int32).cuda()
    before = k_pages.clone(), v_pages.clone()
    rotated_k = ops.rotary(k, positions, w, layout=layout, amplitude=1.5) if pairs else k
    expected_q = (ops.rotary(q, positions, w, layout=layout, amplitude=1.5) if pairs else q) if q_heads else None
    for i, (row, place) in enumerate(zip(rows, places)):
        if row >= 0:
            page = int(tables[row, place // size])
            before[0][page, :, place % size], before[1][page, :, place % size] = rotated_k[i], v[i]
    result = ops.paged_append(k, v, k_pages, v_pages, tables, torch.tensor(rows, dtype=torch.int32).cuda(), positions, frequencies=w, layout=layout,
                              amplitude=1.5, q=q if q_heads else None)
    assert torch.equal(k_pages, before[0]) and torch.equal(v_pages, before[1])
    assert result is None if not q_heads else torch.equal(result, expected_q)
    if q_heads:
        again = ops.paged_append(k, v, k_pages, v_pages, tables, torch.tensor(rows, dtype=torch.int32).cuda(), positions.long(), frequencies=w,
                                 layout=layout, amplitude=1.5, q=q, q_out=q)
        assert again is q and torch.equal(q, expected_q) and torch.equal(k_pages, before[0])


def test_append_reports_places_outside_the_cache(cuda):
    k_pages, v_pages, tables, _ = M.a_cache([10, 10], 2, 64, torch.float16, 4, 'cuda')
    k, v = normal((1, 2, 64), torch.float16, 1), normal((1, 2, 64), torch.float16, 2)
    tables[1, 1] = k_pages.shape[0]
    tables[1, 2] = -1
    before = k_pages.clone(), v_pages.clone()
    for row, place in ((2, 0), (0, 12), (0, -1), (1, 4), (1, 8), (0, 2 ** 31 - 1)):
        ops.paged_append(k, v, k_pages, v_pages, tables, torch.tensor([row], dtype=torch.int32).cuda(),
                         torch.tensor([place], dtype=torch.int32).cuda())
        with pytest.raises(native.PageError, match='paged append'):
            ops.check_device_status()
    assert torch.equal(k_pages, before[0]) and torch.equal(v_pages, before[1])


# -- attention -----------------------------------------------------------------------------------

def attend_both(lengths, q_heads, kv_heads, dim, dtype, size, window=0, rows=None, out_dtype=torch.float32, fill=float('nan'), seed=0, gain=1.0):
    k_pages, v_pages, tables, lens = M.a_cache(lengths, kv_heads, dim, dtype, size, 'cuda', seed=seed, fill=fill)
    n = len(lengths) if rows is None else len(rows)
    q = normal((n, q_heads, dim), dtype, seed + 9) * gain
    chosen = None if rows is None else torch.tensor(rows, dtype=torch.int32).cuda()
    out = None if out_dtype == torch.float32 else torch.full((n, q_heads, dim), 9.0, dtype=out_dtype, device='cuda')
    y = ops.paged_attention(q, k_pages, v_pages, tables, lens, M.scale_of(dim), rows=chosen, window=window, out=out)
    assert y.dtype == out_dtype and (out is None or y is out)
    exact, bound = M.attend(q, k_pages, v_pages, tables, lens, M.scale_of(dim), rows=rows, window=window, out_dtype=out_dtype)
    within(y, exact, bound)
    assert torch.equal(y, ops.paged_attention(q, k_pages, v_pages, tables, lens, M.scale_of(dim), rows=chosen, window=window, out=torch.empty_like(y)))
    return y


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads', [(1, 1), (4, 4), (32, 8), (7, 1), (10, 2), (16, 1), (24, 2), (40, 1), (9, 3), (70, 2)])
def test_attention_over_groups_of_heads(cuda, heads, dtype):
    attend_both([0, 1, 63, 200, 37], *heads, 128, dtype, 16)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('dim', [4, 8, 16, 24, 64, 72, 80, 96, 120, 128, 136, 192, 248, 256])
def test_attention_over_head_sizes(cuda, dim, dtype):
    if dim % (16 // dtype.itemsize):
        pytest.skip('heads of whole 16-byte vectors')
    attend_both([5, 130, 64], 4, 2, dim, dtype, 16)
    attend_both([33], 24, 2, dim, dtype, 8, out_dtype=dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [1, 3, 8, 16, 24, 50, 128, 1000])
def test_attention_over_page_sizes_and_lengths(cuda, size, dtype):
    attend_both([0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300], 8, 2, 64, dtype, size)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('window', [1, 5, 16, 64, 100, 1000, 2 ** 40])
def test_attention_of_the_last_tokens(cuda, window, dtype):
    attend_both([0, 1, 5, 64, 101, 333], 8, 2, 64, dtype, 24, window=window)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [8, 16, 24, 64])
def test_what_lies_before_the_window_does_not_matter(cuda, size, dtype):
    lengths, window = [300, 41, 77, 16, 100], 40
    k_pages, v_pages, tables, lens = M.a_cache(lengths, 2, 64, dtype, size, 'cuda')
    q = normal((5, 8, 64), dtype, 2)
    exact, bound = M.attend(q, k_pages, v_pages, tables, lens, 0.125, window=window)
    for row, length in enumerate(lengths):
        for position in range(max(0, length - window)):
            page = int(tables[row, position // size])
            k_pages[page, :, position % size], v_pages[page, :, position % size] = float('nan'), float('-inf')
    within(ops.paged_attention(q, k_pages, v_pages, tables, lens, 0.125, window=window), exact, bound)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads', [(8, 8), (8, 2), (12, 1), (32, 1)])
def test_long_ragged_batches_are_joined(cuda, heads, dtype):
    attend_both([5000, 1, 0, 777, 12_345, 64], *heads, 64, dtype, 16)
    attend_both([9001], *heads, 128, dtype, 64, out_dtype=dtype)
    attend_both([3, 2000] * 100, *heads, 64, dtype, 32)


@pytest.mark.parametrize('dtype', TYPES)
def test_rows_choose_sequences_and_pad_the_batch(cuda, dtype):
    y = attend_both([70, 0, 41, 9], 8, 2, 128, dtype, 16, rows=[2, -1, 0, 0, 1, -3, 3])
    assert not y[1].any() and not y[4].any() and not y[5].any()
    attend_both([12] * 300, 4, 4, 64, dtype, 16, rows=[i % 300 for i in range(700)])
    attend_both([20, 30], 2, 1, 64, dtype, 8, rows=[])


@pytest.mark.parametrize('dtype', TYPES)
def test_large_scores_and_fillings(cuda, dtype):
    # scores of several hundred: the maximum is what keeps the exponentials in range
    attend_both([100, 700], 8, 2, 64, dtype, 16, gain=64.0)
    for fill in (float('inf'), float('-inf'), torch.finfo(dtype).min):
        attend_both([1, 50, 0, 17], 8, 2, 64, dtype, 16, fill=fill)


@pytest.mark.parametrize('dtype', TYPES)
def test_nan_and_infinite_values_that_are_seen_come_through(cuda, dtype):
    k_pages, v_pages, tables, lens = M.a_cache([40, 40, 40, 40], 1, 64, dtype, 16, 'cuda')
    q = normal((4, 4, 64), dtype, 2)
    k_pages[int(tables[0, 1]), 0, 3] = float('nan')
    v_pages[int(tables[1, 0]), 0, 0, 5] = float('inf')
    k_pages[tables[2].long()] = float('-inf')
    q[2] = 1.0                                     # every score of sequence 2 is -inf
    y = ops.paged_attention(q, k_pages, v_pages, tables, lens, 0.125)
    assert y[0].isnan().all() and y[2].isnan().all()
    assert torch.isposinf(y[1, :, 5]).all() and y[1, :, :5].isfinite().all() and y[3].isfinite().all()


@pytest.mark.parametrize('dtype', TYPES)
def test_attention_of_strided_tensors(cuda, dtype):
    k_pages, v_pages, tables, lens = M.a_cache([100, 37, 64], 2, 64, dtype, 16, 'cuda')
    pool = torch.stack([k_pages, v_pages], dim=1).contiguous()          # keys and values of a page side by side
    k_pages, v_pages = pool[:, 0], pool[:, 1]
    wide = torch.zeros(6, 20, dtype=torch.int32, device='cuda')
    wide[::2, :tables.shape[1]] = tables
    tables = wide[::2, :tables.shape[1]]
    projected = normal((3, 14, 64), dtype, 1)
    q = projected[:, 3:11]
    target = torch.full((3, 10, 70), 5.0, device='cuda')
    y = ops.paged_attention(q, k_pages, v_pages, tables, lens, 0.3, out=target[:, 1:9, 2:66])
    exact, bound = M.attend(q, k_pages, v_pages, tables, lens, 0.3)
    within(y, exact, bound)
    target[:, 1:9, 2:66] = 5.0
    assert torch.equal(target, torch.full_like(target, 5.0))
    negative, bound = M.attend(q, k_pages, v_pages, tables, lens, -0.3)
    within(ops.paged_attention(q, k_pages, v_pages, tables, lens, -0.3), negative, bound)


def test_attention_reports_places_outside_the_cache(cuda):
    k_pages, v_pages, tables, lens = M.a_cache([100, 100, 30], 2, 64, torch.float16, 16, 'cuda')
    q = normal((3, 4, 64), torch.float16)
    exact, bound = M.attend(q, k_pages, v_pages, tables, lens, 0.125)
    for wrong in (-1, k_pages.shape[0], 2 ** 31 - 1, -2 ** 31):
        bad = tables.clone()
        bad[1, 3] = wrong
        y = ops.paged_attention(q, k_pages, v_pages, bad, lens, 0.125)
        with pytest.raises(native.PageError, match='paged attention'):
            ops.check_device_status()
        assert y[1].isnan().all()
        within(y[[0, 2]], exact[[0, 2]], bound[[0, 2]])
    longer = lens.clone()
    longer[0] = 7 * 16 + 1                                              # the tables cover 112 tokens; the seventh page has no entry beyond 100
    tables[tables < 0] = 0
    ops.paged_attention(q, k_pages, v_pages, tables, longer, 0.125)
    with pytest.raises(native.PageError):
        ops.check_device_status()
    y = ops.paged_attention(q, k_pages, v_pages, tables, lens, 0.125, rows=torch.tensor([3, 0, 1], dtype=torch.int32).cuda())
    with pytest.raises(native.PageError):
        ops.check_device_status()
    assert not y[0].any()
    negative = lens.clone()
    negative[2] = -4
    assert not ops.paged_attention(q, k_pages, v_pages, tables, negative, 0.125)[2].any()
    empty = k_pages[:0]
    assert ops.paged_attention(q, empty, empty, tables, torch.zeros_like(lens), 0.125).abs().max() == 0
    assert ops.paged_attention(q, empty, empty, tables, lens, 0.125).isnan().all()
    with pytest.raises(native.PageError):
        ops.check_device_status()


def test_offsets_pass_32_bits(cuda):
    # two pages 2^32 bytes and more apart; a third behind them
    stride = 2 ** 31 + 2 ** 12
    buffer = torch.empty(2 * stride + 16 * 2 * 64, dtype=torch.float16, device='cuda')
    pages = buffer.as_strided((3, 2, 8, 64), (stride, 8 * 64, 64, 1))
    values = buffer[16 * 64:].as_strided((3, 2, 8, 64), (stride, 8 * 64, 64, 1))
    k, v = normal((24, 2, 64), torch.float16, 1), normal((24, 2, 64), torch.float16, 2)
    tables = torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda()
    rows = torch.zeros(24, dtype=torch.int32, device='cuda')
    ops.paged_append(k, v, pages, values, tables, rows, torch.arange(24, device='cuda'))
    lens = torch.tensor([23], dtype=torch.int32).cuda()
    q = normal((1, 4, 64), torch.float16, 3)
    exact, bound = M.attend(q, pages, values, tables, lens, 0.125)
    within(ops.paged_attention(q, pages, values, tables, lens, 0.125), exact, bound)
    ops.copy_pages(pages, torch.tensor([2], dtype=torch.int32).cuda(), torch.tensor([1], dtype=torch.int32).cuda())
    assert torch.equal(pages[1], pages[2]) and torch.equal(pages[2], k[:8].transpose(0, 1))


# -- pages ---------------------------------------------------------------------------------------

@pytest.mark.parametrize('dtype', TYPES + [torch.uint8])
@pytest.mark.parametrize('shape', [(9, 2, 16, 64), (3, 9, 1, 8, 24), (2, 2, 30, 4, 16, 128), (1, 9, 1, 1, 3), (5, 40, 1, 50, 7), (2, 9, 8, 128, 256), (4, 2, 9, 5, 3, 2)])
def test_copies_of_pages(cuda, shape, dtype):
    pool = (torch.randn(shape, generator=torch.Generator().manual_seed(1)) * 50).to(dtype).cuda()
    count = shape[-4]
    order = torch.randperm(count, generator=torch.Generator().manual_seed(2))
    pairs = count // 2
    src, dst = order[:pairs].int().cuda(), order[pairs:2 * pairs].int().cuda()
    src[0] = src[-1]                                                    # one page copied twice
    expected = pool.clone()
    expected[..., dst.long(), :, :, :] = pool[..., src.long(), :, :, :]
    assert ops.copy_pages(pool, src, dst) is None
    assert torch.equal(pool, expected)
    ops.copy_pages(pool, src[:0], dst[:0])
    assert torch.equal(pool, expected)


def test_copies_of_pages_report_numbers_outside_the_pool(cuda):
    pool = normal((2, 6, 1, 4, 8), torch.float32)
    before = pool.clone()
    for pair in ((0, 6), (6, 0), (-1, 2), (2, -1), (2 ** 31 - 1, 1)):
        ops.copy_pages(pool, torch.tensor([pair[0]], dtype=torch.int32).cuda(), torch.tensor([pair[1]], dtype=torch.int32).cuda())
        with pytest.raises(native.PageError, match='copy of pages'):
            ops.check_device_status()
        assert torch.equal(pool, before)


def test_copies_of_pages_in_a_strided_pool(cuda):
    pool = normal((3, 2, 12, 2, 8, 16), torch.float16)
    before = pool.clone()
    ops.copy_pages(pool[1, 1], torch.tensor([3], dtype=torch.int32).cuda(), torch.tensor([5], dtype=torch.int32).cuda())
    before[1, 1, 5] = before[1, 1, 3]
    ops.copy_pages(pool[:, 0, ::2], torch.tensor([1, 4], dtype=torch.int32).cuda(), torch.tensor([0, 5], dtype=torch.int32).cuda())
    before[:, 0, 0], before[:, 0, 10] = before[:, 0, 2], before[:, 0, 8]
    assert torch.equal(pool, before)
    with pytest.raises(ValueError, match='evenly'):
        ops.copy_pages(pool[:, :, ::2].transpose(0, 1), torch.tensor([1], dtype=torch.int32).cuda(), torch.tensor([2], dtype=torch.int32).cuda())


# -- together ------------------------------------------------------------------------------------

def test_tensors_of_the_cpu_and_streams(cuda):
    q = torch.zeros(1, 2, 64)
    pool = torch.zeros(1, 1, 16, 64)
    with pytest.raises(ValueError, match='CUDA'):
        ops.paged_attention(q, pool, pool, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1.0)
    k_pages, v_pages, tables, lens = M.a_cache([3000, 70], 2, 64, torch.float16, 16, 'cuda')
    q = normal((2, 8, 64), torch.float16)
    expected = ops.paged_attention(q, k_pages, v_pages, tables, lens, 0.125)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for _ in range(20):                                                 # calls that may overlap share nothing
        for stream in streams:
            with torch.cuda.stream(stream):
                results.append(ops.paged_attention(q, k_pages, v_pages, tables, lens, 0.125))
    torch.cuda.synchronize()
    assert all(torch.equal(y, expected) for y in results)


def test_host_threads_on_their_own_streams(cuda):
    import threading
    k_pages, v_pages, tables, lens = M.a_cache([3000, 70], 2, 64, torch.float16, 16, 'cuda')
    q = normal((2, 8, 64), torch.float16)
    expected = ops.paged_attention(q, k_pages, v_pages, tables, lens, 0.125)
    torch.cuda.synchronize()
    results = {}

    def work(number):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            results[number] = [ops.paged_attention(q, k_pages, v_pages, tables, lens, 0.125) for _ in range(50)]
            stream.synchronize()

    threads = [threading.Thread(target=work, args=(number,)) for number in range(4)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert all(torch.equal(y, expected) for number in range(4) for y in results[number])


def test_captured_graphs_share_no_workspace(cuda):
    k_pages, v_pages, tables, lens = M.a_cache([5000, 170], 2, 64, torch.float16, 16, 'cuda')
    q = [normal((2, 8, 64), torch.float16, seed) for seed in range(2)]
    expected = [ops.paged_attention(x, k_pages, v_pages, tables, lens, 0.125) for x in q]
    graphs, outs = [], []
    for x in q:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.paged_attention(x, k_pages, v_pages, tables, lens, 0.125))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(30):                                                 # replayed beside one another and beside eager calls
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = ops.paged_attention(q[0], k_pages, v_pages, tables, lens, 0.125)
    torch.cuda.synchronize()
    assert torch.equal(eager, expected[0])
    for out, y in zip(outs, expected):
        assert torch.equal(out, y)
    lens.copy_(torch.tensor([12, 0], dtype=torch.int32))                # the lengths are read on the device: a replay follows them
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for out, x in zip(outs, q):
        exact, bound = M.attend(x, k_pages, v_pages, tables, lens, 0.125)
        within(out, exact, bound)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_prompts_steps_forks_and_compaction_together(cuda, layout, dtype):
    # a decoder's use: prompts, steps, a fork into three, a close, compaction, drafts that are taken back. Beside it every
    # sequence's keys and values are kept whole, and every step's attention is held to the 64-bit form over them
    layers, q_heads, kv_heads, dim, size = 2, 6, 2, 64, 8
    cache = PagedCache(layers=layers, pages=30, page_size=size, kv_heads=kv_heads, head_dim=dim, max_sequences=6, max_pages_per_sequence=12, dtype=dtype)
    cache.pool.fill_(float('nan'))
    w, amplitude = ops.rotary_frequencies(48, scaling='yarn', factor=4.0, original_length=64)
    g = torch.Generator(device='cuda').manual_seed(5)
    kept = {}   # row: per layer a list of (key, value) rows

    def step(rows, counts):
        token_rows, positions = cache.extend(rows, counts)
        n = token_rows.numel()
        results = []
        for layer in range(layers):
            q, k, v = torch.randn(n, q_heads + 2 * kv_heads, dim, device='cuda', generator=g).to(dtype).split([q_heads, kv_heads, kv_heads], dim=1)
            turned = cache.append(layer, k, v, token_rows, positions, frequencies=w, layout=layout, amplitude=amplitude, q=q)
            keys = ops.rotary(k, positions, w, layout=layout, amplitude=amplitude)
            assert torch.equal(turned, ops.rotary(q, positions, w, layout=layout, amplitude=amplitude))
            for i, row in enumerate(token_rows.tolist()):
                kept[row][layer].append((keys[i], v[i]))
            results.append(turned)
        return token_rows, results

    def check(token_rows, queries):
        last = {row: i for i, row in enumerate(token_rows.tolist())}
        rows = sorted(last)
        for layer in range(layers):
            q = queries[layer][[last[row] for row in rows]]
            y = cache.attend(layer, q, M.scale_of(dim), rows=torch.tensor(rows, dtype=torch.int32).cuda())
            for i, row in enumerate(rows):
                k = torch.stack([pair[0] for pair in kept[row][layer]]).transpose(0, 1)[None]
                v = torch.stack([pair[1] for pair in kept[row][layer]]).transpose(0, 1)[None]
                exact, bound = M.attend(q[i:i + 1], k, v, torch.zeros(1, 1, dtype=torch.int32).cuda(), [k.shape[2]], M.scale_of(dim))
                within(y[i:i + 1], exact, bound)

    a, b = cache.open(), cache.open()
    kept[a], kept[b] = [[] for _ in range(layers)], [[] for _ in range(layers)]
    check(*step([a, b], [13, 30]))
    for _ in range(3):
        check(*step([b, a], [1, 1]))
    forks = [cache.fork(a) for _ in range(2)]
    for row in forks:
        kept[row] = [list(layer) for layer in kept[a]]
    for _ in range(9):
        check(*step([a, *forks], [1, 1, 1]))
    cache.close(b)
    del kept[b]
    assert cache.compact() > 0
    assert int(cache.tables[sorted(kept)].max()) < 30 - cache.book.free_pages
    check(*step([forks[1], a], [1, 5]))
    cache.truncate(a, 11)
    kept[a] = [layer[:11] for layer in kept[a]]
    check(*step([a, forks[0]], [2, 1]))
    with pytest.raises(PagesExhausted):
        cache.extend([a, *forks], [70, 70, 70])
    with pytest.raises(ValueError):
        cache.extend([a], [100])
    check(*step([a, *forks], [1, 1, 1]))


def test_a_captured_step_follows_the_cache(cuda):
    cache = PagedCache(layers=1, pages=64, page_size=16, kv_heads=2, head_dim=64, max_sequences=4)
    w, _ = ops.rotary_frequencies(64)
    rows = [cache.open() for _ in range(3)]
    token_rows, positions = cache.extend(rows, [40, 7, 100])
    fill = torch.randn(147, 2, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    cache.append(0, fill, fill.flip(0), token_rows, positions, frequencies=w)
    batch_rows = torch.full((4,), -1, dtype=torch.int32, device='cuda')       # one slot is padding
    batch_positions = torch.zeros(4, dtype=torch.int32, device='cuda')
    q, k, v = (torch.zeros(4, heads, 64, dtype=torch.float16, device='cuda') for heads in (8, 2, 2))

    def body():
        turned = cache.append(0, k, v, batch_rows, batch_positions, frequencies=w, q=q)
        return cache.attend(0, turned, 0.125, rows=batch_rows)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = body()
    for i in range(20):
        if i == 10:
            cache.close(rows[1])
            rows[1] = cache.fork(rows[0])
            cache.compact()
        token_rows, positions = cache.extend(rows, [1, 1, 1])
        batch_rows[:3], batch_positions[:3] = token_rows, positions
        for n, x in enumerate((q, k, v)):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 * i + n)).half())
        graph.replay()
        eager = body()                                                        # writes the same keys and values again
        assert torch.equal(captured, eager) and not captured[3].any()
        turned = ops.rotary(q, batch_positions, w)
        exact, bound = M.attend(turned[:3], cache.keys(0), cache.values(0), cache.tables, cache.lengths, 0.125, rows=rows)
        within(captured[:3], exact, bound)
