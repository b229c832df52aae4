"""Calls of the paged operators that must be reported or must not disturb others."""
import subprocess
import sys
import textwrap
import threading
from pathlib import Path

import pytest
import torch

import paged_math as M
from deuteron_b200 import native, ops
from deuteron_b200.paged import PagedCache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(cuda):
    native.device_status(0)
    yield
    ops.check_device_status()


def test_appends_outside_what_a_row_holds_are_reported(cuda):
    cache = PagedCache(layers=1, pages=8, page_size=4, kv_heads=2, head_dim=64, max_sequences=4, max_pages_per_sequence=5)
    cache.pool.fill_(3.0)
    closed, kept, cut, fresh = (cache.open() for _ in range(4))
    cache.extend([closed, cut], [6, 10])
    cache.close(closed)
    cache.extend([kept], [12])                       # takes the pages of the closed row
    cache.truncate(cut, 3)
    before = cache.pool.clone()
    k = torch.ones(1, 2, 64, dtype=torch.float16, device='cuda')
    for row, position in ((closed, 0), (closed, 5), (cut, 4), (cut, 9), (cut, 12), (fresh, 0), (kept, 12)):
        cache.append(0, k, k, torch.tensor([row], dtype=torch.int32).cuda(), torch.tensor([position], dtype=torch.int32).cuda())
        with pytest.raises(native.PageError, match='paged append'):
            ops.check_device_status()
        assert torch.equal(cache.pool, before), (row, position)
    reopened = cache.open()                          # the closed row's number
    assert reopened == closed
    cache.append(0, k, k, torch.tensor([reopened], dtype=torch.int32).cuda(), torch.tensor([0], dtype=torch.int32).cuda())
    with pytest.raises(native.PageError, match='paged append'):
        ops.check_device_status()
    assert torch.equal(cache.pool, before)
    rows, positions = cache.extend([kept], [1])
    cache.append(0, k, k, rows, positions)
    ops.check_device_status()
    assert not torch.equal(cache.pool, before)


def test_a_new_cache_leaves_reports_standing(cuda):
    pool = torch.zeros(1, 1, 4, 64, dtype=torch.float16, device='cuda')
    one = torch.tensor([1], dtype=torch.int32).cuda()
    ops.copy_pages(pool, one, one)                   # a page outside the pool
    torch.cuda.synchronize()
    PagedCache(layers=1, pages=2, page_size=4, kv_heads=1, head_dim=64, max_sequences=1)
    with pytest.raises(native.PageError, match='copy of pages'):
        ops.check_device_status()
    native.call('dtn_selftest_wait_timeout', 1000, torch.cuda.current_stream().cuda_stream)   # a wait with a budget that runs out
    torch.cuda.synchronize()
    PagedCache(layers=1, pages=2, page_size=4, kv_heads=1, head_dim=64, max_sequences=1)
    with pytest.raises(native.DeviceWaitError, match='self-test'):
        ops.check_device_status()


def test_a_cache_made_in_a_capture(cuda):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache = PagedCache(layers=1, pages=2, page_size=4, kv_heads=1, head_dim=64, max_sequences=2)
    graph.replay()
    assert bool((cache.tables == -1).all()) and not cache.lengths.any()


def test_threads_call_first_on_one_shared_stream(cuda):
    k_pages, v_pages, tables, lens = M.a_cache([3000, 70], 2, 64, torch.float16, 16, 'cuda')
    q = torch.randn(2, 8, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    expected = ops.paged_attention(q, k_pages, v_pages, tables, lens, 0.125)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    results, meeting = {}, threading.Barrier(6)

    def work(number):
        with torch.cuda.stream(stream):
            meeting.wait(30)
            results[number] = [ops.paged_attention(q, k_pages, v_pages, tables, lens, 0.125) for _ in range(20)]

    threads = [threading.Thread(target=work, args=(number,)) for number in range(6)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert all(torch.equal(y, expected) for number in range(6) for y in results[number])


def test_the_book_does_not_change_inside_a_capture(cuda):
    cache = PagedCache(layers=1, pages=8, page_size=4, kv_heads=1, head_dim=64, max_sequences=3)
    a = cache.open()
    cache.extend([a], [6])
    fork = cache.fork(a)
    state = cache.tables.tolist(), cache.lengths.tolist(), cache.book.tables.tolist(), cache.book.references.tolist()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: cache.extend([a], [1]), lambda: cache.extend([fork], [0]), lambda: cache.close(a), lambda: cache.fork(a), lambda: cache.truncate(a, 2),
                     cache.compact):
            with pytest.raises(RuntimeError, match='outside captures'):
                call()
        graph_only = torch.zeros(1, device='cuda')
    graph.replay()
    assert not graph_only.any()
    assert (cache.tables.tolist(), cache.lengths.tolist(), cache.book.tables.tolist(), cache.book.references.tolist()) == state
    cache.extend([a, fork], [1, 1])
    assert torch.equal(cache.tables.cpu(), torch.from_numpy(cache.book.tables)) and cache.lengths.tolist()[:2] == [7, 7]


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_the_gradient_of_rotary_is_recorded(cuda, layout, dtype):
    g = torch.Generator().manual_seed(2)
    projected = torch.randn(7, 6, 64, generator=g).to(dtype).cuda().requires_grad_()
    positions = torch.randint(0, 5000, (7,), generator=g).cuda()
    w, amplitude = ops.rotary_frequencies(48, scaling='yarn', factor=4.0, original_length=64)
    weight = torch.randn(7, 4, 64, generator=g).to(dtype).cuda()
    x = projected[:, 1:5]
    y = ops.rotary(x, positions, w, layout=layout, amplitude=amplitude)
    with torch.no_grad():
        plain = ops.rotary(x, positions, w, layout=layout, amplitude=amplitude)
    assert y.requires_grad and not plain.requires_grad and torch.equal(y, plain)
    y.backward(weight)
    expected = torch.zeros_like(projected)
    expected[:, 1:5] = ops.rotary_backward(weight, positions, w, layout=layout, amplitude=amplitude)
    assert torch.equal(projected.grad, expected)
    projected.grad = None
    ops.rotary(projected, positions, w, layout=layout).sum().backward()          # the gradient arrives as one expanded value
    assert torch.equal(projected.grad, ops.rotary_backward(torch.ones_like(projected), positions, w, layout=layout).detach())
    back = ops.rotary_backward(x, positions, w, layout=layout)
    gradient, = torch.autograd.grad(back, projected, weight, create_graph=True)
    assert torch.equal(gradient[:, 1:5], ops.rotary(weight, positions, w, layout=layout))
    # of the gradient as a function of what it is applied to: the map is linear
    leaf = weight.clone().requires_grad_()
    first, = torch.autograd.grad(ops.rotary(x, positions, w, layout=layout), projected, leaf, create_graph=True)
    second, = torch.autograd.grad(first[:, 1:5], leaf, weight)
    assert torch.equal(second, ops.rotary(weight, positions, w, layout=layout))


def test_rotary_records_on_streams_and_in_captures(cuda):
    x = torch.randn(9, 3, 32, generator=torch.Generator().manual_seed(3)).cuda().requires_grad_()
    positions, (w, _) = torch.arange(9, device='cuda'), ops.rotary_frequencies(32)
    expected = ops.rotary_backward(torch.ones(9, 3, 32, device='cuda'), positions, w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            gradient, = torch.autograd.grad(ops.rotary(x, positions, w).sum(), x)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(gradient, expected)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured, = torch.autograd.grad(ops.rotary(x, positions, w).sum(), x)
    captured.zero_()
    graph.replay()
    assert torch.equal(captured, expected)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('heads', [(8, 2), (16, 1), (3, 3)])
@pytest.mark.parametrize('dim', [64, 128, 256])
def test_attention_in_place_of_its_queries(cuda, dim, heads, dtype):
    # 20 long sequences are split between blocks, others are empty or short
    k_pages, v_pages, tables, lens = M.a_cache([9000, 0, 5, 130] + [700] * 20, heads[1], dim, dtype, 16, 'cuda')
    projected = torch.randn(24, heads[0] + 2, dim, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    v_pages[int(tables[3, 0]), :, 0, 1] = float('inf')                 # a second pass over one of them
    for q in (projected[:, 1:-1], projected[:, 1:-1].contiguous()):
        expected = ops.paged_attention(q, k_pages, v_pages, tables, lens, 0.1, out=torch.empty_like(q))
        for _ in range(5):
            place = projected.clone()[:, 1:-1] if not q.is_contiguous() else q.clone()
            assert ops.paged_attention(place, k_pages, v_pages, tables, lens, 0.1, out=place) is place and torch.equal(place, expected)


def test_a_bad_page_does_not_cover_a_wait_that_ran_out(cuda):
    pool = torch.zeros(2, 1, 4, 64, dtype=torch.float16, device='cuda')
    two = torch.tensor([2], dtype=torch.int32).cuda()
    tables, lens = torch.tensor([[2]], dtype=torch.int32).cuda(), torch.tensor([3], dtype=torch.int32).cuda()
    one = torch.zeros(1, 1, 64, dtype=torch.float16, device='cuda')
    row = torch.zeros(1, dtype=torch.int32, device='cuda')
    for call in (lambda: ops.copy_pages(pool, two, two), lambda: ops.paged_append(one, one, pool, pool, tables, row, row),
                 lambda: ops.paged_attention(one, pool, pool, tables, lens, 1.0)):
        native.call('dtn_selftest_wait_timeout', 1000, torch.cuda.current_stream().cuda_stream)
        call()
        with pytest.raises(native.DeviceWaitError, match='self-test'):
            ops.check_device_status()
        call()
        with pytest.raises(native.PageError):
            ops.check_device_status()


def alone(code):
    """Runs code in a fresh process, where no operator has been called yet."""
    root = Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, '-c', 'import sys; sys.path.insert(0, sys.argv[1])\n' + textwrap.dedent(code), str(root)], capture_output=True, text=True, timeout=180)
    assert done.returncode == 0, done.stdout + done.stderr


def test_the_status_word_is_not_made_inside_a_capture(cuda):
    alone("""
        import torch
        from deuteron_b200 import native, ops
        x = torch.zeros(8, device='cuda')
        y = x + 1
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = x + 1
            native.call('dtn_device_status_prepare', torch.cuda.current_stream().cuda_stream)
        graph.replay()
        torch.cuda.synchronize()
        assert y.sum().item() == 8
        native.call('dtn_device_status_prepare', 0)
        assert native.device_status() == 0
    """)


def test_the_status_word_beside_a_capture_that_blocks_the_default_stream(cuda):
    # the default stream cannot be asked then: the word is not made, the capture goes on
    alone("""
        import torch
        from cuda.bindings import runtime
        from deuteron_b200 import native
        torch.zeros(1, device='cuda')
        error, stream = runtime.cudaStreamCreate()
        assert int(error) == 0
        native.call('dtn_capture_begin', int(stream))
        native.call('dtn_device_status_prepare', 0)
        error, graph = runtime.cudaStreamEndCapture(stream)
        assert int(error) == 0, error
        native.call('dtn_device_status_prepare', 0)
        assert native.device_status() == 0
    """)


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('pairs', [32, 13])
def test_strides_beyond_32_bits(cuda, pairs, layout):
    # tokens, then heads, 2^31 elements and more apart
    stride = 2 ** 31 + 2 ** 10
    buffer = torch.empty(2 * stride + 6 * 64, dtype=torch.float16, device='cuda')
    w, _ = ops.rotary_frequencies(2 * pairs)
    positions = torch.tensor([5, 100, 7000]).cuda()
    x = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(6)).half().cuda()
    expected = ops.rotary(x, positions, w, layout=layout)
    for strides in ((stride, 64, 1), (64, stride, 1)):
        view = buffer.as_strided((3, 2, 64), strides)
        view.copy_(x)
        assert torch.equal(ops.rotary(view, positions, w, layout=layout), expected)
        assert ops.rotary(view, positions, w, layout=layout, out=view) is view and torch.equal(view, expected)
    tables, rows = torch.tensor([[1, 0]], dtype=torch.int32).cuda(), torch.zeros(3, dtype=torch.int32, device='cuda')
    k_pages, v_pages = torch.zeros(2, 2, 2, 4, 64, dtype=torch.float16, device='cuda')
    positions = torch.arange(3, device='cuda')
    view.copy_(x)
    result = ops.paged_append(view, view, k_pages, v_pages, tables, rows, positions, frequencies=w, layout=layout, q=view)
    assert torch.equal(result, ops.rotary(x, positions, w, layout=layout))
    assert torch.equal(k_pages[1, :, :3].transpose(0, 1), result) and torch.equal(v_pages[1, :, :3].transpose(0, 1), x)
    lens, step = torch.tensor([3], dtype=torch.int32).cuda(), view[:1]
    step.copy_(result[2:])
    plain = ops.paged_attention(result[2:], k_pages, v_pages, tables, lens, 0.125, out=torch.empty_like(result[2:]))
    assert torch.equal(ops.paged_attention(step, k_pages, v_pages, tables, lens, 0.125, out=step), plain)
