"""Accuracy of attention over a paged cache where little of the mass counts: small probabilities beside a large one."""
import pytest
import torch

import paged_math as M
from deuteron_b200 import native, ops

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.fixture(autouse=True)
def clean_status(cuda):
    native.device_status(0)
    yield
    ops.check_device_status()


def within(actual, exact, bound):
    off = (actual.double() - exact).abs()
    assert not torch.isnan(off).any()
    worst = (off / bound).max().item()
    assert worst <= 1, f'{worst} times the bound; largest error {off.max().item()} of {exact.abs().max().item()}'


def tail_below_a_sink(length, heads, dim, dtype, page_size, below, sink):
    """One sequence whose token `sink` has score 0 and value 0; every other one scores -below and has positive values.

    Returns the kernel's result, the exact one and a bound. Queries are the first unit vector and a key's first element is its
    score, so scores are exact. In base 2 a score is rounded three times (log2 e, the product, the difference to the maximum), to
    2^-24 of `below` each in natural units; ex2 is good to 2^-21, the terms of a product to 2^-22, sums of n tokens to
    (n + 64) 2^-23, for numerators and denominators alike. f16 terms may leave 2^-44 of a probability of 1 in each."""
    q_heads, kv_heads = heads
    k_pages, v_pages, tables, lens = M.a_cache([length], kv_heads, dim, dtype, page_size, 'cuda', seed=3)
    v_pages.abs_()
    k_pages.zero_()
    k_pages[..., 0] = -float(below)
    page = int(tables[0, sink // page_size])
    k_pages[page, :, sink % page_size, 0] = 0.0
    v_pages[page, :, sink % page_size] = 0.0
    q = torch.zeros(1, q_heads, dim, dtype=dtype, device='cuda')
    q[..., 0] = 1.0
    y = ops.paged_attention(q, k_pages, v_pages, tables, lens, 1.0)
    v = M.gathered(v_pages, tables[0], 0, length)                           # [kv_heads, length, dim]
    scores = torch.full((length,), -float(below), dtype=torch.float64, device='cuda')
    scores[sink] = 0.0
    p = torch.softmax(scores, dim=0)
    exact = torch.einsum('t,htd->hd', p, v)
    relative = 3 * 2.0 ** -24 * below + 2.0 ** -21 + 2.0 ** -22 + (length + 64) * 2.0 ** -23
    bound = 2 * relative * exact + (2.0 ** -44 * v.sum(dim=1) if dtype == torch.float16 else 0.0) + exact * 2.0 ** -24
    group = q_heads // kv_heads
    return y, exact.repeat_interleave(group, dim=0)[None], bound.repeat_interleave(group, dim=0)[None]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('below', [0, 6, 12, 14, 16, 18, 22])
@pytest.mark.parametrize('length', [2, 12, 48, 700, 4096])
def test_small_probabilities_beside_a_sink(cuda, length, below, dtype):
    for sink in sorted({0, length // 2, length - 1}):
        within(*tail_below_a_sink(length, (8, 2), 128, dtype, 16, below, sink))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads', [(1, 1), (16, 1), (32, 1), (40, 1)])
@pytest.mark.parametrize('dim', [64, 80, 128, 192, 256])
def test_small_probabilities_in_every_form(cuda, dim, heads, dtype):
    for page_size in (16, 24):
        within(*tail_below_a_sink(90, heads, dim, dtype, page_size, 16, 5))


@pytest.mark.parametrize('dtype', TYPES)
def test_a_long_tail_of_one_sign(cuda, dtype):
    within(*tail_below_a_sink(30_000, (8, 8), 64, dtype, 64, 18, 4))        # 2^-26 each


# -- values near the end of the type's range -----------------------------------------------------

@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('heads', [(1, 1), (4, 1), (8, 1), (12, 1), (32, 1)])
@pytest.mark.parametrize('dim', [64, 128, 256])
def test_the_largest_values_have_a_finite_mean(cuda, dim, heads, dtype):
    # their sum passes FP32, the result does not: the second pass scales by powers of two, which round nothing
    lengths = [40, 1, 700, 0, 5000]
    k_pages, v_pages, tables, lens = M.a_cache(lengths, heads[1], dim, dtype, 16, 'cuda', seed=4)
    largest = torch.finfo(dtype).max
    sign = torch.where(torch.arange(dim, device='cuda') % 2 == 0, 1.0, -1.0)
    v_pages.copy_(((0.5 + 0.49 * torch.rand(v_pages.shape, generator=torch.Generator().manual_seed(6)).cuda()).double() * largest * sign).to(dtype))
    q = torch.randn(5, heads[0], dim, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    for window in (0, 100):
        exact, bound = M.attend(q, k_pages, v_pages, tables, lens, M.scale_of(dim), window=window)
        y = ops.paged_attention(q, k_pages, v_pages, tables, lens, M.scale_of(dim), window=window)
        empty = lens == 0
        assert not y[empty].any()
        within(y[~empty], exact[~empty], bound[~empty])
        narrow = ops.paged_attention(q, k_pages, v_pages, tables, lens, M.scale_of(dim), window=window, out=torch.empty_like(q))
        assert narrow.isfinite().all()


@pytest.mark.parametrize('dtype', TYPES)
def test_infinite_values_of_a_small_probability(cuda, dtype):
    # e^-76 is above 2^-126: the result is infinite, in the column and the query heads that see it only
    k_pages, v_pages, tables, lens = M.a_cache([50, 50], 1, 64, dtype, 16, 'cuda')
    k_pages.zero_()
    page = int(tables[0, 1])
    k_pages[page, 0, 3, 0] = -76.0
    v_pages[page, 0, 3, 7] = float('-inf')
    q = torch.zeros(2, 4, 64, dtype=dtype, device='cuda')
    q[..., 0] = 1.0
    y = ops.paged_attention(q, k_pages, v_pages, tables, lens, 1.0)
    assert torch.isneginf(y[0, :, 7]).all()
    y[0, :, 7] = 0.0
    assert y.isfinite().all()
