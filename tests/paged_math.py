"""Plain 64-bit forms of the paged-cache operators, and the error bounds that their FP32 arithmetic allows (test infrastructure)."""
import math

import torch

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step, relative


def tiny(dtype):
    """Half of the smallest step of a type: what a rounding of a subnormal result may be off by."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rotate(x, positions, frequencies, layout, amplitude, sign=1.0):
    """x[t, h] with its pairs turned by complex factors; 64 bits."""
    pairs = frequencies.numel()
    y = x.double().clone()
    angle = positions.double()[:, None] * frequencies[None, :] * sign
    c, s = angle.cos()[:, None, :] * amplitude, angle.sin()[:, None, :] * amplitude
    first, second = (slice(0, pairs), slice(pairs, 2 * pairs)) if layout == 'half' else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


def rotation_bound(x, exact, positions, frequencies, layout, amplitude):
    """|error| of one rotated element. The fraction of a turn is rounded to 32 bits (half_turns in [-1, 1]: 2^-25, pi times that in
    radians: 1.6 x 2^-24), sincospif is good to 2 ulp (2^-22 of 1 at most, taken whole), the amplitude and the two products
    and the sum round to 2^-24 each: below 2^-21 (|a| + |b|) * amplitude in all. The angle itself is rounded twice in 64 bits on
    either side: 4 x 2^-53 of position * frequency. Then one rounding to the type."""
    pairs = frequencies.numel()
    first, second = (slice(0, pairs), slice(pairs, 2 * pairs)) if layout == 'half' else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
    size = torch.zeros_like(exact)
    both = (x[..., first].double().abs() + x[..., second].double().abs()) * amplitude
    angle = (2.0 ** -21 + (positions.double().abs()[:, None] * frequencies[None, :]) * 2.0 ** -51)[:, None, :]
    size[..., first] = both * angle
    size[..., second] = both * angle
    rounded = exact.abs() * EPS[x.dtype] + tiny(x.dtype)
    rounded[..., 2 * pairs:] = 0.0   # copied
    return size * (1 + EPS[x.dtype]) + rounded


def gathered(pages, table, first, length):
    """Tokens first..length of one sequence, [kv_heads, tokens, dim] in 64 bits."""
    size = pages.shape[2]
    used = table[: -(-length // size)].long()
    return pages[used].transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, first:length].double()


def attend(q, k_pages, v_pages, tables, lengths, scale, rows=None, window=0, out_dtype=torch.float32):
    """Result and error bound of one-token attention over pages.

    The bound: a score is a sum of `dim` exact (16-bit storage) or rounded products added in FP32, off by at most
    (dim + 4) 2^-24 of the sum of magnitudes A, scaled and put in base 2 (3 more roundings): E = (dim + 8) 2^-24 * A * scale.
    A probability is then off by e^(2 E) - 1 from its score and its maximum together, by 2^-21 from ex2, and by 2^-22 from the
    terms it is split into for the 16-bit products (2^-24 absolute for f16, whose smallest step is 2^-24). The sums over n tokens,
    numerator and denominator alike, and their rescalings round to (n + 64) 2^-23 (accumulators may truncate)."""
    n, q_heads, dim = q.shape
    kv_heads = k_pages.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for i in range(n):
        row = i if rows is None else int(rows[i])
        length = int(lengths[row]) if row >= 0 else 0
        first = max(0, length - window) if window else 0
        if length <= 0:
            continue
        k, v = gathered(k_pages, tables[row], first, length), gathered(v_pages, tables[row], first, length)
        x = q[i].double().reshape(kv_heads, -1, dim)
        scores = x @ k.transpose(-1, -2) * scale
        p = torch.softmax(scores, dim=-1)
        y = p @ v
        e = (dim + 8) * 2.0 ** -24 * ((x.abs() @ k.abs().transpose(-1, -2)) * abs(scale)).amax(dim=-1, keepdim=True)
        relative = torch.expm1(2 * e) + 2.0 ** -21 + 2.0 ** -22 + (v.shape[1] + 64) * 2.0 ** -23
        spread = p @ v.abs()
        absolute = 2.0 ** -24 * v.abs().sum(dim=1, keepdim=True) if q.dtype == torch.float16 else 0.0
        off = 2 * relative * spread + 2 * absolute
        out[i] = y.reshape(q_heads, dim)
        bound[i] = (off * (1 + EPS[out_dtype]) + y.abs() * EPS[out_dtype] + tiny(out_dtype)).reshape(q_heads, dim)
    return out, bound


def a_cache(lengths, kv_heads, dim, dtype, page_size, device, seed=0, spare=2, width=None, fill=None):
    """Pools with shuffled pages, tables and lengths; the places behind a sequence's end and the unused pages hold `fill` (None: values)."""
    g = torch.Generator(device='cpu').manual_seed(seed)
    needed = [-(-n // page_size) for n in lengths]
    total = sum(needed) + spare
    order = torch.randperm(total, generator=g).tolist()
    width = max(1, max(needed, default=0)) if width is None else width
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    pools = torch.randn(2, total, kv_heads, page_size, dim, generator=g)
    at = 0
    unused = torch.ones(total, page_size, dtype=torch.bool)
    for i, (n, count) in enumerate(zip(lengths, needed)):
        tables[i, :count] = torch.tensor(order[at:at + count], dtype=torch.int32)
        for j in range(count):
            unused[order[at + j], : min(page_size, n - j * page_size)] = False
        at += count
    if fill is not None:
        pools = pools.masked_fill(unused[None, :, None, :, None], fill)
    pools = pools.to(dtype).to(device)
    return pools[0], pools[1], tables.to(device), torch.tensor(lengths, dtype=torch.int32, device=device)


def scale_of(dim):
    return 1.0 / math.sqrt(dim)
