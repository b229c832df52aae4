"""The cases by which the operators of a decode step over a paged key-value cache are measured.

Four operators: rotary positions (forward and backward), appending rotated keys and values to the pages of a cache,
attention of one new token per sequence over those pages, and copying pages. Where `own` is false `run` computes them
with elementary torch operations; where it is true it calls the framework's operators.
"""
import math
import random

import torch

own = False

DTYPES = {'f16': torch.float16, 'bf16': torch.bfloat16, 'f32': torch.float32}
BYTES = {'f16': 2, 'bf16': 2, 'f32': 4}


def listed():
    return [
        # one token of one user: the projection's 32 query and 8 key heads, far into a conversation
        {'name': 'rotary_one_token', 'op': 'rotary', 'backward': False, 'tokens': 1, 'heads': 40, 'dim': 128, 'rotary': 128, 'layout': 'half',
         'dtype': 'f16', 'far': 100_000, 'scaling': 'none', 'extra_heads': 8},
        # a batch of prompts: query and key heads of a fused projection, rotated where they lie between the value heads
        {'name': 'rotary_prompts', 'op': 'rotary', 'backward': False, 'tokens': 16384, 'heads': 40, 'dim': 128, 'rotary': 128, 'layout': 'half',
         'dtype': 'bf16', 'far': 131_072, 'scaling': 'yarn', 'extra_heads': 8},
        # gradients of a training step, pairs interleaved, a part of an odd-sized head
        {'name': 'rotary_gradient', 'op': 'rotary', 'backward': True, 'tokens': 4095, 'heads': 20, 'dim': 96, 'rotary': 32, 'layout': 'interleaved',
         'dtype': 'f32', 'far': 4095, 'scaling': 'linear', 'extra_heads': 0},
        # one decode step of 64 users
        {'name': 'append_step', 'op': 'append', 'tokens': 64, 'per_sequence': 1, 'q_heads': 32, 'kv_heads': 8, 'dim': 128, 'rotary': 128, 'layout': 'half',
         'dtype': 'f16', 'page_size': 16, 'start': 1000, 'padded': 3},
        # prompts of 8 users written to the cache
        {'name': 'append_prompts', 'op': 'append', 'tokens': 16000, 'per_sequence': 2000, 'q_heads': 32, 'kv_heads': 8, 'dim': 128, 'rotary': 64,
         'layout': 'interleaved', 'dtype': 'bf16', 'page_size': 32, 'start': 0, 'padded': 0},
        # one user at the beginning of a conversation: latency
        {'name': 'attention_first_tokens', 'op': 'attention', 'sequences': 1, 'shortest': 37, 'longest': 37, 'q_heads': 32, 'kv_heads': 8, 'dim': 128,
         'dtype': 'f16', 'page_size': 16, 'window': 0, 'padded': 0, 'wide': True},
        # 16 users, ragged, in a batch padded to a captured size
        {'name': 'attention_batch', 'op': 'attention', 'sequences': 16, 'shortest': 1, 'longest': 4096, 'q_heads': 32, 'kv_heads': 8, 'dim': 128,
         'dtype': 'f16', 'page_size': 16, 'window': 0, 'padded': 2, 'wide': True},
        # one user with a long document
        {'name': 'attention_long', 'op': 'attention', 'sequences': 1, 'shortest': 131_071, 'longest': 131_071, 'q_heads': 32, 'kv_heads': 8, 'dim': 128,
         'dtype': 'bf16', 'page_size': 64, 'window': 0, 'padded': 0, 'wide': False},
        # a full server: 96 users, ragged up to 8192 tokens
        {'name': 'attention_server', 'op': 'attention', 'sequences': 96, 'shortest': 17, 'longest': 8192, 'q_heads': 32, 'kv_heads': 8, 'dim': 128,
         'dtype': 'f16', 'page_size': 16, 'window': 0, 'padded': 0, 'wide': False},
        # full precision, every query head with its own keys, small heads, an odd page size and a window
        {'name': 'attention_f32', 'op': 'attention', 'sequences': 9, 'shortest': 100, 'longest': 4096, 'q_heads': 16, 'kv_heads': 16, 'dim': 64,
         'dtype': 'f32', 'page_size': 24, 'window': 2048, 'padded': 0, 'wide': True},
        # a beam of 8 forks: the last page of each in 32 layers' keys and values
        {'name': 'pages_fork', 'op': 'pages', 'planes': 64, 'pages': 256, 'pairs': 8, 'kv_heads': 8, 'page_size': 16, 'dim': 128, 'dtype': 'f16'},
        # compacting a cache after many users left
        {'name': 'pages_compact', 'op': 'pages', 'planes': 32, 'pages': 1600, 'pairs': 600, 'kv_heads': 8, 'page_size': 16, 'dim': 128, 'dtype': 'f16'},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(('rotary', 'rotary', 'append', 'attention', 'attention', 'attention', 'pages'))
    dtype = rng.choice(('f16', 'bf16', 'f32'))
    vector = 16 // BYTES[dtype]
    if op == 'rotary':
        heads, dim = rng.randint(1, 48), rng.choice((16, 40, 64, 72, 80, 96, 128, 160, 192, 256))
        most = max(1, min(16384, 16384 * 40 * 128 // (heads * dim) * 2 // BYTES[dtype]))
        return {'op': op, 'backward': rng.random() < 0.5, 'tokens': _log(rng, 1, most), 'heads': heads, 'dim': dim, 'rotary': 2 * rng.randint(1, dim // 2),
                'layout': rng.choice(('half', 'interleaved')), 'dtype': dtype, 'far': _log(rng, 100, 1_000_000),
                'scaling': rng.choice(('none', 'linear', 'ntk', 'yarn')), 'extra_heads': rng.choice((0, 1, 8))}
    kv_heads = rng.choice((1, 2, 3, 4, 5, 8))
    q_heads = kv_heads * rng.choice((1, 2, 4, 5, 7, 8, 12, 16))
    page_size = rng.choice((1, 8, 16, 16, 24, 32, 50, 64, 128))
    dim = rng.choice((vector * rng.randint(2, 256 // vector), 64, 80, 96, 128, 128, 256))
    if op == 'append':
        per_sequence = _log(rng, 1, 2000)
        most = max(per_sequence, 16000 * 48 * 128 * 2 // ((q_heads + 2 * kv_heads) * dim * BYTES[dtype]))
        tokens = per_sequence * max(1, _log(rng, 1, most) // per_sequence)
        return {'op': op, 'tokens': tokens, 'per_sequence': per_sequence, 'q_heads': q_heads, 'kv_heads': kv_heads, 'dim': dim,
                'rotary': 2 * rng.randint(1, dim // 2), 'layout': rng.choice(('half', 'interleaved')), 'dtype': dtype, 'page_size': page_size,
                'start': rng.choice((0, 0, 7, 1000)), 'padded': rng.choice((0, 0, 1, 5))}
    if op == 'attention':
        # the longest row of every sequence counts: the plain form gathers all of them to it
        token_bytes = 2 * kv_heads * dim * BYTES[dtype]
        longest = _log(rng, 1, min(131_072, 1_400_000_000 // token_bytes))
        sequences = _log(rng, 1, max(1, min(256, 1_400_000_000 // (token_bytes * longest), 25_000_000 // (q_heads * longest), 1_000_000 // longest)))
        return {'op': op, 'sequences': sequences, 'shortest': rng.randint(0, longest), 'longest': longest, 'q_heads': q_heads, 'kv_heads': kv_heads,
                'dim': dim, 'dtype': dtype, 'page_size': page_size, 'window': rng.choice((0, 0, 0, _log(rng, 1, 2 * longest))),
                'padded': rng.choice((0, 0, 1, 4)) if sequences > 4 else 0, 'wide': rng.random() < 0.5}
    page_bytes = kv_heads * page_size * dim * BYTES[dtype]
    planes = _log(rng, 1, 64)
    pairs = _log(rng, 1, max(1, min(1000, 700_000_000 // (planes * page_bytes))))
    return {'op': op, 'planes': planes, 'pages': 2 * pairs + rng.randint(0, 1 + pairs // 2), 'pairs': pairs, 'kv_heads': kv_heads, 'page_size': page_size,
            'dim': dim, 'dtype': dtype}


def _lengths(case):
    """The sequences' lengths: spread between the shortest and the longest by the golden ratio, the same for every seed but for their order."""
    low, high, count = case['shortest'], case['longest'], case['sequences']
    return [high if i == 0 else low + int((high - low) * ((i * 0.6180339887498949) % 1.0)) for i in range(count)]


def _frequencies(rotary, scaling, base=10000.0, factor=8.0, original=4096.0):
    """Radians per position of each pair, and the amplitude, for the scalings of long contexts."""
    pairs = torch.arange(rotary // 2, dtype=torch.float64)
    if scaling == 'ntk':
        base = base * factor ** (rotary / max(rotary - 2, 1))
    w = base ** (-2.0 * pairs / rotary)
    if scaling == 'linear':
        w = w / factor
    if scaling == 'yarn':
        turns = original * w / (2 * math.pi)   # turns within the trained length: many keep their frequency, few are stretched
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        w = w * keep + w / factor * (1.0 - keep)
        return w, 0.1 * math.log(factor) + 1.0
    return w, 1.0


def prepare(case, seed):
    device = torch.device('cuda', 0)
    g = torch.Generator(device=device).manual_seed(seed)
    order = random.Random(seed)
    dtype = DTYPES[case['dtype']]

    def normal(*shape):
        return torch.randn(shape, device=device, dtype=dtype, generator=g)

    state = dict(case)
    if case['op'] == 'rotary':
        w, amplitude = _frequencies(case['rotary'], case['scaling'])
        # heads of a wider projection, the other heads beside them
        whole = normal(case['tokens'], case['heads'] + case['extra_heads'], case['dim'])
        state['x'] = whole[:, :case['heads']]
        first = max(0, case['far'] - case['tokens'])
        state['positions'] = torch.arange(first, first + case['tokens'], device=device) % max(case['far'], 1)
        state['frequencies'], state['amplitude'] = w.to(device), amplitude
        return state
    if case['op'] == 'pages':
        state['pool'] = normal(case['planes'], case['pages'], case['kv_heads'], case['page_size'], case['dim'])
        chosen = list(range(case['pages']))
        order.shuffle(chosen)
        state['sources'] = torch.tensor(chosen[:case['pairs']], dtype=torch.int32, device=device)
        state['destinations'] = torch.tensor(chosen[case['pairs']:2 * case['pairs']], dtype=torch.int32, device=device)
        return state

    size, kv_heads, dim = case['page_size'], case['kv_heads'], case['dim']
    if case['op'] == 'append':
        count = case['tokens'] // case['per_sequence']
        ends = [case['start'] + case['per_sequence']] * count
    else:
        ends = _lengths(case)
        order.shuffle(ends)
    width = max(1, -(-max(ends) // size))
    needed = torch.tensor([-(-end // size) for end in ends], device=device)
    used = int(needed.sum())
    # pages handed out in no order, as after a while of serving; one is nobody's
    pages = torch.randperm(used + 1, device=device, generator=g).int()
    state['tables'] = torch.zeros(len(ends), width, dtype=torch.int32, device=device)
    state['tables'][torch.arange(width, device=device)[None, :] < needed[:, None]] = pages[:used]
    state['spare'] = pages[used].long()
    pool = normal(2, used + 1, kv_heads, size, dim)
    state['k_pages'], state['v_pages'] = pool[0], pool[1]
    padded = [-1] * case['padded']
    if case['op'] == 'append':
        w, state['amplitude'] = _frequencies(case['rotary'], 'none')
        state['frequencies'] = w.to(device)
        each = torch.arange(case['start'], case['start'] + case['per_sequence'], device=device, dtype=torch.int32)
        state['positions'] = torch.cat([each.repeat(len(ends)), torch.zeros(case['padded'], dtype=torch.int32, device=device)])
        owner = torch.arange(len(ends), device=device, dtype=torch.int32).repeat_interleave(case['per_sequence'])
        state['rows'] = torch.cat([owner, torch.tensor(padded, dtype=torch.int32, device=device)])
        projected = normal(case['tokens'] + case['padded'], case['q_heads'] + 2 * kv_heads, dim)
        state['q'] = projected[:, :case['q_heads']]
        state['k'] = projected[:, case['q_heads']:case['q_heads'] + kv_heads]
        state['v'] = projected[:, case['q_heads'] + kv_heads:]
        return state
    state['lengths'] = torch.tensor(ends, dtype=torch.int32, device=device)
    served = list(range(len(ends))) + padded
    order.shuffle(served)
    state['rows'] = torch.tensor(served, dtype=torch.int32, device=device)
    state['q'] = normal(len(served), case['q_heads'], dim)
    state['scale'] = 1.0 / math.sqrt(dim)
    state['out'] = torch.empty(len(served), case['q_heads'], dim, device=device, dtype=torch.float32 if case['wide'] else dtype)
    return state


def _rotated(x, positions, frequencies, amplitude, layout, sign):
    angle = positions.double()[:, None] * frequencies[None, :]   # 64 bits: far positions lose their angle in 32
    cos = (angle.cos() * amplitude).float()[:, None, :]
    sin = (angle.sin() * (sign * amplitude)).float()[:, None, :]
    half = frequencies.numel()
    wide = x.float()
    turned, rest = wide[..., :2 * half], wide[..., 2 * half:]
    if layout == 'half':
        a, b = turned[..., :half], turned[..., half:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2), rest], dim=-1)
    return y.to(x.dtype)


def _plain_append(s):
    q = _rotated(s['q'], s['positions'], s['frequencies'], s['amplitude'], s['layout'], 1.0)
    k = _rotated(s['k'], s['positions'], s['frequencies'], s['amplitude'], s['layout'], 1.0)
    rows, positions, size = s['rows'].long(), s['positions'].long(), s['page_size']
    kept = rows >= 0
    page = s['tables'][rows.clamp(min=0), positions // size].long()
    # a padded token writes back what the page that is nobody's holds
    page, slot = torch.where(kept, page, s['spare']), torch.where(kept, positions % size, 0)
    for pages, values in ((s['k_pages'], k), (s['v_pages'], s['v'])):
        pages[page, :, slot] = torch.where(kept[:, None, None], values, pages[s['spare'], :, 0])
    return {'q': q, 'k_pages': s['k_pages'], 'v_pages': s['v_pages']}


def _plain_attention(s):
    rows = s['rows'].long()
    kept = rows >= 0
    rows = rows.clamp(min=0)
    lengths = torch.where(kept, s['lengths'][rows], torch.zeros_like(s['lengths'][rows])).long()
    pages = s['tables'][rows].long()
    count, width = pages.shape
    group, size, dim = s['q_heads'] // s['kv_heads'], s['page_size'], s['dim']
    longest = width * size
    k = s['k_pages'][pages].float().permute(0, 2, 1, 3, 4).reshape(count, s['kv_heads'], longest, dim)
    scores = (s['q'].float() * s['scale']).reshape(count, s['kv_heads'], group, dim) @ k.transpose(-1, -2)
    del k
    token = torch.arange(longest, device=rows.device)[None, :]
    first = (lengths - s['window']).clamp(min=0) if s['window'] else torch.zeros_like(lengths)
    seen = (token < lengths[:, None]) & (token >= first[:, None])
    scores = scores.masked_fill(~seen[:, None, None, :], float('-inf'))
    top = scores.amax(dim=-1, keepdim=True)
    p = (scores - top.masked_fill(top == float('-inf'), 0.0)).exp()
    del scores
    total = p.sum(dim=-1, keepdim=True)
    p = p / total.masked_fill(total == 0.0, 1.0)
    v = s['v_pages'][pages].float().permute(0, 2, 1, 3, 4).reshape(count, s['kv_heads'], longest, dim)
    v = v.masked_fill(~seen[:, None, :, None], 0.0)   # what is not seen may hold anything
    return (p @ v).reshape(count, s['q_heads'], dim).to(s['out'].dtype)


def _framework(s):
    from deuteron_b200 import ops
    if s['op'] == 'rotary':
        call = ops.rotary_backward if s['backward'] else ops.rotary
        return call(s['x'], s['positions'], s['frequencies'], layout=s['layout'], amplitude=s['amplitude'])
    if s['op'] == 'append':
        q = ops.paged_append(s['k'], s['v'], s['k_pages'], s['v_pages'], s['tables'], s['rows'], s['positions'], frequencies=s['frequencies'],
                             layout=s['layout'], amplitude=s['amplitude'], q=s['q'])
        return {'q': q, 'k_pages': s['k_pages'], 'v_pages': s['v_pages']}
    if s['op'] == 'attention':
        return ops.paged_attention(s['q'], s['k_pages'], s['v_pages'], s['tables'], s['lengths'], s['scale'], rows=s['rows'], window=s['window'],
                                   out=s['out'])
    ops.copy_pages(s['pool'], s['sources'], s['destinations'])
    return s['pool']


def run(state):
    if own:
        return _framework(state)
    if state['op'] == 'rotary':
        return _rotated(state['x'], state['positions'], state['frequencies'], state['amplitude'], state['layout'], -1.0 if state['backward'] else 1.0)
    if state['op'] == 'append':
        return _plain_append(state)
    if state['op'] == 'attention':
        return _plain_attention(state)
    state['pool'][:, state['destinations'].long()] = state['pool'][:, state['sources'].long()]
    return state['pool']


def work(case):
    e = BYTES[case['dtype']]
    if case['op'] == 'rotary':
        return {'bytes': 2 * case['tokens'] * case['heads'] * case['dim'] * e + 8 * case['tokens'] + 4 * case['rotary'],
                'flops': 3 * case['tokens'] * case['heads'] * case['rotary']}
    if case['op'] == 'append':
        kv, q = 2 * case['tokens'] * case['kv_heads'] * case['dim'], (case['tokens'] + case['padded']) * case['q_heads'] * case['dim']
        return {'bytes': 2 * (kv + q) * e + 12 * case['tokens'] + 4 * case['rotary'], 'flops': 3 * case['tokens'] * (case['q_heads'] + case['kv_heads']) * case['rotary']}
    if case['op'] == 'attention':
        tokens = sum(min(n, case['window'] or n) for n in _lengths(case))
        rows = (case['sequences'] + case['padded']) * case['q_heads'] * case['dim']
        return {'bytes': 2 * tokens * case['kv_heads'] * case['dim'] * e + rows * (e + (4 if case['wide'] else e)) + 4 * tokens // case['page_size'],
                'flops': 4 * tokens * case['q_heads'] * case['dim']}
    return {'bytes': 2 * case['planes'] * case['pairs'] * case['kv_heads'] * case['page_size'] * case['dim'] * e + 8 * case['pairs'], 'flops': 0}


def _turned(x, positions, frequencies, amplitude, layout, sign):
    """The rotation as a product of complex numbers in 64 bits."""
    half = frequencies.numel()
    y = x.double().clone()
    turn = torch.polar(torch.full_like(frequencies, amplitude)[None, :].expand(positions.numel(), half).contiguous(),
                       (positions.double()[:, None] * frequencies * sign))[:, None, :]
    places = (slice(0, half), slice(half, 2 * half)) if layout == 'half' else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    z = torch.complex(y[..., places[0]], y[..., places[1]]) * turn
    y[..., places[0]], y[..., places[1]] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if s['op'] == 'rotary':
        return _turned(s['x'], s['positions'], s['frequencies'], s['amplitude'], s['layout'], -1.0 if s['backward'] else 1.0)
    if s['op'] == 'pages':
        pool = s['pool'].double()
        for a, b in zip(s['sources'].tolist(), s['destinations'].tolist()):
            pool[:, b] = pool[:, a]
        return pool
    if s['op'] == 'append':
        q, k = (_turned(s[n], s['positions'], s['frequencies'], s['amplitude'], s['layout'], 1.0) for n in ('q', 'k'))
        k_pages, v_pages, tables = s['k_pages'].double(), s['v_pages'].double(), s['tables'].tolist()
        places = [(t, tables[r][p // s['page_size']], p % s['page_size']) for t, (r, p) in enumerate(zip(s['rows'].tolist(), s['positions'].tolist())) if r >= 0]
        if not places:
            return {'q': q, 'k_pages': k_pages, 'v_pages': v_pages}
        token, page, slot = (torch.tensor(x, device=q.device) for x in zip(*places))
        at = page * s['page_size'] + slot
        for pages, values in ((k_pages, k), (v_pages, s['v'].double())):
            flat = pages.transpose(1, 2).reshape(-1, s['kv_heads'], s['dim'])
            flat[at] = values[token]
            pages.copy_(flat.reshape(-1, s['page_size'], s['kv_heads'], s['dim']).transpose(1, 2))
        return {'q': q, 'k_pages': k_pages, 'v_pages': v_pages}
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device=s['q'].device)
    lengths, group = s['lengths'].tolist(), s['q_heads'] // s['kv_heads']
    for i, row in enumerate(s['rows'].tolist()):
        length = lengths[row] if row >= 0 else 0
        first = max(0, length - s['window']) if s['window'] else 0
        if length == 0:
            continue
        used = s['tables'][row, :-(-length // s['page_size'])].long()
        k, v = (s[n][used].transpose(0, 1).reshape(s['kv_heads'], -1, s['dim'])[:, first:length].double() for n in ('k_pages', 'v_pages'))
        q = s['q'][i].double().reshape(s['kv_heads'], group, s['dim'])
        p = torch.softmax(torch.einsum('hgd,htd->hgt', q, k) * s['scale'], dim=-1)
        out[i] = torch.einsum('hgt,htd->hgd', p, v).reshape(s['q_heads'], s['dim'])
    return out
