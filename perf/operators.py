"""What is timed of the paged key-value cache and of rotary positions with several axes.

Every case is a dict of plain values with a ``kind``:

* ``attend``  one new token of every request over a key-value cache kept in pages
              (``paged_attention``), with or without a mask;
* ``write``   new key/value rows into their pages (``paged_write``): a decode step's one token
              per request, or a padded batch of prompts;
* ``rotary``  queries and keys rotated by positions of several axes (``rotary_axes``).

Pages are handed out in random order, as a server that has run for a while has them; table
entries past a request's pages hold -1.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DEVICE = 'cuda'
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
SIZES = {'bf16': 2, 'fp16': 2, 'fp32': 4, 'bool': 1}
THETA = 1_000_000.0


def listed():
    return [
        # one user alone on the server, 300 tokens into speech: latency
        dict(name='attend_1', kind='attend', batch=1, low=299, high=299, page=16, q_heads=16, kv_heads=8, width=128,
             dtype='bf16', mask='none'),
        # the talker's step: 64 requests somewhere between 64 and 1023 tokens into speech
        dict(name='attend_64', kind='attend', batch=64, low=64, high=1023, page=16, q_heads=16, kv_heads=8, width=128,
             dtype='bf16', mask='none'),
        # a full server of long conversations: HBM
        dict(name='attend_128_long', kind='attend', batch=128, low=100, high=4095, page=64, q_heads=32, kv_heads=8,
             width=128, dtype='bf16', mask='none'),
        # one long document: the cache's length split over the card
        dict(name='attend_1_long', kind='attend', batch=1, low=65000, high=65000, page=256, q_heads=28, kv_heads=4,
             width=128, dtype='fp16', mask='none'),
        # a float32 model with narrow heads under a mask that hides keys, one request's all of them;
        # pages of an odd size
        dict(name='attend_21_masked', kind='attend', batch=21, low=1, high=700, page=24, q_heads=12, kv_heads=12,
             width=64, dtype='fp32', mask='bool'),
        # a bf16 model handed an additive mask of the type's lowest value, one request all of it
        dict(name='attend_32_lowest', kind='attend', batch=32, low=30, high=2047, page=32, q_heads=32, kv_heads=4,
             width=128, dtype='bf16', mask='lowest'),
        # the keys and values of a 64-request decode step
        dict(name='write_64', kind='write', batch=64, tokens=1, low=1, high=1, start=1000, page=16, kv_heads=8, width=128,
             dtype='bf16'),
        # an admission burst: 16 prompts, right-padded, into fresh pages
        dict(name='write_16_prompts', kind='write', batch=16, tokens=1024, low=60, high=1024, start=0, page=16, kv_heads=8,
             width=128, dtype='bf16'),
        # rotary of a 64-request decode step, the talker's sections
        dict(name='rotary_64', kind='rotary', batch=64, tokens=1, q_heads=16, kv_heads=8, width=128, sections='24 20 20',
             interleaved=True, far=4096, dtype='bf16'),
        # a batch of images and videos: every token at its own (time, height, width)
        dict(name='rotary_images', kind='rotary', batch=4, tokens=4099, q_heads=28, kv_heads=4, width=128,
             sections='16 24 24', interleaved=False, far=300, dtype='bf16'),
        # a float32 model with a part of each head rotated, far into a stream
        dict(name='rotary_far', kind='rotary', batch=2, tokens=777, q_heads=12, kv_heads=12, width=64, sections='8 4 4',
             interleaved=False, far=1 << 24, dtype='fp32'),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(['attend', 'attend', 'attend', 'write', 'rotary', 'rotary'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    width = rng.choice([64, 128, 128])
    if kind == 'attend':
        q_heads, kv_heads = rng.choice([(16, 8), (32, 8), (8, 8), (28, 4), (12, 12), (16, 1), (32, 4), (40, 2), (3, 3)])
        batch = _log_int(rng, 1, 200)
        # never more bytes than the largest listed case reads
        most = 128 * 2000 * 8 * 128 * 2 // (batch * kv_heads * width * SIZES[dtype])
        high = _log_int(rng, 1, min(65536, most)) - 1
        return dict(kind=kind, batch=batch, low=rng.randrange(0, high + 1), high=high,
                    page=rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 256]), q_heads=q_heads, kv_heads=kv_heads,
                    width=width, dtype=dtype, mask=rng.choice(['none', 'none', 'none', 'bool', 'lowest', 'infinite']))
    if kind == 'write':
        tokens = rng.choice([1, 2, _log_int(rng, 3, 1024)])
        batch = _log_int(rng, 1, 256 if tokens < 3 else max(1, 16384 // tokens))
        low = rng.randrange(1, tokens + 1)
        return dict(kind=kind, batch=batch, tokens=tokens, low=low, high=tokens, start=rng.randrange(0, 2048),
                    page=rng.choice([1, 8, 16, 24, 64, 256]), kv_heads=rng.choice([1, 2, 4, 8, 12]), width=width, dtype=dtype)
    half = rng.choice([width // 2, width // 2, width // 4])
    first = rng.randrange(1, half // 2)
    second = rng.randrange(1, (half - first) // 2 + 1)
    batch = _log_int(rng, 1, 200)
    return dict(kind='rotary', batch=batch, tokens=rng.choice([1, _log_int(rng, 1, 16384 // batch)]),
                q_heads=rng.choice([8, 12, 16, 28, 32]), kv_heads=rng.choice([1, 4, 8]), width=width,
                sections='%d %d %d' % (half - first - second, first, second), interleaved=rng.random() < 0.4,
                far=_log_int(rng, 16, 1 << 24), dtype=dtype)


# ---- inputs -------------------------------------------------------------------------------

def _normal(gen, *shape, dtype, scale=1.0):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=dtype).mul_(scale)


def _pages(counts, host):
    """A page table (B, widest) for ``counts`` pages per request, and the pool's size: pages in
    random order, some left free."""
    total = int(counts.sum())
    pool = total + 1 + total // 8
    order = torch.randperm(pool, generator=host)[:total].to(torch.int32)
    table = torch.full((len(counts), int(counts.max())), -1, dtype=torch.int32)
    table[torch.arange(table.shape[1])[None] < counts[:, None]] = order
    return table, pool


def _contexts(case):
    """Position of every request's token: the case's own, whatever the seed, so that every pass of a
    case is the same work."""
    gen = torch.Generator().manual_seed(7)
    return torch.randint(case['low'], case['high'] + 1, (case['batch'],), generator=gen)


def _mask(case, contexts, capacity, host):
    """(B, 1, 1, capacity): about a quarter of the keys hidden, and the first request's all of them
    when there are several."""
    hidden = torch.rand(case['batch'], capacity, generator=host) < 0.25
    if case['batch'] > 1:
        hidden[0] = True
        # a request that the mask leaves something keeps its newest key
        hidden[torch.arange(1, case['batch']), contexts[1:]] = False
    if case['mask'] == 'bool':
        return ~hidden[:, None, None]
    # an additive mask in the cache's type, or, in 16 bits with fp16, in bf16: the lowest fp16 is not
    # far enough from the scores to stand for hidden
    dtype = torch.bfloat16 if case['dtype'] == 'fp16' else TYPES[case['dtype']]
    low = torch.finfo(dtype).min if case['mask'] == 'lowest' else -math.inf
    return torch.zeros(hidden.shape, dtype=dtype).masked_fill(hidden, low)[:, None, None]


def _attend_inputs(case, seed):
    host, gen = torch.Generator().manual_seed(seed), torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, batch, page = TYPES[case['dtype']], case['batch'], case['page']
    contexts = _contexts(case)[torch.randperm(batch, generator=host)]
    table, pool = _pages(contexts // page + 1, host)
    s = SimpleNamespace(contexts=contexts, page=page, mask=None)
    s.key_pages = _normal(gen, pool, case['kv_heads'], page, case['width'], dtype=dtype)
    s.value_pages = _normal(gen, pool, case['kv_heads'], page, case['width'], dtype=dtype)
    s.query = _normal(gen, batch, 1, case['q_heads'], case['width'], dtype=dtype, scale=2.0)
    if case['mask'] != 'none':
        s.mask = _mask(case, contexts, table.shape[1] * page, host).to(DEVICE)
    s.table, s.positions = table.to(DEVICE), contexts.to(DEVICE)
    return s


def _write_inputs(case, seed):
    host, gen = torch.Generator().manual_seed(seed), torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, batch, tokens, page = TYPES[case['dtype']], case['batch'], case['tokens'], case['page']
    # the case's own lengths and starts, in the seed's order
    own_gen, order = torch.Generator().manual_seed(7), torch.randperm(batch, generator=host)
    lengths = torch.randint(case['low'], case['high'] + 1, (batch,), generator=own_gen)[order]
    starts = torch.randint(0, case['start'] + 1, (batch,), generator=own_gen)[order]
    table, pool = _pages((starts + lengths + page - 1) // page, host)
    s = SimpleNamespace(page=page, tokens=tokens)
    s.key_pages = _normal(gen, pool, case['kv_heads'], page, case['width'], dtype=dtype)
    s.value_pages = _normal(gen, pool, case['kv_heads'], page, case['width'], dtype=dtype)
    # rows of the fused projection (B, tokens, 2 * heads, width), as views in (B, heads, tokens, width)
    rows = _normal(gen, batch, tokens, 2 * case['kv_heads'], case['width'], dtype=dtype)
    s.keys = rows[:, :, :case['kv_heads']].transpose(1, 2)
    s.values = rows[:, :, case['kv_heads']:].transpose(1, 2)
    s.table, s.starts = table.to(DEVICE), starts.to(DEVICE)
    s.lengths = lengths.to(DEVICE, torch.int32) if tokens > 1 else None
    return s


def _rotary_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, batch, tokens = TYPES[case['dtype']], case['batch'], case['tokens']
    heads = case['q_heads'] + case['kv_heads']
    rows = _normal(gen, batch, tokens, heads, case['width'], dtype=dtype)
    s = SimpleNamespace(query=rows[:, :, :case['q_heads']], key=rows[:, :, case['q_heads']:])
    s.positions = torch.randint(0, case['far'], (3, batch, tokens), generator=gen, device=DEVICE)
    s.sections, s.interleaved = tuple(map(int, case['sections'].split())), case['interleaved']
    return s


def prepare(case, seed):
    return {'attend': _attend_inputs, 'write': _write_inputs, 'rotary': _rotary_inputs}[case['kind']](case, seed)


# ---- one pass -----------------------------------------------------------------------------

def _attend(s):
    """Every request's keys gathered into one padded batch, then softmax attention in float32."""
    batch, _, q_heads, width = s.query.shape
    kv_heads = s.key_pages.shape[1]
    capacity = s.table.shape[1] * s.page
    keys = torch.arange(capacity, device=DEVICE)
    pages, rows = s.table.long()[:, keys // s.page].clamp(min=0)[:, None], keys % s.page
    heads = torch.arange(kv_heads, device=DEVICE)[:, None]
    k, v = s.key_pages[pages, heads, rows].float(), s.value_pages[pages, heads, rows].float()  # (B, heads, keys, width)
    q = s.query.float().reshape(batch, kv_heads, q_heads // kv_heads, width)
    scores = torch.matmul(q, k.transpose(2, 3)) * width ** -0.5
    hidden = (keys[None] > s.positions[:, None])[:, None, None]
    if s.mask is not None and s.mask.dtype == torch.bool:
        hidden = hidden | ~s.mask
    elif s.mask is not None:
        scores = scores + s.mask.float()
    scores = scores.masked_fill(hidden, -math.inf)
    highest = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - highest.masked_fill(highest == -math.inf, 0.0))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, v) / total.masked_fill(total == 0, 1.0)
    return out.reshape(batch, 1, q_heads, width).to(s.query.dtype)


def _write(s):
    """The rows that a request has, each to its page and row."""
    tokens = torch.arange(s.tokens, device=DEVICE)
    at = s.starts[:, None] + tokens
    pages = s.table.long().gather(1, (at // s.page).clamp(max=s.table.shape[1] - 1))
    pages, rows = pages[:, None], (at % s.page)[:, None]
    heads = torch.arange(s.keys.shape[1], device=DEVICE)[None, :, None]
    if s.lengths is None:
        s.key_pages[pages, heads, rows] = s.keys
        s.value_pages[pages, heads, rows] = s.values
    else:
        used = (tokens < s.lengths[:, None])[:, None].expand(s.keys.shape[:3])
        at = pages.expand(used.shape)[used], heads.expand(used.shape)[used], rows.expand(used.shape)[used]
        s.key_pages[at] = s.keys[used]
        s.value_pages[at] = s.values[used]
    return s.key_pages, s.value_pages


def _axis_of(sections, interleaved):
    """The axis of every frequency."""
    half, frequency = sum(sections), torch.arange(sum(sections), device=DEVICE)
    if not interleaved:
        return torch.bucketize(frequency, torch.tensor(sections, device=DEVICE).cumsum(0), right=True)
    axis, limits = frequency % len(sections), torch.tensor(sections, device=DEVICE) * len(sections)
    return torch.where(frequency < limits[axis], axis, torch.zeros(half, dtype=torch.long, device=DEVICE))


def _rotate(x, cos, sin):
    half = cos.shape[-1]
    first, second = x[..., :half].float(), x[..., half:2 * half].float()
    turned = torch.cat((first * cos - second * sin, second * cos + first * sin, x[..., 2 * half:].float()), -1)
    return turned.to(x.dtype)


def _rotary(s):
    half = sum(s.sections)
    frequency = THETA ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
    position = s.positions[_axis_of(s.sections, s.interleaved)].permute(1, 2, 0)
    angle = position.double() * frequency  # float32 would be off by radians at far positions
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    return _rotate(s.query, cos, sin), _rotate(s.key, cos, sin)


def _package():
    import __graft_entry__
    return __graft_entry__.import_package()


def run(state):
    s = state
    if hasattr(s, 'sections'):
        if own:
            return _package().rotary_axes(s.query, s.key, s.positions, s.sections, interleaved=s.interleaved, theta=THETA)
        return _rotary(s)
    if hasattr(s, 'keys'):
        if own:
            _package().paged_write(s.keys, s.values, s.key_pages, s.value_pages, s.table, s.starts, s.lengths)
            return s.key_pages, s.value_pages
        return _write(s)
    if own:
        return _package().paged_attention(s.query, s.key_pages, s.value_pages, s.table, s.positions, mask=s.mask)
    return _attend(s)


def work(case):
    size, width = SIZES[case['dtype']], case['width']
    if case['kind'] == 'attend':
        keys = int((_contexts(case) + 1).sum())
        rows = 2 * case['batch'] * case['q_heads'] * width * size
        mask = 0 if case['mask'] == 'none' else keys * (1 if case['mask'] == 'bool' else size)
        pages = int((_contexts(case) // case['page'] + 1).sum()) * 4
        return {'bytes': keys * case['kv_heads'] * 2 * width * size + rows + mask + pages + 8 * case['batch'],
                'flops': 4 * keys * case['q_heads'] * width}
    if case['kind'] == 'write':
        gen = torch.Generator().manual_seed(7)
        rows = int(torch.randint(case['low'], case['high'] + 1, (case['batch'],), generator=gen).sum())
        return {'bytes': 2 * 2 * rows * case['kv_heads'] * width * size, 'flops': 0}
    tokens, heads = case['batch'] * case['tokens'], case['q_heads'] + case['kv_heads']
    return {'bytes': 2 * tokens * heads * width * size + 24 * tokens, 'flops': 3 * tokens * heads * width}


# ---- in 64 bits ----------------------------------------------------------------------------

def _exact_attend(s):
    batch, _, q_heads, width = s.query.shape
    kv_heads = s.key_pages.shape[1]
    out = torch.zeros(batch, 1, q_heads, width, device=DEVICE, dtype=torch.float64)
    for b in range(batch):
        length = int(s.contexts[b]) + 1
        pages = s.table[b, :(length + s.page - 1) // s.page].long()
        for h in range(kv_heads):
            k = s.key_pages[pages, h].reshape(-1, width)[:length].double()
            v = s.value_pages[pages, h].reshape(-1, width)[:length].double()
            group = slice(h * (q_heads // kv_heads), (h + 1) * (q_heads // kv_heads))
            scores = (s.query[b, 0, group].double() @ k.T) / math.sqrt(width)
            if s.mask is not None:
                term = s.mask[b, 0, 0, :length]
                shown = term if term.dtype == torch.bool else term != -math.inf
                if not bool(shown.any()):
                    continue
                scores, v = scores[:, shown], v[shown]
                if term.dtype != torch.bool:
                    scores = scores + term[shown].double()
            out[b, 0, group] = torch.softmax(scores, -1) @ v
    return out


def _exact_write(s):
    pools = [s.key_pages.double(), s.value_pages.double()]
    for b in range(s.keys.shape[0]):
        count = s.tokens if s.lengths is None else int(s.lengths[b])
        at = int(s.starts[b]) + torch.arange(count, device=DEVICE)
        page = s.table[b].long()[torch.div(at, s.page, rounding_mode='floor')]
        for pool, rows in zip(pools, (s.keys, s.values)):
            pool[page, :, at % s.page] = rows[b, :, :count].double().transpose(0, 1)
    return tuple(pools)


def _exact_rotary(s):
    half, axes = sum(s.sections), len(s.sections)
    outs = [s.query.double(), s.key.double()]
    for i in range(half):
        axis = 0
        if s.interleaved:
            if i < axes * s.sections[i % axes]:
                axis = i % axes
        else:
            while i >= sum(s.sections[:axis + 1]):
                axis += 1
        angle = (s.positions[axis].double() * THETA ** (-i / half))[:, :, None]
        for x, y in zip((s.query, s.key), outs):
            a, b = x[..., i].double(), x[..., i + half].double()
            y[..., i] = a * torch.cos(angle) - b * torch.sin(angle)
            y[..., i + half] = b * torch.cos(angle) + a * torch.sin(angle)
    return tuple(outs)


def exact(case, seed):
    s = prepare(case, seed)
    return {'attend': _exact_attend, 'write': _exact_write, 'rotary': _exact_rotary}[case['kind']](s)
