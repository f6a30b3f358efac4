"""What is timed of the paged cache held in 8 bits and of attention over a prefix that a batch shares.

Every case is a dict of plain values with a ``kind``:

* ``attend``  one new token of every request over a paged cache of int8 or e4m3 rows, each row with
              a float32 scale (``paged_attention`` with ``scales``), with or without a mask;
* ``store``   new key/value rows quantised into their pages and read back in the rows' own type, as
              a request that is admitted and later moved elsewhere has them (``paged_write`` and
              ``paged_read`` with ``scales``); the rows that come back are the values that the
              pages stand for;
* ``read``    requests' rows gathered from their pages into padded rows (``paged_read``), out of 8
              bits or out of pages of the rows' own type;
* ``shared``  one new token of every request of a batch whose requests all begin with the same
              pages (``paged_attention`` with ``shared_pages``).

A row's scale: with a = max(|x|, 2^-100) over the row, int8 rows hold x * (127 / a) rounded to the
nearest whole number (ties to even) and the scale a / 127; e4m3 rows hold x / s rounded to the
nearest e4m3 value, s being the smallest power of two for which a / s is at most 448.  Pages are
handed out in random order, as a server that has run for a while has them; table entries past a
request's pages hold -1.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DEVICE = 'cuda'
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
STORES = {'int8': torch.int8, 'e4m3': torch.float8_e4m3fn}
SIZES = {'bf16': 2, 'fp16': 2, 'fp32': 4, 'bool': 1, 'int8': 1, 'e4m3': 1}


def listed():
    return [
        # one user alone on the server, 300 tokens into speech: latency
        dict(name='attend_1', kind='attend', batch=1, low=299, high=299, page=16, q_heads=16, kv_heads=8, width=128,
             dtype='bf16', store='int8', mask='none'),
        # the talker's step: 64 requests somewhere between 64 and 1023 tokens into speech
        dict(name='attend_64', kind='attend', batch=64, low=64, high=1023, page=16, q_heads=16, kv_heads=8, width=128,
             dtype='bf16', store='e4m3', mask='none'),
        # a full server of long conversations, which 8 bits are for: HBM
        dict(name='attend_128_long', kind='attend', batch=128, low=100, high=4095, page=64, q_heads=32, kv_heads=8,
             width=128, dtype='bf16', store='int8', mask='none'),
        # a float32 model with narrow heads under a mask that hides keys, one request's all of them;
        # pages of an odd size
        dict(name='attend_21_masked', kind='attend', batch=21, low=1, high=700, page=24, q_heads=12, kv_heads=12,
             width=64, dtype='fp32', store='e4m3', mask='bool'),
        # the keys and values of a 64-request decode step
        dict(name='store_64', kind='store', batch=64, tokens=1, low=1, high=1, start=1000, page=16, kv_heads=8, width=128,
             dtype='bf16', store='e4m3'),
        # an admission burst: 16 prompts, right-padded, into fresh pages
        dict(name='store_16_prompts', kind='store', batch=16, tokens=1024, low=60, high=1024, start=0, page=16, kv_heads=8,
             width=128, dtype='bf16', store='int8'),
        # one request leaves the paged cache for a slot of the arena
        dict(name='read_1', kind='read', batch=1, tokens=300, low=300, high=300, start=0, page=16, kv_heads=8, width=128,
             dtype='bf16', store='int8'),
        # a narrow fp16 model's whole batch is moved, ragged, from pages of an odd size
        dict(name='read_48', kind='read', batch=48, tokens=777, low=1, high=777, start=30, page=24, kv_heads=12, width=64,
             dtype='fp16', store='e4m3'),
        # a few users with one voice prompt: latency
        dict(name='shared_8', kind='shared', batch=8, prefix=512, low=0, high=300, page=16, q_heads=16, kv_heads=8,
             width=128, dtype='bf16', mask='none'),
        # the talker's step where every request carries the same 4096 tokens of instructions
        dict(name='shared_64', kind='shared', batch=64, prefix=4096, low=64, high=1023, page=16, q_heads=16, kv_heads=8,
             width=128, dtype='bf16', mask='none'),
        # many answers to one long document: matrix products
        dict(name='shared_128_long', kind='shared', batch=128, prefix=16384, low=0, high=511, page=64, q_heads=32,
             kv_heads=8, width=128, dtype='bf16', mask='none'),
        # a float32 model with narrow heads, the prefix in pages of an odd size, under a mask that hides
        # keys, one request's all of them
        dict(name='shared_21_masked', kind='shared', batch=21, prefix=792, low=0, high=400, page=24, q_heads=12,
             kv_heads=12, width=64, dtype='fp32', mask='bool'),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(['attend', 'attend', 'store', 'read', 'shared', 'shared'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    store = rng.choice(['int8', 'e4m3'])
    width = rng.choice([64, 128, 128])
    heads = [(16, 8), (32, 8), (8, 8), (28, 4), (12, 12), (16, 1), (32, 4), (40, 2), (3, 3)]
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 256])
    mask = rng.choice(['none', 'none', 'none', 'bool', 'lowest', 'infinite'])
    if kind == 'attend':
        q_heads, kv_heads = rng.choice(heads)
        batch = _log_int(rng, 1, 200)
        # never more keys than the largest listed case has
        most = 128 * 2000 * 8 * 128 // (batch * kv_heads * width)
        high = _log_int(rng, 1, min(65536, most)) - 1
        return dict(kind=kind, batch=batch, low=rng.randrange(0, high + 1), high=high, page=page, q_heads=q_heads,
                    kv_heads=kv_heads, width=width, dtype=dtype, store=store, mask=mask)
    if kind == 'shared':
        q_heads, kv_heads = rng.choice(heads)
        batch = _log_int(rng, 2, 200)
        # never more products or bytes than the largest listed case has (float32's products run at a fraction of the rate)
        most = 128 * 32 * 16384 * 128 // (16 if dtype == 'fp32' else 1) // (batch * q_heads * width)
        rows = _log_int(rng, 16, max(17, min(32768, most)))
        high = _log_int(rng, 1, max(2, min(2048, 128 * 256 * 8 * 128 * 2 // (batch * kv_heads * width * SIZES[dtype])))) - 1
        return dict(kind=kind, batch=batch, prefix=max(1, rows // page) * page, low=rng.randrange(0, high + 1), high=high,
                    page=page, q_heads=q_heads, kv_heads=kv_heads, width=width, dtype=dtype, mask=mask)
    tokens = rng.choice([1, 2, _log_int(rng, 3, 1024), _log_int(rng, 3, 1024)])
    batch = _log_int(rng, 1, 256 if tokens < 3 else max(1, 16384 // tokens))
    if kind == 'read':
        store = rng.choice(['int8', 'e4m3', dtype])
    return dict(kind=kind, batch=batch, tokens=tokens, low=rng.randrange(1, tokens + 1), high=tokens,
                start=rng.randrange(0, 2048), page=page, kv_heads=rng.choice([1, 2, 4, 8, 12]), width=width, dtype=dtype,
                store=store)


# ---- inputs -------------------------------------------------------------------------------

def _normal(gen, *shape, dtype, scale=1.0):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=dtype).mul_(scale)


def _rows(gen, *shape, dtype):
    """Normal rows, some of whose channels are several times larger, as keys' often are."""
    x = _normal(gen, *shape, dtype=dtype)
    x[..., 5::31] *= 4
    return x


def _quantised(x, store):
    """x's rows in 8 bits, and their scales, in float32 arithmetic throughout."""
    largest = x.float().abs().amax(-1).clamp(min=2.0 ** -100)
    if store == 'int8':
        inverse = torch.full_like(largest, 127.0) / largest  # (127 / largest would be 127 times the reciprocal)
        return (x.float() * inverse[..., None]).round().to(torch.int8), largest / 127
    part, exponent = torch.frexp(largest)  # part in [1/2, 1)
    exponent = exponent - torch.where(part <= 0.875, 9, 8)
    power = lambda n: (n + 127 << 23).to(torch.int32).view(torch.float32)  # 2^n, exactly
    return (x.float() * power(-exponent)[..., None]).to(torch.float8_e4m3fn), power(exponent)


def _quantised_pool(x, store):
    """_quantised in parts, so that the float32 copies stay small."""
    parts = [_quantised(part, store) for part in x.split(max(1, (1 << 26) // x[0].numel()))]
    rows = torch.cat([rows.view(torch.uint8) for rows, _ in parts]).view(STORES[store])
    return rows, torch.cat([scales for _, scales in parts])


def _pages(counts, host, shared=0):
    """A page table (B, widest) for ``counts`` pages per request behind ``shared`` pages of all, and the
    pool's size: pages in random order, some left free."""
    total = int(counts.sum()) + shared
    pool = total + 1 + total // 8
    order = torch.randperm(pool, generator=host)[:total].to(torch.int32)
    table = torch.full((len(counts), shared + int(counts.max())), -1, dtype=torch.int32)
    table[:, :shared] = order[:shared]
    table[:, shared:][torch.arange(table.shape[1] - shared)[None] < counts[:, None]] = order[shared:]
    return table, pool


def _contexts(case):
    """Position of every request's token behind the prefix: the case's own, whatever the seed, so that
    every pass of a case is the same work."""
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
    # an additive mask in the queries' type, or, in 16 bits with fp16, in bf16: the lowest fp16 is not
    # far enough from the scores to stand for hidden
    dtype = torch.bfloat16 if case['dtype'] == 'fp16' else TYPES[case['dtype']]
    low = torch.finfo(dtype).min if case['mask'] == 'lowest' else -math.inf
    return torch.zeros(hidden.shape, dtype=dtype).masked_fill(hidden, low)[:, None, None]


def _attend_inputs(case, seed):
    host, gen = torch.Generator().manual_seed(seed), torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, batch, page = TYPES[case['dtype']], case['batch'], case['page']
    shared = case.get('prefix', 0) // page
    behind = _contexts(case)[torch.randperm(batch, generator=host)]
    table, pool = _pages(behind // page + 1, host, shared)
    contexts = behind + shared * page
    s = SimpleNamespace(kind=case['kind'], contexts=contexts, page=page, shared=shared, mask=None, scales=None)
    s.key_pages = _rows(gen, pool, case['kv_heads'], page, case['width'], dtype=dtype)
    s.value_pages = _normal(gen, pool, case['kv_heads'], page, case['width'], dtype=dtype)
    if 'store' in case:
        s.key_pages, keys = _quantised_pool(s.key_pages, case['store'])
        s.value_pages, values = _quantised_pool(s.value_pages, case['store'])
        s.scales = keys, values
    s.query = _normal(gen, batch, 1, case['q_heads'], case['width'], dtype=dtype, scale=1.5)
    if case['mask'] != 'none':
        s.mask = _mask(case, contexts, table.shape[1] * page, host).to(DEVICE)
    s.table, s.positions = table.to(DEVICE), contexts.to(DEVICE)
    return s


def _store_inputs(case, seed):
    host, gen = torch.Generator().manual_seed(seed), torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, batch, tokens, page = TYPES[case['dtype']], case['batch'], case['tokens'], case['page']
    # the case's own lengths and starts, in the seed's order
    own_gen, order = torch.Generator().manual_seed(7), torch.randperm(batch, generator=host)
    lengths = torch.randint(case['low'], case['high'] + 1, (batch,), generator=own_gen)[order]
    starts = torch.randint(0, case['start'] + 1, (batch,), generator=own_gen)[order]
    table, pool = _pages((starts + lengths + page - 1) // page, host)
    s = SimpleNamespace(kind=case['kind'], page=page, tokens=tokens, dtype=dtype, scales=None)
    shape = pool, case['kv_heads'], page, case['width']
    if case['kind'] == 'store':  # pages that held other requests' rows
        s.key_pages, s.value_pages = (torch.zeros(shape, dtype=torch.uint8, device=DEVICE).view(STORES[case['store']]) for _ in range(2))
        s.scales = tuple(torch.ones(shape[:3], device=DEVICE) for _ in range(2))
        # rows of the fused projection (B, tokens, 2 * heads, width), as views in (B, heads, tokens, width)
        rows = _rows(gen, batch, tokens, 2 * case['kv_heads'], case['width'], dtype=dtype)
        s.keys = rows[:, :, :case['kv_heads']].transpose(1, 2)
        s.values = rows[:, :, case['kv_heads']:].transpose(1, 2)
    else:
        s.key_pages, s.value_pages = _rows(gen, *shape, dtype=dtype), _normal(gen, *shape, dtype=dtype)
        if case['store'] in STORES:
            s.key_pages, keys = _quantised_pool(s.key_pages, case['store'])
            s.value_pages, values = _quantised_pool(s.value_pages, case['store'])
            s.scales = keys, values
    s.store = case['store']
    s.table, s.starts = table.to(DEVICE), starts.to(DEVICE)
    s.lengths = lengths.to(DEVICE, torch.int32) if tokens > 1 else None
    return s


def prepare(case, seed):
    return (_attend_inputs if case['kind'] in ('attend', 'shared') else _store_inputs)(case, seed)


# ---- one pass -----------------------------------------------------------------------------

def _gathered(pool, scales, pages, heads, rows):
    """Rows of a pool in float32, as the values that they stand for."""
    if scales is None:
        return pool[pages, heads, rows].float()
    held = pool.view(torch.uint8)[pages, heads, rows].view(pool.dtype).float()
    return held * scales[pages, heads, rows][..., None]


def _attend(s):
    """The shared prefix' keys once, every request's others gathered into one padded batch; then softmax
    attention in float32."""
    batch, _, q_heads, width = s.query.shape
    kv_heads = s.key_pages.shape[1]
    group = q_heads // kv_heads
    capacity, first = s.table.shape[1] * s.page, s.shared * s.page
    keys = torch.arange(capacity, device=DEVICE)
    heads = torch.arange(kv_heads, device=DEVICE)[:, None]
    key_scales, value_scales = s.scales if s.scales else (None, None)
    pages, rows = s.table.long()[:, keys[first:] // s.page].clamp(min=0)[:, None], keys[first:] % s.page
    k = _gathered(s.key_pages, key_scales, pages, heads, rows)  # (B, heads, keys, width)
    v = _gathered(s.value_pages, value_scales, pages, heads, rows)
    q = s.query.float().reshape(batch, kv_heads, group, width)
    scores = torch.matmul(q, k.transpose(2, 3))
    if first:
        pages, rows = s.table[0].long()[keys[:first] // s.page], keys[:first] % s.page
        prefix_k = _gathered(s.key_pages, key_scales, pages, heads, rows)  # (heads, keys, width)
        prefix_v = _gathered(s.value_pages, value_scales, pages, heads, rows)
        columns = q.transpose(0, 1).reshape(kv_heads, batch * group, width)
        prefix = torch.matmul(columns, prefix_k.transpose(1, 2)).reshape(kv_heads, batch, group, first)
        scores = torch.cat((prefix.transpose(0, 1), scores), -1)
    scores = scores * width ** -0.5
    hidden = (keys[None] > s.positions[:, None])[:, None, None]
    if s.mask is not None and s.mask.dtype == torch.bool:
        hidden = hidden | ~s.mask
    elif s.mask is not None:
        scores = scores + s.mask.float()
    scores = scores.masked_fill(hidden, -math.inf)
    highest = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - highest.masked_fill(highest == -math.inf, 0.0))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights[..., first:], v)
    if first:
        columns = weights[..., :first].transpose(0, 1).reshape(kv_heads, batch * group, first)
        out = out + torch.matmul(columns, prefix_v).reshape(kv_heads, batch, group, width).transpose(0, 1)
    return (out / total.masked_fill(total == 0, 1.0)).reshape(batch, 1, q_heads, width).to(s.query.dtype)


def _places(s):
    """(pages, heads, rows) of the rows of every request, (B, heads, tokens), and which of them it has."""
    tokens = torch.arange(s.tokens, device=DEVICE)
    at = s.starts[:, None] + tokens
    pages = s.table.long().gather(1, (at // s.page).clamp(max=s.table.shape[1] - 1))[:, None]
    heads = torch.arange(s.key_pages.shape[1], device=DEVICE)[None, :, None]
    used = None if s.lengths is None else (tokens < s.lengths[:, None])[:, None]
    return pages, heads, (at % s.page)[:, None], used


def _write(s):
    """The rows that a request has, each to its page and row."""
    pages, heads, rows, used = _places(s)
    for x, pool, scales in zip((s.keys, s.values), (s.key_pages, s.value_pages), s.scales):
        held, scale = _quantised(x, s.store)
        at = pages, heads, rows
        if used is not None:
            there = used.expand(x.shape[:3])
            at = tuple(i.expand(x.shape[:3])[there] for i in at)
            held, scale = held.view(torch.uint8)[there].view(held.dtype), scale[there]
        pool.view(torch.uint8)[at] = held.view(torch.uint8)
        scales[at] = scale


def _read(s):
    """(B, heads, tokens, width) keys and values, zeros past a request's rows."""
    pages, heads, rows, used = _places(s)
    found = []
    for pool, scales in zip((s.key_pages, s.value_pages), s.scales or (None, None)):
        x = _gathered(pool, scales, pages.clamp(min=0), heads, rows)
        found.append((x if used is None else x.masked_fill(~used[..., None], 0.0)).to(s.dtype))
    return tuple(found)


def _package():
    import __graft_entry__
    return __graft_entry__.import_package()


def run(state):
    s = state
    if s.kind in ('attend', 'shared'):
        if own:
            return _package().paged_attention(s.query, s.key_pages, s.value_pages, s.table, s.positions, mask=s.mask,
                                              scales=s.scales, shared_pages=s.shared)
        return _attend(s)
    if own:
        if s.kind == 'store':
            _package().paged_write(s.keys, s.values, s.key_pages, s.value_pages, s.table, s.starts, s.lengths, scales=s.scales)
        return _package().paged_read(s.key_pages, s.value_pages, s.table, s.starts, s.tokens, s.lengths, scales=s.scales,
                                     dtype=s.dtype)
    if s.kind == 'store':
        _write(s)
    return _read(s)


def work(case):
    size, width, heads = SIZES[case['dtype']], case['width'], case['kv_heads']
    held = 2 * (width * SIZES[case['store']] + (4 if case['store'] in STORES else 0)) if 'store' in case else 2 * width * size
    if case['kind'] in ('attend', 'shared'):
        prefix = case.get('prefix', 0)
        behind = int((_contexts(case) + 1).sum())
        keys = behind + prefix * case['batch']
        rows = 2 * case['batch'] * case['q_heads'] * width * size
        mask = 0 if case['mask'] == 'none' else keys * (1 if case['mask'] == 'bool' else size)
        pages = int((_contexts(case) // case['page'] + 1).sum()) + prefix // case['page']
        return {'bytes': (behind + prefix) * heads * held + rows + mask + 4 * pages + 8 * case['batch'],
                'flops': 4 * keys * case['q_heads'] * width}
    gen = torch.Generator().manual_seed(7)
    rows = int(torch.randint(case['low'], case['high'] + 1, (case['batch'],), generator=gen).sum()) * heads
    padded = case['batch'] * case['tokens'] * heads
    if case['kind'] == 'store':  # read, held, read back
        return {'bytes': rows * (2 * width * size + 2 * held) + padded * 2 * width * size, 'flops': 0}
    return {'bytes': rows * held + padded * 2 * width * size, 'flops': 0}


# ---- in 64 bits ----------------------------------------------------------------------------

def _power64(n):
    """2^n in float64, exactly."""
    return (n.long() + 1023 << 52).view(torch.float64)


def _values64(pool, scales, index):
    """Rows of a pool, by an index of its pages, heads and rows, as float64."""
    if scales is None:
        return pool[index].double()
    return pool.view(torch.uint8)[index].view(pool.dtype).double() * scales[index].double()[..., None]


def _exact_attend(s):
    batch, _, q_heads, width = s.query.shape
    kv_heads = s.key_pages.shape[1]
    group = q_heads // kv_heads
    key_scales, value_scales = s.scales if s.scales else (None, None)
    out = torch.zeros(batch, 1, q_heads, width, device=DEVICE, dtype=torch.float64)
    for b in range(batch):
        length = int(s.contexts[b]) + 1
        j = torch.arange(length, device=DEVICE)
        if s.mask is not None:
            term = s.mask[b, 0, 0, :length]
            j = j[term if term.dtype == torch.bool else term != -math.inf]
            if not j.numel():
                continue
        index = (s.table[b].long()[torch.div(j, s.page, rounding_mode='floor')][:, None],
                 torch.arange(kv_heads, device=DEVICE)[None], (j % s.page)[:, None])
        k = _values64(s.key_pages, key_scales, index).permute(1, 2, 0).contiguous()  # (heads, width, keys)
        v = _values64(s.value_pages, value_scales, index).transpose(0, 1).contiguous()
        scores = s.query[b, 0].double().reshape(kv_heads, group, width) @ k / math.sqrt(width)
        if s.mask is not None and s.mask.dtype != torch.bool:
            scores = scores + term[j].double()
        out[b, 0] = (torch.softmax(scores, -1) @ v).reshape(q_heads, width)
    return out


def _exact_store(s):
    """The rows after quantising, or those of the pages: (keys, values), zeros past a request's rows."""
    batch, heads, width = s.table.shape[0], s.key_pages.shape[1], s.key_pages.shape[3]
    found = []
    for n, pool in enumerate((s.key_pages, s.value_pages)):
        out = torch.zeros(batch, heads, s.tokens, width, dtype=torch.float64, device=DEVICE)
        for b in range(batch):
            count = s.tokens if s.lengths is None else int(s.lengths[b])
            if s.kind == 'read':
                at = int(s.starts[b]) + torch.arange(count, device=DEVICE)
                index = (s.table[b].long()[torch.div(at, s.page, rounding_mode='floor')][None],
                         torch.arange(heads, device=DEVICE)[:, None], (at % s.page)[None])
                out[b, :, :count] = _values64(pool, s.scales[n] if s.scales else None, index)
                continue
            x = (s.keys, s.values)[n][b, :, :count].double()
            a = x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
            if s.store == 'int8':
                out[b, :, :count] = torch.round(x * 127 / a) * (a / 127)
                continue
            _, above = torch.frexp(a / 448 * (1 - 2.0 ** -50))  # the smallest power of two at or over a / 448 (not the next for a power)
            step = _power64(above)
            y = x / step
            # e4m3: four significant bits, whole multiples of 2^-9 below 2^-6
            _, above = torch.frexp(y.abs().clamp(min=2.0 ** -6))
            unit = _power64(above - 4)
            out[b, :, :count] = torch.round(y / unit) * unit * step
        found.append(out)
    return tuple(found)


def exact(case, seed):
    s = prepare(case, seed)
    return (_exact_attend if case['kind'] in ('attend', 'shared') else _exact_store)(s)
