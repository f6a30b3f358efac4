"""``paged_write`` bit for bit, and the arena and cache of pages through ``PackedAttention``."""
import math

import pytest
import torch

from tests._paged import assert_within, attention64
from tests._talker import Talker
from tests._util import assert_attention_close, f64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _reference(keys, values, key_pages, value_pages, table, positions, lengths=None):
    """The write, row by row on the host."""
    pools = [key_pages.cpu().clone(), value_pages.cpu().clone()]
    pages, _, page, _ = pools[0].shape
    for b in range(keys.shape[0]):
        used = keys.shape[2] if lengths is None else max(0, min(int(lengths[b]), keys.shape[2]))
        for t in range(used):
            j = int(positions[b]) + t
            if not 0 <= j < table.shape[1] * page:
                continue
            at = int(table[b, j // page])
            if 0 <= at < pages:
                for pool, rows in zip(pools, (keys, values)):
                    pool[at, :, j % page] = rows[b, :, t].cpu()
    return pools


def _bits(t):
    return t.cpu().contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def _check(pkg, rows, pools, table, positions, lengths=None):
    want = _reference(*rows, *pools, table, positions, lengths)
    pkg.paged_write(*rows, *pools, table, positions, lengths)
    for pool, expected in zip(pools, want):
        assert torch.equal(_bits(pool), _bits(expected))


def _pools(device, pages, heads, page, width, dtype, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return [torch.randn(pages, heads, page, width, generator=gen, device=device).to(dtype) for _ in range(2)]


def _rows(device, batch, heads, tokens, width, dtype, seed=1):
    """Views of fused projection rows."""
    gen = torch.Generator(device=device).manual_seed(seed)
    fused = torch.randn(batch, tokens, 2 * heads + 1, width, generator=gen, device=device).to(dtype)
    return fused[:, :, 1:heads + 1].transpose(1, 2), fused[:, :, heads + 1:].transpose(1, 2)


def _table(device, batch, width, pages, seed=2):
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:batch * width]
    return order.view(batch, width).to(torch.int32).to(device)


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('width', [1, 6, 20, 64, 128, 130])
@pytest.mark.parametrize('page', [1, 7, 16])
def test_one_token(pkg, device, dtype, width, page):
    pools = _pools(device, 40, 3, page, width, dtype)
    table = _table(device, 6, 6, 40)
    positions = torch.tensor([0, page - 1, page, 6 * page - 1, 2 * page, 1], device=device)
    _check(pkg, _rows(device, 6, 3, 1, width, dtype), pools, table, positions)


@pytest.mark.parametrize('page', [1, 16, 24])
@pytest.mark.parametrize('tokens', [2, 17, 70])
def test_padded_batch(pkg, device, page, tokens):
    batch, width = 7, -(-(tokens + 40) // page)
    pools = _pools(device, batch * width + 5, 8, page, 128, BF16)
    table = _table(device, batch, width, batch * width + 5)
    starts = torch.tensor([0, 1, 39, 16, 5, 0, 40], device=device)
    lengths = torch.tensor([tokens, 0, 1, tokens - 1, tokens + 9, -3, tokens // 2], device=device, dtype=torch.int32)
    _check(pkg, _rows(device, batch, 8, tokens, 128, BF16), pools, table, starts, lengths)
    _check(pkg, _rows(device, batch, 8, tokens, 128, BF16, seed=3), pools, table, starts)


def test_rows_outside_are_skipped(pkg, device):
    """Positions outside the table's rows and pages outside the pool write nothing, whatever the
    request's other rows do."""
    pools = _pools(device, 30, 2, 4, 64, BF16)
    table = _table(device, 8, 3, 30)
    table[5, 1], table[6, 0], table[7, 2] = -1, 30, 2 ** 31 - 1
    positions = torch.tensor([-3, 10, 2 ** 63 - 1, -2 ** 63, 12, 2, 0, 6], device=device)
    _check(pkg, _rows(device, 8, 2, 6, 64, BF16), pools, table, positions)


def test_layouts(pkg, device):
    """Pools with the heads inside the pages' rows, pools within one tensor, rows of a prefill
    cache, rows and pools that only narrow units fit."""
    dtype, table, positions = BF16, _table(device, 3, 4, 16), torch.tensor([0, 5, 30], device=device)
    nhd = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in _pools(device, 16, 4, 8, 64, dtype)]
    _check(pkg, _rows(device, 3, 4, 2, 64, dtype), nhd, table, positions)
    both = torch.randn(16, 2, 4, 8, 64, device=device).to(dtype)
    _check(pkg, _rows(device, 3, 4, 2, 64, dtype), [both[:, 0], both[:, 1]], table, positions)
    bnsd = [torch.randn(3, 4, 2, 64, device=device).to(dtype) for _ in range(2)]
    _check(pkg, bnsd, _pools(device, 16, 4, 8, 64, dtype), table, positions)
    flat = torch.randn(2 * 3 * 4 * 2 * 64 + 1, device=device).to(dtype)[1:].view(2, 3, 4, 2, 64)
    _check(pkg, list(flat), _pools(device, 16, 4, 8, 64, dtype), table, positions)


@pytest.mark.parametrize('tokens', [1, 3])
def test_more_requests_than_a_grid_is_wide(pkg, device, tokens):
    batch = 70001
    keys, values = _rows(device, batch, 1, tokens, 4, BF16)
    pools = _pools(device, batch + 5, 1, 4, 4, BF16)
    table = torch.randperm(batch + 5, generator=torch.Generator().manual_seed(9))[:batch].to(torch.int32)[:, None].to(device)
    positions = torch.arange(batch, device=device) % 3
    want = [pool.clone() for pool in pools]
    for t in range(tokens):
        fits = positions + t < 4
        for pool, rows in zip(want, (keys, values)):
            pool[table[fits, 0].long(), 0, positions[fits] + t] = rows[fits, 0, t]
    pkg.paged_write(keys, values, *pools, table, positions)
    for pool, expected in zip(pools, want):
        assert torch.equal(_bits(pool), _bits(expected))


def test_special_values_are_copied_as_they_are(pkg, device):
    rows = torch.tensor([0x7fc1, 0xff81, 0x0001, 0x8000] * 16, dtype=torch.int32).to(torch.int16).view(BF16)
    rows = rows.view(1, 1, 1, 64).to(device)
    pools = _pools(device, 2, 1, 4, 64, BF16)
    _check(pkg, (rows, rows.flip(3).contiguous()), pools, _table(device, 1, 2, 2), torch.tensor([5], device=device))


def test_pool_past_four_gigabytes(pkg, device):
    pages = (1 << 32) // (8 * 16 * 128 * 2) + 16
    pool = torch.empty(2, pages, 8, 16, 128, dtype=BF16, device=device)
    pool[:, -3:] = 0
    rows = _rows(device, 1, 8, 20, 128, BF16)
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device=device)
    pkg.paged_write(*rows, pool[0], pool[1], table, torch.tensor([1], device=device))
    for plane, given in zip(pool, rows):
        got = torch.cat([plane[-1], plane[-3]], 1)[:, 1:21]
        assert torch.equal(_bits(got), _bits(given[0]))
        assert (plane[-2] == 0).all() and (plane[-3, :, 5:] == 0).all()


def test_empty_calls(pkg, device):
    pools = _pools(device, 4, 2, 4, 64, BF16)
    before = [p.clone() for p in pools]
    for batch, tokens in ((0, 1), (2, 0)):
        pkg.paged_write(*_rows(device, batch, 2, tokens, 64, BF16), *pools, _table(device, 2, 2, 4)[:batch],
                        torch.zeros(batch, dtype=torch.int64, device=device))
    assert all(torch.equal(p, b) for p, b in zip(pools, before))


def _model(pkg, device, dtype=BF16, layers=2):
    model = Talker(layers=layers, hidden=256, seed=3, dtype=dtype).to(device).eval()
    pkg.install_packed_attention(model, native_gqa=True, text_only_rope=True, triton_talker_rope=True)
    return model


def _step(model, cache, hidden, positions, mask=None):
    tables = model.rotary_emb(hidden, positions.expand(3, -1)[..., None])
    for layer in model.layers:
        hidden = layer(hidden, attention_mask=mask, past_key_values=cache, position_embeddings=tables)[0]
    return model.norm(hidden)


@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
def test_a_paged_step_follows_the_slot_arena(pkg, device, dtype):
    """Requests admitted from a prefill cache and stepped on pages and on slots: every step's new rows
    bit for bit, and the outputs within the attention bar of each other (both within half of it of
    the exact values), while pages are added as the requests grow, one request leaves and another
    takes its pages."""
    model = _model(pkg, device, dtype)
    lengths, capacity, page = [30, 47, 1, 16], 96, 16
    gen = torch.Generator(device=device).manual_seed(4)
    prompt = torch.randn(4, 4, 8, 47, 128, generator=gen, device=device).to(dtype)
    prefill = type('Cache', (), {'layers': [type('Layer', (), {'keys': prompt[i], 'values': prompt[2 + i]})() for i in range(2)]})()
    slots = pkg.SlotArena(model, 4, capacity, packed_kv=True)
    arena = pkg.PagedArena(model, pages=24, page_size=page)
    arena.packed.fill_(math.nan)
    owned = [arena.allocate(arena.pages_for(n)) for n in lengths]
    table = arena.page_table(owned, width=capacity // page)
    arena.load(table, prefill, torch.tensor(lengths, dtype=torch.int32, device=device))
    for b, n in enumerate(lengths):
        slots.packed[:, b, :, :n] = prompt[:, b, :, :n]
    positions = torch.tensor(lengths, device=device)
    paged, slot = pkg.PagedCache(arena, table, positions), pkg.SlotCache(slots, positions)
    with torch.inference_mode():
        for step in range(20):
            for b in range(4):
                if int(positions[b]) == len(owned[b]) * page:  # the next row needs a page
                    owned[b] += arena.allocate(1)
            table.copy_(arena.page_table(owned, width=capacity // page))
            if step == 9:  # request 1 leaves, a shorter one takes its place and its pages
                arena.release(owned[1])
                owned[1] = arena.allocate(1)
                table.copy_(arena.page_table(owned, width=capacity // page))
                positions[1] = 0
            hidden = torch.randn(4, 1, 256, generator=gen, device=device).to(dtype)
            out, want = _step(model, paged, hidden, positions), _step(model, slot, hidden, positions)
            assert_attention_close(f64(out), f64(want), max_abs=2 * 3e-2, mean_abs=2 * 3e-3)
            # layer 0 sees the same rows on both sides: its new ones are equal
            for b in range(4):
                at = int(positions[b])
                row = arena.packed[:, owned[b][at // page], :, at % page]
                for plane in (0, 2):
                    assert torch.equal(row[plane], slots.packed[plane, b, :, at])
            positions += 1


def test_a_paged_step_applies_its_mask(pkg, device):
    model = _model(pkg, device, layers=1)
    arena = pkg.PagedArena(model, pages=9, page_size=16)
    arena.packed.normal_()
    table = arena.page_table([arena.allocate(3) for _ in range(3)])
    positions = torch.tensor([40, 20, 47], device=device)
    cache = pkg.PagedCache(arena, table, positions)
    mask = torch.zeros(3, 1, 1, 48, dtype=BF16, device=device)
    mask[0, ..., :9] = torch.finfo(BF16).min
    mask[2, ..., 3] = -math.inf
    seen = []
    attention = model.layers[0].self_attn
    attention.reference.o_proj.register_forward_hook(lambda m, args, out: seen.append(args[0]))
    queries = []
    attention.reference.q_norm.register_forward_hook(lambda m, args, out: queries.append(out))
    hidden = torch.randn(3, 1, 256, device=device, dtype=BF16)
    with torch.inference_mode():
        _step(model, cache, hidden, positions, mask)
        cos, sin = model.rotary_emb(hidden, positions[None, :, None])
        query = pkg.rotary(queries[0].contiguous(), cos[0].contiguous(), sin[0].contiguous())
    want, tol = attention64(query, arena.keys[0], arena.values[0], table, positions, mask=mask)
    assert_within(seen[0].view(3, 1, 16, 128), want, tol)


def test_paged_cache_refuses_what_it_cannot_do(pkg, device):
    model = _model(pkg, device, layers=1)
    arena = pkg.PagedArena(model, pages=4, page_size=16)
    table = arena.page_table([arena.allocate(2), arena.allocate(2)])
    before = arena.packed.clone()
    cache = pkg.PagedCache(arena, table, torch.tensor([3, 5], device=device))
    hidden = torch.randn(2, 3, 256, device=device, dtype=BF16)
    tables = model.rotary_emb(hidden, torch.arange(3, device=device).expand(3, 2, 3))
    with torch.inference_mode(), pytest.raises(ValueError):
        model.layers[0](hidden, past_key_values=cache, position_embeddings=tables)
    model.train()
    tables = tuple(t[:, :, :1] for t in tables)
    with torch.inference_mode(), pytest.raises(ValueError):
        model.layers[0](hidden[:, :1], past_key_values=cache, position_embeddings=tables)
    assert torch.equal(arena.packed, before)


def test_captured_step_follows_positions_and_table(pkg, device):
    """A paged step captured once and replayed over growing requests, against the eager step on a
    twin arena."""
    model = _model(pkg, device)
    arenas = [pkg.PagedArena(model, pages=12, page_size=16) for _ in range(2)]
    arenas[0].packed.normal_()
    arenas[1].packed.copy_(arenas[0].packed)
    owned = [arenas[0].allocate(2) for _ in range(3)]
    table = arenas[0].page_table(owned, width=4)
    positions = torch.full((3,), -1, device=device)
    caches = [pkg.PagedCache(arena, table, positions) for arena in arenas]
    hidden = torch.zeros(3, 1, 256, device=device, dtype=BF16)
    with torch.inference_mode():
        _step(model, caches[0], hidden, positions)  # no position: nothing is written
        torch.cuda.synchronize(device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(model, caches[0], hidden, positions)
        torch.cuda.synchronize(device)
        assert torch.equal(arenas[0].packed, arenas[1].packed)
        positions.copy_(torch.tensor([20, 3, 29]))
        for step in range(8):
            if step == 3:
                owned[2] += arenas[0].allocate(1)
                table.copy_(arenas[0].page_table(owned, width=4))
            hidden.normal_()
            graph.replay()
            want = _step(model, caches[1], hidden, positions)
            torch.cuda.synchronize(device)
            assert torch.equal(out, want)
            assert torch.equal(arenas[0].packed, arenas[1].packed)
            positions += 1
