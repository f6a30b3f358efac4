"""The paged cache in 8 bits: ``paged_write``, ``paged_read`` and ``paged_attention`` with ``scales``."""
import math

import pytest
import torch

from tests._paged import assert_within
from tests._paged_more import HELD, bits, expected, problem, quantised, run, stands_for

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
RAGGED = [1, 15, 16, 17, 31, 32, 33, 64, 65, 0, 127, 128, 129, 300]


# ---- written and read ----------------------------------------------------------------------

def _pools(device, pages, heads, page, width, held, seed=0):
    gen = torch.Generator().manual_seed(seed)
    pools = [torch.randint(0, 120, (pages, heads, page, width), generator=gen, dtype=torch.uint8).view(held).to(device) for _ in range(2)]
    return pools, tuple(torch.rand(pages, heads, page, generator=gen).to(device) for _ in range(2))


def _rows(device, batch, heads, tokens, width, dtype, seed=1):
    """Views of fused projection rows, of all sizes."""
    gen = torch.Generator().manual_seed(seed)
    fused = torch.randn(batch, tokens, 2 * heads + 1, width, generator=gen) * torch.logspace(-3, 3, 2 * heads + 1)[:, None]
    fused = fused.to(dtype).to(device)
    return fused[:, :, 1:heads + 1].transpose(1, 2), fused[:, :, heads + 1:].transpose(1, 2)


def _table(device, batch, width, pages, seed=2):
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:batch * width]
    return order.view(batch, width).to(torch.int32).to(device)


def _places(table, positions, tokens, lengths, page, pages):
    """(b, t, page, row) of every row that a call has."""
    for b in range(table.shape[0]):
        used = tokens if lengths is None else max(0, min(int(lengths[b]), tokens))
        for t in range(used):
            j = int(positions[b]) + t
            if 0 <= j < table.shape[1] * page and 0 <= int(table[b, j // page]) < pages:
                yield b, t, int(table[b, j // page]), j % page


def _check(pkg, rows, pools, scales, table, positions, lengths=None):
    """A write bit for bit, everything else as it was, and the rows read back."""
    held, (batch, heads, tokens, width), (pages, _, page, _) = pools[0].dtype, rows[0].shape, pools[0].shape
    places = list(_places(table.cpu(), positions.cpu(), tokens, lengths, page, pages))
    want = []
    for x, pool, scale in zip(rows, pools, scales):
        elements, own = quantised(x, held)
        pool, scale = bits(pool).clone(), scale.cpu().clone()
        for b, t, at, r in places:
            pool[at, :, r], scale[at, :, r] = bits(elements)[b, :, t], own[b, :, t]
        want.append((pool, scale))
    pkg.paged_write(*rows, *pools, table, positions, lengths, scales=scales)
    for pool, scale, (w_pool, w_scale) in zip(pools, scales, want):
        assert torch.equal(bits(pool), w_pool)
        assert torch.equal(bits(scale), bits(w_scale))
    for dtype in (BF16, F16, F32):
        back = pkg.paged_read(*pools, table, positions, tokens, lengths, scales=scales, dtype=dtype)
        for x, (pool, scale), got in zip(rows, want, back):
            expected_rows = torch.zeros(batch, heads, tokens, width, dtype=dtype)
            values = (pool.view(held).float() * scale[..., None]).to(dtype)
            for b, t, at, r in places:
                expected_rows[b, :, t] = values[at, :, r]
            assert got.dtype == dtype and torch.equal(bits(got), bits(expected_rows))


@pytest.mark.parametrize('held', HELD, ids=str)
@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('width', [64, 128])
@pytest.mark.parametrize('tokens', [1, 2, 37])
def test_rows_are_written_and_read(pkg, device, held, dtype, width, tokens):
    pools, scales = _pools(device, 40, 3, 16, width, held)
    table = _table(device, 5, 6, 40)
    positions = torch.tensor([0, 7, 16, 50, 95], device=device)
    lengths = None if tokens == 2 else torch.tensor([tokens, 1, 0, tokens + 5, -3], dtype=torch.int32, device=device)
    _check(pkg, _rows(device, 5, 3, tokens, width, dtype), pools, scales, table, positions, lengths)


@pytest.mark.parametrize('page', [1, 5, 24, 100])
@pytest.mark.parametrize('held', HELD, ids=str)
def test_page_sizes_and_pages_outside_the_pool(pkg, device, page, held):
    pools, scales = _pools(device, 30, 2, page, 128, held)
    table = _table(device, 3, 10, 30)
    table[0, 1], table[1, 0], table[2, 9] = -1, 30, 2 ** 31 - 1
    positions = torch.tensor([-5, 3 * page - 1, 2 ** 62], device=device)
    _check(pkg, _rows(device, 3, 2, 9, 128, BF16), pools, scales, table, positions)


@pytest.mark.parametrize('held', HELD, ids=str)
@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
def test_values_at_the_ends_of_their_range(pkg, device, held, dtype):
    """Zeros, subnormals, the largest values, powers of two, ties, infinities and NaN."""
    top, low = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    rows = torch.zeros(12, 128)
    rows[1, 5], rows[2], rows[3, ::2] = -0.0, low / 4, top
    rows[4], rows[4, 0] = torch.arange(-64, 64) / 2.0, 127.0  # halves: ties of int8
    rows[5], rows[5, 0] = torch.arange(128) * 1.0, 448.0      # ties of e4m3
    rows[6, 3], rows[7, 4], rows[8, 1:3] = math.inf, -math.inf, torch.tensor([math.nan, 3.0])
    rows[9], rows[9, 7] = 1e-3, 1.75
    rows[10], rows[10, 7] = 1e-3, math.nextafter(1.75, 2) if dtype == F32 else 1.7578125
    rows[11] = torch.logspace(-12, 4, 128)
    x = rows.to(dtype).view(1, 1, 12, 128).to(device)
    pools, scales = _pools(device, 3, 1, 16, 128, held)
    table = torch.tensor([[2]], dtype=torch.int32, device=device)
    start = torch.zeros(1, dtype=torch.int64, device=device)
    pkg.paged_write(x, -x, *pools, table, start, scales=scales)
    for given, pool, scale in zip((x, -x), pools, scales):
        elements, own = quantised(given, held)
        finite = torch.isfinite(own[0, 0])
        assert finite.tolist() == [i not in (6, 7, 8) for i in range(12)]
        assert torch.equal(bits(scale)[2, 0, :12][finite], bits(own)[0, 0][finite])
        assert scale[2, 0, :12].cpu()[~finite].isnan().all()
        assert torch.equal(bits(pool)[2, 0, :12], bits(elements)[0, 0])
    back = pkg.paged_read(*pools, table, start, 12, scales=scales, dtype=F32)
    # (row 3 may stand for infinity: 255 * 2^120 is held as 256 * 2^120 in e4m3, and a / 127 may be rounded up)
    for given, got in zip((x, -x), back):
        elements, own = quantised(given, held)
        assert torch.equal(got[0, 0].cpu().nan_to_num(7.0), (elements.float() * own[..., None])[0, 0].nan_to_num(7.0))
        assert got[0, 0, 6:9].isnan().all()
        assert torch.isfinite(got[0, 0, [0, 1, 2, 4, 5, 9, 10, 11]]).all()


@pytest.mark.parametrize('held', HELD, ids=str)
def test_an_element_is_off_by_half_a_step_at_most(pkg, device, held):
    """int8: half of a / 127; e4m3: 2^-4 of its own size, or 2^-10 of the scale."""
    x = torch.randn(3, 4, 50, 128, generator=torch.Generator().manual_seed(5)).to(device)
    pools, scales = _pools(device, 60, 4, 8, 128, held)
    table, start = _table(device, 3, 10, 60), torch.zeros(3, dtype=torch.int64, device=device)
    pkg.paged_write(x, x, *pools, table, start, scales=scales)
    a = x.abs().amax(-1, keepdim=True)
    half = a / 254 if held == torch.int8 else torch.maximum(x.abs() * 2.0 ** -4, a / 224 * 2.0 ** -10)
    for back in pkg.paged_read(*pools, table, start, 50, scales=scales, dtype=F32):
        assert ((back - x).abs() <= half * (1 + 1e-5)).all()


@pytest.mark.parametrize('held', [*HELD, BF16], ids=str)
@pytest.mark.parametrize('tokens', [1, 33, 700])  # (two rows a thread in the last)
def test_either_order_of_tokens_and_heads(pkg, device, held, tokens):
    """Rows of a prefill cache, head by head, and of a projection, token by token."""
    batch, heads, width, page, wide = 26, 7, 64, 24, 31
    rows = _rows(device, batch, heads, tokens, width, BF16)
    pools, scales = _pools(device, batch * wide + 3, heads, page, width, torch.int8 if held == BF16 else held)
    table = _table(device, batch, wide, batch * wide + 3)
    positions = torch.arange(batch, device=device) * 2
    lengths = (torch.arange(batch, device=device) * 29 % (tokens + 1)).to(torch.int32)
    if held == BF16:
        pools, scales = [x.to(BF16) for x in pools], None
    else:
        _check(pkg, [x.contiguous() for x in rows], pools, scales, table, positions, lengths)
        by_head = [bits(x).clone() for x in (*pools, *scales)]
        pkg.paged_write(*rows, *pools, table, positions, lengths, scales=scales)
        assert all(torch.equal(bits(x), y) for x, y in zip((*pools, *scales), by_head))
    want = pkg.paged_read(*pools, table, positions, tokens, lengths, scales=scales, dtype=BF16)
    out = tuple(torch.full((batch, tokens, heads, width), 7.0, device=device, dtype=BF16).transpose(1, 2) for _ in range(2))
    for x, y in zip(pkg.paged_read(*pools, table, positions, tokens, lengths, scales=scales, out=out), want):
        assert torch.equal(bits(x), bits(y))


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
def test_a_negative_zero_is_held_and_read(pkg, device, dtype):
    pools, scales = _pools(device, 2, 1, 16, 64, torch.float8_e4m3fn)
    x = torch.zeros(1, 1, 4, 64, device=device, dtype=dtype)
    x[..., 1::2], x[..., 2, 0] = -0.0, -5.0
    table, start = torch.ones(1, 1, dtype=torch.int32, device=device), torch.zeros(1, dtype=torch.int64, device=device)
    pkg.paged_write(x, x, *pools, table, start, scales=scales)
    for back in pkg.paged_read(*pools, table, start, 4, scales=scales, dtype=dtype):
        assert torch.equal(bits(back), bits(x))


@pytest.mark.parametrize('held', HELD, ids=str)
def test_rows_off_16_bytes_and_pools_by_strides(pkg, device, held):
    big = torch.randn(2, 9, 3, 131, device=device).to(BF16)
    rows = big[..., 1:129].transpose(1, 2), big[..., 3:131].transpose(1, 2)
    pools, scales = _pools(device, 20, 16, 3, 128, held)  # (pages, page, heads, width) in memory
    pools = [x.transpose(1, 2) for x in pools]
    scales = tuple(torch.rand(20, 2, 16, 3, device=device)[:, 1].transpose(1, 2) for _ in range(2))
    table, positions = _table(device, 2, 3, 20), torch.tensor([5, 30], device=device)
    _check(pkg, rows, pools, scales, table, positions)
    out = tuple(torch.full((2, 3, 9, 130), 7.0, device=device, dtype=BF16)[..., 1:129] for _ in range(2))
    got = pkg.paged_read(*pools, table, positions, 9, scales=scales, out=out)
    fresh = pkg.paged_read(*pools, table, positions, 9, scales=scales)
    for x, y, o in zip(got, fresh, out):
        assert x is o and torch.equal(bits(x), bits(y))
        assert (x.as_strided((2, 3, 9, 1), x.stride(), x.storage_offset() + 128) == 7).all()


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('width', [1, 5, 12, 64, 128, 200])
@pytest.mark.parametrize('page', [7, 16])
def test_rows_of_their_own_type_are_read_bit_for_bit(pkg, device, dtype, width, page):
    gen = torch.Generator().manual_seed(3)
    pools = [torch.randn(20, 3, page, width, generator=gen).to(dtype).to(device) for _ in range(2)]
    table = _table(device, 4, 5, 20)
    table[1, 1] = -1
    positions = torch.tensor([0, 3, 2 * page - 1, 4 * page], device=device)
    lengths = torch.tensor([30, 12, 0, 100], dtype=torch.int32, device=device)
    got = pkg.paged_read(*pools, table, positions, 30, lengths)
    for pool, rows in zip(pools, got):
        want = torch.zeros(4, 3, 30, width, dtype=dtype)
        for b, t, at, r in _places(table.cpu(), positions.cpu(), 30, lengths, page, 20):
            want[b, :, t] = pool[at, :, r].cpu()
        assert torch.equal(bits(rows), bits(want))


# ---- attended ------------------------------------------------------------------------------

@pytest.mark.parametrize('held', HELD, ids=str)
@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('width', [64, 128])
@pytest.mark.parametrize('heads', [(16, 8), (8, 8), (16, 1), (20, 1), (28, 4), (3, 3)], ids=str)
def test_types_widths_and_head_layouts(pkg, device, held, dtype, width, heads):
    p = problem(device, RAGGED, held=held, q_heads=heads[0], kv_heads=heads[1], width=width, dtype=dtype, seed=1)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('page', [1, 5, 8, 16, 24, 32, 64, 100, 256])
@pytest.mark.parametrize('held,width,layout', [(HELD[0], 128, 'nhd'), (HELD[1], 64, 'hnd'), (HELD[1], 128, 'hnd')], ids=str)
def test_page_sizes_and_layouts(pkg, device, page, held, width, layout):
    p = problem(device, RAGGED, held=held, width=width, page=page, layout=layout, seed=2)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('length', [1, 2, 31, 32, 33, 63, 65, 257, 1000, 4097, 20011])
@pytest.mark.parametrize('held,dtype,width', [(HELD[0], BF16, 128), (HELD[1], F16, 64), (HELD[1], F32, 128)], ids=str)
def test_one_request_of_any_length(pkg, device, length, held, dtype, width):
    p = problem(device, [length], held=held, width=width, dtype=dtype, q_heads=8, kv_heads=2, seed=3)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('held', HELD, ids=str)
@pytest.mark.parametrize('lengths', [[1] * 700, [70] * 300, [5] + [1500] * 3 + [0] * 5 + [64] * 200, [9000, 3, 1, 9000],
                                     [900] * 90, [4000] * 70 + [1, 0, 17]], ids=['700x1', '300x70', 'mixed', 'two long', '90x900', '70 long'])
def test_many_requests_share_the_card(pkg, device, held, lengths):
    p = problem(device, lengths, held=held, q_heads=8, kv_heads=4, page=32, seed=4)
    assert_within(run(pkg, p), *expected(p))


MASKS = [torch.bool, BF16, F16, F32]


@pytest.mark.parametrize('held,width', [(HELD[0], 128), (HELD[1], 128), (HELD[0], 64), (HELD[1], 64)], ids=str)
@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
@pytest.mark.parametrize('kind', MASKS, ids=str)
@pytest.mark.parametrize('page', [16, 24, 64])
def test_masks(pkg, device, held, width, dtype, kind, page):
    """Hidden keys in every place, requests that are left nothing, and hidden rows that hold NaN."""
    lengths = [1, 40, 300, 17, 129, 0, 900]
    p = problem(device, lengths, held=held, width=width, dtype=dtype, page=page, seed=5)
    ctx = p.table.shape[1] * page
    shown = torch.rand(len(lengths), 1, 1, ctx, generator=torch.Generator().manual_seed(6)) < 0.7
    shown[3] = False
    shown[4, ..., 64:128] = False
    for b, n in enumerate(lengths):
        if n > 40 and b != 3:
            j = 37
            shown[b, ..., j] = False
            at = int(p.table[b, j // page])
            p.scales[0][at, :, j % page] = math.nan
            p.scales[1][at, :, j % page] = math.inf
            p.value_pages.view(torch.uint8)[at, :, j % page] = 0xff
    mask = shown if kind == torch.bool else torch.where(shown, torch.rand(shown.shape), -math.inf).to(kind)
    mask = mask.to(device)
    out = run(pkg, p, mask=mask)
    assert (out[3] == 0).all() and (out[5] == 0).all()
    assert_within(out, *expected(p, mask=mask))


@pytest.mark.parametrize('held', HELD, ids=str)
@pytest.mark.parametrize('dtype,kind', [(BF16, BF16), (F16, F16), (F32, F32)], ids=str)
@pytest.mark.parametrize('lengths', [[100, 40, 300], [5000, 2000, 33]], ids=['short', 'cut'])
def test_masks_of_the_types_lowest_value(pkg, device, held, dtype, kind, lengths):
    """Terms that hide nothing where all keys of a request have them."""
    p = problem(device, lengths, held=held, dtype=dtype, seed=12)
    low = torch.rand(3, 1, 1, p.table.shape[1] * 16, generator=torch.Generator().manual_seed(13)) < 0.3
    low[1] = True
    mask = torch.where(low, torch.finfo(kind).min, 0.0).to(kind).to(device)
    assert_within(run(pkg, p, mask=mask), *expected(p, mask=mask))


@pytest.mark.parametrize('held', HELD, ids=str)
@pytest.mark.parametrize('lengths', [[100, 40], [5000, 2000]], ids=['short', 'cut'])
def test_rows_that_stand_for_nan_show(pkg, device, held, lengths):
    """An attended row of values whose scale is NaN makes its head's outputs NaN, and so does one of keys; others keep theirs."""
    p = problem(device, lengths, held=held, q_heads=4, kv_heads=2, seed=7)
    clean, tol = expected(p)
    p.scales[1][int(p.table[0, 1]), 0, 3] = math.nan
    p.scales[0][int(p.table[1, 1]), 1, 3] = math.nan
    out = run(pkg, p).cpu()
    assert out[0, 0, :2].isnan().all() and out[1, 0, 2:].isnan().all()
    out[0, 0, :2], clean[0, 0, :2], out[1, 0, 2:], clean[1, 0, 2:] = 0, 0, 0, 0
    assert_within(out, clean, tol)


@pytest.mark.parametrize('held', HELD, ids=str)
def test_positions_outside_the_table_and_pages_outside_the_pool(pkg, device, held):
    p = problem(device, [40, 41, 42, 43, 44, 40], held=held, seed=8)
    p.positions = torch.tensor([-1, 48, -2 ** 62, 2 ** 62, 43, 39], device=device)
    p.table[4, 1], p.table[5] = 2 ** 31 - 1, -1
    out = run(pkg, p)
    assert (out[:4] == 0).all() and (out[5] == 0).all()
    assert_within(out, *expected(p))


@pytest.mark.parametrize('held', HELD, ids=str)
def test_scales_of_any_size(pkg, device, held):
    """Rows of every magnitude that float32 products allow."""
    p = problem(device, [200, 77], held=held, dtype=F32, q_heads=4, kv_heads=2, seed=9)
    p.scales[0].mul_(2.0 ** -40)
    p.query *= 2.0 ** 40
    p.scales[1].mul_(torch.logspace(-20, 20, p.scales[1].numel(), device=device).view_as(p.scales[1]))
    assert_within(run(pkg, p), *expected(p))


def test_out_strides_and_the_query_itself(pkg, device):
    p = problem(device, [100, 3, 0, 333], held=HELD[0], seed=10)
    want = run(pkg, p)
    room = torch.zeros(4, 1, 40, 130, device=device, dtype=BF16)
    out = room[:, :, 3:35:2, 1:129]
    assert run(pkg, p, out=out) is out and torch.equal(out, want)
    assert run(pkg, p, out=p.query) is p.query and torch.equal(p.query, want)


@pytest.mark.parametrize('held', HELD, ids=str)
def test_write_attend_and_read_in_a_graph(pkg, device, held):
    """A step captured once and replayed as positions, rows and tables change, with eager work in between."""
    p = problem(device, [100, 40, 260], held=held, table_width=20, seed=11)
    rows = [torch.randn(3, 8, 1, 128, device=device).to(BF16) for _ in range(2)]

    def step():
        pkg.paged_write(*rows, p.key_pages, p.value_pages, p.table, p.positions, scales=p.scales)
        out = run(pkg, p)
        return out, *pkg.paged_read(p.key_pages, p.value_pages, p.table, p.positions, 1, scales=p.scales)
    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        with torch.cuda.graph(graph, stream=side):
            held_out = step()
    torch.cuda.current_stream().wait_stream(side)
    for n in range(4):
        for x in rows:
            x.normal_()
        p.positions -= n
        graph.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in held_out]
        eager = step()
        assert all(torch.equal(x, y) for x, y in zip(replayed, eager))
        assert_within(replayed[0], *expected(p))
