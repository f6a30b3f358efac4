"""``paged_attention`` against the definition in float64, at the sizes, layouts, masks and page
tables where it can go wrong.  Tolerances are worked out in tests/_paged.py."""
import math

import pytest
import torch

from tests._paged import assert_within, attention64, expected, problem, run

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
RAGGED = [1, 15, 16, 17, 33, 64, 65, 0, 127, 128, 129, 300]


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('width', [64, 128])
@pytest.mark.parametrize('heads', [(16, 8), (8, 8), (32, 4), (16, 1), (20, 1), (40, 2), (28, 4), (3, 3), (9, 3)], ids=str)
def test_types_widths_and_head_layouts(pkg, device, dtype, width, heads):
    p = problem(device, RAGGED, q_heads=heads[0], kv_heads=heads[1], width=width, dtype=dtype, seed=1)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('page', [1, 2, 5, 8, 24, 32, 64, 100, 128, 256, 1000])
@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
def test_page_sizes(pkg, device, page, dtype):
    p = problem(device, RAGGED, page=page, dtype=dtype, seed=2)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('length', [1, 2, 31, 32, 63, 64, 65, 255, 256, 257, 511, 513, 1000, 4097, 20011])
@pytest.mark.parametrize('dtype,width', [(BF16, 128), (F16, 64), (F32, 128)], ids=str)
def test_one_request_of_any_length(pkg, device, length, dtype, width):
    p = problem(device, [length], width=width, dtype=dtype, q_heads=8, kv_heads=2, seed=3)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('lengths', [[1] * 700, [70] * 300, [5] + [1500] * 3 + [0] * 5 + [64] * 200, [9000, 3, 1, 9000],
                                     list(range(0, 520)), [i % 37 for i in range(9001)]], ids=['700x1', '300x70', 'mixed', 'two long', 'ramp', '9001'])
def test_many_requests_share_the_card(pkg, device, lengths):
    p = problem(device, lengths, q_heads=4, kv_heads=2, seed=4)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('dtype,width', [(BF16, 128), (BF16, 64), (F16, 128), (F16, 64), (F32, 128), (F32, 64)], ids=str)
@pytest.mark.parametrize('heads', [(16, 8), (8, 1), (20, 1)], ids=str)
def test_table_wider_than_the_requests_need(pkg, device, masked, dtype, width, heads):
    """Tables of 32000 rows a request, for which the launch takes larger workgroups; entries past a
    request's pages are not looked at (they hold -7 here)."""
    p = problem(device, RAGGED + [2100, 900], q_heads=heads[0], kv_heads=heads[1], width=width, dtype=dtype, table_width=1000,
                page=32, seed=5)
    mask = None
    if masked:
        mask = torch.ones(len(p.lengths), 1, 1, 32000, dtype=torch.bool, device=device)
        mask[:, :, :, 3::7] = False
        mask[5] = False
    assert_within(run(pkg, p, mask=mask), *expected(p, mask=mask))


@pytest.mark.parametrize('lengths', [[4000] * 70 + [1, 0, 17], [900] * 90, [30000, 31000, 5, 64]], ids=['70 long', '90x900', 'two'])
def test_launches_that_fill_the_card(pkg, device, lengths):
    p = problem(device, lengths, q_heads=16, kv_heads=8, page=64, seed=27)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('dtype,width', [(BF16, 128), (F16, 128), (BF16, 64), (F32, 64)], ids=str)
@pytest.mark.parametrize('heads', [(16, 1), (22, 2), (48, 1)], ids=str)
def test_large_groups_over_long_requests(pkg, device, masked, dtype, width, heads):
    """Many parts of states of up to 16 rows, merged in two steps."""
    lengths = [9000, 3, 0, 20001, 190, 700]
    p = problem(device, lengths, q_heads=heads[0], kv_heads=heads[1], width=width, dtype=dtype, page=32, seed=30)
    mask = None
    if masked:
        mask = torch.ones(len(lengths), 1, 1, 20001, dtype=torch.bool, device=device)
        mask[:, :, :, 5::11] = False
        mask[3, :, :, 4000:8000] = False
    assert_within(run(pkg, p, mask=mask), *expected(p, mask=mask))


@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('dtype,width', [(BF16, 128), (F32, 64), (BF16, 64)], ids=str)
@pytest.mark.parametrize('page', [16, 24, 64])
@pytest.mark.parametrize('lengths,rows', [([n % 749 for n in range(1, 40 * 173, 173)], 768), ([n % 1009 for n in range(3, 20 * 277, 277)], 960),
                                          ([690, 3, 0, 64, 65, 512, 513], 696)], ids=['40', '20', 'few'])
def test_a_workgroup_for_each_pair(pkg, device, lengths, rows, page, dtype, width, masked):
    """Launches at the capacities up to which no pair is cut."""
    lengths = [min(n, rows // page * page) for n in lengths]
    p = problem(device, lengths, q_heads=16, kv_heads=8, width=width, dtype=dtype, page=page, table_width=rows // page, seed=32)
    mask = None
    if masked:
        mask = torch.zeros(len(lengths), 1, 1, rows // page * page, device=device)
        mask[:, :, :, 3::9] = -math.inf
        mask[4] = -math.inf
    assert_within(run(pkg, p, mask=mask), *expected(p, mask=mask))


@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('dtype', [BF16, F16], ids=str)
@pytest.mark.parametrize('page', [16, 32, 48])
@pytest.mark.parametrize('lengths', [[0, 1, 16, 17, 31, 33, 47, 49, 200, 255, 500], [n % 960 for n in range(1, 17 * 271, 271)]], ids=['few', 'more'])
def test_narrow_rows_in_pages_of_half_a_stage(pkg, device, lengths, page, dtype, masked):
    p = problem(device, lengths, q_heads=16, kv_heads=8, width=64, dtype=dtype, page=page, seed=31)
    ctx = p.table.shape[1] * page
    mask = None
    if masked:
        mask = torch.ones(len(p.lengths), 1, 1, ctx, dtype=torch.bool, device=device)
        mask[:, :, :, 1::6] = False
        mask[8] = False
    assert_within(run(pkg, p, mask=mask), *expected(p, mask=mask))


@pytest.mark.parametrize('lengths', [[800] * 16, [n % 801 for n in range(0, 24 * 331, 331)]], ids=['equal', 'ragged'])
def test_pairs_for_more_than_half_of_the_card(pkg, device, lengths):
    p = problem(device, lengths, q_heads=16, kv_heads=8, table_width=50, page=16, seed=29)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('dtype,width', [(BF16, 128), (BF16, 64), (F16, 128), (F16, 64), (F32, 64)], ids=str)
@pytest.mark.parametrize('heads', [(16, 8), (20, 1)], ids=str)
def test_short_requests_of_a_workgroup_each(pkg, device, masked, dtype, width, heads):
    """Tables of 448 rows, of which a workgroup attends any number for itself."""
    p = problem(device, [0, 1, 15, 16, 17, 127, 128, 129, 130, 255, 257, 300, 385, 447, 448], q_heads=heads[0], kv_heads=heads[1],
                width=width, dtype=dtype, table_width=14, page=32, seed=28)
    mask = None
    if masked:
        mask = torch.ones(len(p.lengths), 1, 1, 448, dtype=torch.bool, device=device)
        mask[:, :, :, 2::5] = False
        mask[4] = False
    assert_within(run(pkg, p, mask=mask), *expected(p, mask=mask))


@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
def test_positions_outside_the_table_attend_nothing(pkg, device, dtype):
    p = problem(device, [40, 41, 42, 43, 44], dtype=dtype, seed=6)
    p.positions = torch.tensor([-1, 48, -2 ** 62, 2 ** 62, 43], device=device)  # the table holds 48 rows
    out = run(pkg, p)
    assert (out[:4] == 0).all()
    assert_within(out, *expected(p))


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('width', [64, 128])
def test_keys_on_no_page_do_not_exist(pkg, device, dtype, width):
    """Page numbers below zero and past the pool, within the requests' keys."""
    p = problem(device, [200, 100, 33, 16, 700], dtype=dtype, width=width, seed=7)
    pages = p.key_pages.shape[0]
    p.table[0, 3], p.table[0, 12], p.table[1, 0], p.table[2, 2], p.table[3, 0] = -1, pages, 2 ** 31 - 1, -2 ** 31, pages + 5
    p.table[4, 5:40:3] = -5
    out = run(pkg, p)
    assert (out[3] == 0).all()
    assert_within(out, *expected(p))


def _masks(kind, batch, ctx, device, seed=8):
    gen = torch.Generator().manual_seed(seed)
    hidden = torch.rand(batch, ctx, generator=gen) < 0.4
    if kind == 'bool':
        return ~hidden[:, None, None].to(device)
    dtype = {'bf16': BF16, 'fp16': F16, 'fp32': F32, 'lowest': BF16, 'lowest fp32': F32, 'bias': F32}[kind]
    if kind == 'bias':
        mask = torch.randn(batch, ctx, generator=gen) * 3
    else:
        low = torch.finfo(dtype).min if kind.startswith('lowest') else -math.inf
        mask = torch.zeros(batch, ctx).masked_fill(hidden, low)
    return mask.to(dtype)[:, None, None].to(device)


@pytest.mark.parametrize('kind', ['bool', 'bf16', 'fp16', 'fp32', 'lowest', 'lowest fp32', 'bias'])
@pytest.mark.parametrize('dtype,width', [(BF16, 128), (F16, 128), (BF16, 64), (F32, 128), (F32, 64)], ids=str)
def test_masks(pkg, device, kind, dtype, width):
    p = problem(device, RAGGED + [1500], width=width, dtype=dtype, seed=9)
    ctx = p.table.shape[1] * p.page
    mask = _masks(kind, len(p.lengths), ctx, device)
    assert_within(run(pkg, p, mask=mask), *expected(p, mask=mask))


@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
def test_rows_that_a_mask_leaves_nothing(pkg, device, dtype):
    p = problem(device, [1, 50, 200, 777], dtype=dtype, seed=10)
    ctx = p.table.shape[1] * p.page
    mask = torch.ones(4, 1, 1, ctx, dtype=torch.bool, device=device)
    mask[0] = mask[2] = False
    mask[3, ..., 5:] = False
    out = run(pkg, p, mask=mask)
    assert (out[0] == 0).all() and (out[2] == 0).all()
    assert_within(out, *expected(p, mask=mask))
    infinite = torch.zeros(mask.shape, device=device).masked_fill(~mask, -math.inf)
    assert torch.equal(run(pkg, p, mask=infinite), out)


@pytest.mark.parametrize('mask_type', [BF16, F32], ids=str)
def test_rows_of_the_lowest_value_are_averaged(pkg, device, mask_type):
    """finfo.min swallows the scores: all of a row's keys weigh the same, as SDPA has it."""
    p = problem(device, [1, 50, 333], dtype=BF16, seed=11)
    mask = torch.full((3, 1, 1, p.table.shape[1] * p.page), torch.finfo(mask_type).min, dtype=mask_type, device=device)
    assert_within(run(pkg, p, mask=mask), *expected(p, mask=mask))


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('width', [64, 128])
@pytest.mark.parametrize('what', [math.nan, math.inf, -math.inf])
def test_nothing_of_a_hidden_key_reaches_the_output(pkg, device, dtype, width, what):
    p = problem(device, [40, 130, 700], dtype=dtype, width=width, seed=12)
    ctx = p.table.shape[1] * p.page
    mask = _masks('bool', 3, ctx, device, seed=13)
    for b, n in enumerate(p.lengths):
        for j in range(n):
            if not bool(mask[b, 0, 0, j]):
                page = int(p.table[b, j // p.page])
                p.key_pages[page, :, j % p.page] = what
                p.value_pages[page, :, j % p.page] = what
    assert_within(run(pkg, p, mask=mask), *expected(p, mask=mask))


def test_values_that_are_not_finite_show(pkg, device):
    """An infinity that a request attends is an infinity of its output, a NaN a NaN, and other
    requests and other elements keep their values."""
    p = problem(device, [100, 100], dtype=BF16, seed=14)
    clean, tol = expected(p)
    p.value_pages[int(p.table[0, 2]), 3, 4, 17] = math.inf
    p.value_pages[int(p.table[0, 2]), 3, 4, 18] = math.nan
    out = run(pkg, p).cpu()
    for h in (6, 7):
        assert out[0, 0, h, 17] == math.inf and out[0, 0, h, 18].isnan()
        out[0, 0, h, 17:19], clean[0, 0, h, 17:19] = 0, 0
    assert_within(out, clean, tol)


def test_masks_of_other_shapes_and_strides(pkg, device):
    p = problem(device, [40, 64, 7], dtype=BF16, seed=15)
    ctx = p.table.shape[1] * p.page
    row = _masks('bias', 1, ctx, device)
    want = run(pkg, p, mask=row.expand(3, 1, 1, ctx).contiguous())
    for mask in (row, row[0], row[0, 0], row[0, 0, 0], row.expand(3, 1, 1, ctx)):
        assert torch.equal(run(pkg, p, mask=mask), want)
    for kind in ('bool', 'bf16', 'fp32'):
        mask = _masks(kind, 3, ctx, device)
        want = run(pkg, p, mask=mask)
        wide = torch.stack([mask, mask], -1)[..., 1]                     # every second element
        odd = torch.cat([mask[..., :1], mask], -1).contiguous()[..., 1:]  # rows that start at odd elements
        assert torch.equal(run(pkg, p, mask=wide), want) and torch.equal(run(pkg, p, mask=odd), want)
    # fewer keys than the table: positions past them attend nothing
    short = _masks('bool', 3, 41, device)
    out = run(pkg, p, mask=short)
    assert (out[1] == 0).all()
    assert_within(out, *expected(p, mask=short))
    for bad in (row.expand(3, 1, 2, ctx), row.expand(3, 2, 1, ctx), row[..., :0], row.expand(2, 1, 1, ctx),
                torch.zeros(3, 1, 1, ctx + 1, device=device), row.double(), row.cpu()):
        with pytest.raises(ValueError):
            run(pkg, p, mask=bad)


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
def test_layouts_and_strides(pkg, device, dtype):
    p = problem(device, RAGGED, dtype=dtype, seed=16)
    want = run(pkg, p)
    n = problem(device, RAGGED, dtype=dtype, seed=16, layout='nhd')
    assert not n.key_pages.is_contiguous()
    assert torch.equal(run(pkg, n), want)
    batch, _, heads, width = p.query.shape
    # pools as planes of one tensor, every second page of it
    both = torch.full((p.key_pages.shape[0] * 2, 2, 8, p.page, width), math.nan, dtype=dtype, device=device)
    both[::2, 0], both[::2, 1] = p.key_pages, p.value_pages
    assert torch.equal(pkg.paged_attention(p.query, both[::2, 0], both[::2, 1], p.table, p.positions), want)
    # the query as a view of fused projection rows, and one that 16-byte loads do not fit
    rows = torch.cat([p.query, p.query.new_zeros(batch, 1, 2, width)], 2)
    assert torch.equal(pkg.paged_attention(rows[:, :, :heads], p.key_pages, p.value_pages, p.table, p.positions), want)
    flat = torch.empty(p.query.numel() + 1, dtype=dtype, device=device)
    odd = flat[1:].view(p.query.shape).copy_(p.query)
    assert torch.equal(pkg.paged_attention(odd, p.key_pages, p.value_pages, p.table, p.positions), want)
    # table rows within a wider tensor; outputs within wider and oddly placed rows
    table = torch.full((batch, p.table.shape[1] + 3), 1 << 20, dtype=torch.int32, device=device)
    table[:, :-3] = p.table
    p.table = table[:, :-3]
    for offset, step in ((0, 2 * heads), (1, heads)):
        room = torch.full((batch * step * width + offset,), 7.0, dtype=dtype, device=device)
        out = room[offset:].view(batch, 1, step, width)[:, :, :heads]
        assert run(pkg, p, out=out).data_ptr() == out.data_ptr()
        assert torch.equal(out, want)
        assert (room[:offset] == 7).all() and (room[offset:].view(batch, 1, step, width)[:, :, heads:] == 7).all()
    for bad in (want[:, :, :, :64], want.double(), want[:3], want.cpu()):
        with pytest.raises(ValueError):
            run(pkg, p, out=bad)


def test_refuses_what_it_cannot_read(pkg, device):
    p = problem(device, [20, 30], width=128, seed=17)
    flat = torch.zeros(p.key_pages.numel() + 1, dtype=BF16, device=device)
    for pool in (flat[1:].view(p.key_pages.shape),
                 torch.zeros(5, 8, 16, 132, dtype=BF16, device=device)[..., :128][:p.key_pages.shape[0]]):
        odd = pool if pool.shape == p.key_pages.shape else pool.expand_as(pool)
        with pytest.raises(ValueError):
            pkg.paged_attention(p.query, odd, odd, p.table, p.positions)
    with pytest.raises(ValueError):
        run(pkg, p, out=torch.zeros(2, 1, 1, 128, dtype=BF16, device=device).expand(p.query.shape))
    wide = problem(device, [20], q_heads=8, kv_heads=8, width=96, seed=17)
    with pytest.raises(ValueError):
        run(pkg, wide)


def test_scale_and_shared_pages(pkg, device):
    """Two requests over the same pages (a shared prefix), and a scale of the caller's."""
    p = problem(device, [64, 90], dtype=BF16, seed=18)
    p.table[1, :4] = p.table[0, :4]
    for scale in (0.02, 1.0):
        assert_within(run(pkg, p, scale=scale), *expected(p, scale=scale))


def test_empty_batch(pkg, device):
    p = problem(device, [4], seed=19)
    out = pkg.paged_attention(p.query[:0], p.key_pages, p.value_pages, p.table[:0], p.positions[:0])
    assert out.shape == (0, 1, 16, 128)


@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
def test_scores_far_from_zero(pkg, device, dtype):
    """Large scores, whose maximum comes late, early or with every key."""
    for order in (1, -1, 0):
        p = problem(device, [500, 1203], dtype=dtype, seed=20, query_scale=0.1, q_heads=4, kv_heads=2)
        p.query[..., 0] = 8.0
        for b, n in enumerate(p.lengths):
            for j in range(n):
                p.key_pages[int(p.table[b, j // p.page]), :, j % p.page, 0] = 60.0 * (order * j / n if order else j % 2)
        assert_within(run(pkg, p), *expected(p))


def test_the_same_call_gives_the_same_bits(pkg, device):
    p = problem(device, [3000, 17, 900, 0, 64], seed=21)
    want = run(pkg, p)
    for _ in range(5):
        assert torch.equal(run(pkg, p), want)


def test_pool_past_four_gigabytes(pkg, device):
    """Pages whose byte offsets do not fit 32 bits, read from both ends of the pool."""
    p = problem(device, [100, 333], seed=22)
    pages = (1 << 32) // (8 * 16 * 128 * 2) + 64
    pool = torch.empty(2, pages, 8, 16, 128, dtype=BF16, device=device)
    far = pages - p.key_pages.shape[0]
    pool[0, far:], pool[1, far:] = p.key_pages, p.value_pages
    want = run(pkg, p)
    table = torch.where(p.table >= 0, p.table + far, p.table)
    assert torch.equal(pkg.paged_attention(p.query, pool[0], pool[1], table, p.positions), want)


def test_streams_and_workspaces_of_other_calls(pkg, device):
    """Calls on two streams at once, and between split launches of the slot arena's attention,
    which share the stream's workspace."""
    a, b = problem(device, [2000, 100, 3], seed=23), problem(device, [70] * 40 + [5000], seed=24, dtype=F16)
    want_a, want_b = run(pkg, a), run(pkg, b)
    assert_within(want_a, *expected(a))
    assert_within(want_b, *expected(b))
    query = torch.randn(8, 1, 16, 128, device=device, dtype=BF16)
    keys, values = torch.randn(2, 8, 8, 2048, 128, device=device, dtype=BF16).unbind(0)
    at = torch.full((8,), 2000, device=device)
    want_c = pkg.decode_attention(query, keys, values, at, splits=24)
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(device))
    for _ in range(6):
        for s, p, want in ((streams[0], a, want_a), (streams[1], b, want_b)):
            with torch.cuda.stream(s):
                outs.append((run(pkg, p), want))
                outs.append((pkg.decode_attention(query, keys, values, at, splits=24), want_c))
    torch.cuda.synchronize(device)
    for out, want in outs:
        assert torch.equal(out, want)


def test_captured_calls_follow_their_inputs(pkg, device):
    """Two graphs replayed in turn, the queries, positions, page tables and pools rewritten between
    replays, with eager calls in between: every replay equals the eager call of that moment."""
    lengths = [1200, 30, 64, 500]
    a, b = problem(device, lengths, seed=25), problem(device, [3000], seed=26, dtype=F32)
    graphs = []
    for p in (a, b):
        out = torch.empty_like(run(pkg, p))
        graph = torch.cuda.CUDAGraph()
        with torch.inference_mode(), torch.cuda.graph(graph):
            run(pkg, p, out=out)
        graphs.append((graph, out))
    for step in range(5):
        for p, (graph, out) in zip((a, b), graphs):
            p.positions.copy_(torch.tensor([max(0, n - 1 - 97 * step) for n in p.lengths]))
            p.query.mul_(0.9)
            if step == 2:
                p.table[0, :2] = p.table[0, :2].flip(0)
                p.value_pages.mul_(1.25)
            want = run(pkg, p)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize(device)
            assert torch.equal(out, want)
            assert_within(out, *expected(p))
