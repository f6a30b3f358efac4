"""``paged_attention`` of requests that share their first pages, against the definition in float64."""
import math

import pytest
import torch

from tests._paged import assert_within
from tests._paged_more import HELD, expected, problem, run

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _behind(prefix, own):
    """Lengths of requests of ``own`` keys behind ``prefix`` shared ones."""
    return [prefix + n for n in own]


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('width', [64, 128])
@pytest.mark.parametrize('heads', [(16, 8), (8, 8), (32, 4), (16, 1), (20, 1), (28, 4), (3, 3)], ids=str)
def test_types_widths_and_head_layouts(pkg, device, dtype, width, heads):
    p = problem(device, _behind(208, [1, 15, 16, 17, 40, 100, 333]), shared=13, q_heads=heads[0], kv_heads=heads[1], width=width,
                dtype=dtype, seed=1)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('page', [1, 5, 8, 16, 24, 32, 64, 100, 256])
@pytest.mark.parametrize('dtype,width,layout', [(BF16, 128, 'nhd'), (F32, 64, 'hnd'), (F16, 64, 'hnd')], ids=str)
def test_page_sizes_and_layouts(pkg, device, page, dtype, width, layout):
    shared = max(1, 300 // page)
    p = problem(device, _behind(shared * page, [1, 15, 16, 17, 40, 100, 333]), shared=shared, page=page, dtype=dtype, width=width,
                layout=layout, seed=2)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('shared', [1, 2, 3, 4, 7, 8, 9, 31, 64, 129, 600])
@pytest.mark.parametrize('batch', [1, 2, 5, 33])
def test_lengths_of_the_prefix(pkg, device, shared, batch):
    p = problem(device, _behind(16 * shared, [1 + 7 * b % 50 for b in range(batch)]), shared=shared, q_heads=8, kv_heads=4, seed=3)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('batch', [8, 16, 17, 40, 64, 100, 200])
@pytest.mark.parametrize('heads', [(16, 8), (8, 1), (3, 3)], ids=str)
@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
def test_many_requests(pkg, device, batch, heads, dtype):
    p = problem(device, _behind(640, [b % 90 for b in range(batch)]), shared=20, page=32, q_heads=heads[0], kv_heads=heads[1], dtype=dtype,
                seed=4)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('dtype,width', [(BF16, 128), (F16, 128), (F32, 64)], ids=str)
@pytest.mark.parametrize('own', [[1, 2000, 0, 300, 5], [1] * 24], ids=['ragged', 'one'])
def test_long_prefixes(pkg, device, dtype, width, own):
    p = problem(device, _behind(9000, own), shared=90, page=100, q_heads=8, kv_heads=2, width=width, dtype=dtype, seed=5)
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('batch', [9, 50])
def test_requests_that_end_within_the_shared_pages(pkg, device, dtype, batch):
    """And such that attend nothing, as padded requests of a captured batch."""
    lengths = ([0, 1, 15, 16, 17, 100, 159, 160, 161] * 6)[:batch]
    p = problem(device, lengths, shared=10, dtype=dtype, seed=6)
    out = run(pkg, p)
    assert (out[0] == 0).all()
    assert_within(out, *expected(p))
    p.positions.fill_(-1)
    assert (run(pkg, p) == 0).all()
    p.positions[3], p.positions[4] = 2 ** 62, -2 ** 62
    p.positions[5] = p.table.shape[1] * 16
    assert (run(pkg, p) == 0).all()


@pytest.mark.parametrize('width,dtype,heads', [(128, BF16, (16, 8)), (64, F32, (8, 8)), (128, F16, (24, 2))], ids=str)
@pytest.mark.parametrize('kind', [torch.bool, BF16, F16, F32], ids=str)
@pytest.mark.parametrize('batch', [7, 40])
def test_masks(pkg, device, width, dtype, heads, kind, batch):
    """Keys hidden from some requests and from all, requests that are left nothing, hidden rows that hold NaN."""
    lengths = ([330, 340, 600, 321, 400, 0, 100] * 6)[:batch]
    p = problem(device, lengths, shared=20, page=16, width=width, dtype=dtype, q_heads=heads[0], kv_heads=heads[1], seed=7)
    ctx = p.table.shape[1] * 16
    shown = torch.rand(batch, 1, 1, ctx, generator=torch.Generator().manual_seed(8)) < 0.7
    shown[3] = False
    shown[4, ..., :320] = False
    shown[1, ..., 320:] = False
    shown[..., 64:129] = False  # from all requests
    for pool in (p.key_pages, p.value_pages):
        pool[int(p.table[0, 5])] = math.nan
    mask = shown if kind == torch.bool else torch.where(shown, torch.rand(shown.shape), -math.inf).to(kind)
    mask = mask.to(device)
    out = run(pkg, p, mask=mask)
    assert (out[3] == 0).all() and (out[5] == 0).all()
    want = expected(p, mask=mask)
    assert_within(out, *want)
    strided = torch.full((batch, 1, 1, ctx, 3), 9, device=device).to(mask.dtype)[..., 1].copy_(mask)
    assert torch.equal(run(pkg, p, mask=strided), out)


@pytest.mark.parametrize('scale', [0.0, -0.2, 1e-4])
@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
@pytest.mark.parametrize('masked', [False, True])
def test_scales(pkg, device, scale, dtype, masked):
    p = problem(device, _behind(320, [b % 30 for b in range(40)]), shared=20, dtype=dtype, seed=25)
    mask = torch.ones(40, 1, 1, p.table.shape[1] * 16, dtype=torch.bool, device=device) if masked else None
    assert_within(run(pkg, p, scale=scale, mask=mask), *expected(p, scale=scale, mask=mask))


@pytest.mark.parametrize('scale', [1e-38, -1e-38, 1e-41])
@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
def test_scales_next_to_zero(pkg, device, scale, dtype):
    p = problem(device, _behind(320, [b % 30 for b in range(40)]), shared=20, dtype=dtype, seed=27)
    assert_within(run(pkg, p, scale=scale), *expected(p, scale=scale))


@pytest.mark.parametrize('dtype,width,heads', [(BF16, 128, (16, 8)), (F16, 64, (8, 8)), (F32, 128, (40, 2))], ids=str)
@pytest.mark.parametrize('batch', [3, 20, 70])
@pytest.mark.parametrize('odd', [math.nan, math.inf])
def test_values_that_are_not_finite_behind_the_ends_of_some(pkg, device, dtype, width, heads, batch, odd):
    """Requests that end within the shared pages before such a value, with it, and behind it."""
    lengths = ([700, 705, 64, 65, 66, 640, 0, 900] * 10)[:batch]
    p = problem(device, lengths, shared=40, dtype=dtype, width=width, q_heads=heads[0], kv_heads=heads[1], seed=26)
    clean, tol = expected(p)
    p.value_pages[int(p.table[0, 4]), 1, 0, 9] = odd  # key 64
    out = run(pkg, p).cpu()
    group = slice(heads[0] // heads[1], 2 * heads[0] // heads[1])
    for b, n in enumerate(lengths):
        if n > 64:
            at = out[b, 0, group, 9]
            assert (at.isnan() if math.isnan(odd) else at == odd).all()
            out[b, 0, group, 9], clean[b, 0, group, 9] = 0, 0
    assert_within(out, clean, tol)


@pytest.mark.parametrize('dtype,kind', [(BF16, BF16), (BF16, F32), (F16, BF16), (F16, F16), (F32, F32), (F32, F16)], ids=str)
@pytest.mark.parametrize('batch', [5, 40])
def test_masks_of_the_types_lowest_value(pkg, device, dtype, kind, batch):
    """Terms that hide nothing where all keys of a request have them, in the prefix, behind it or in both."""
    p = problem(device, ([330, 340, 600, 321, 400] * 8)[:batch], shared=20, dtype=dtype, seed=32)
    ctx = p.table.shape[1] * 16
    low = torch.rand(batch, 1, 1, ctx, generator=torch.Generator().manual_seed(33)) < 0.3
    low[0], low[1, ..., :320], low[2, ..., 320:] = True, True, True
    mask = torch.where(low, torch.finfo(kind).min, 0.0).to(kind).to(device)
    assert_within(run(pkg, p, mask=mask), *expected(p, mask=mask))


@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
def test_a_value_hidden_from_some_requests_alone(pkg, device, dtype):
    """A NaN or an infinity among the shared values shows where it is attended, and nowhere else."""
    p = problem(device, _behind(320, [5] * 20), shared=20, q_heads=4, kv_heads=2, dtype=dtype, seed=9)
    mask = torch.ones(20, 1, 1, p.table.shape[1] * 16, dtype=torch.bool, device=device)
    mask[::2, ..., 40] = False
    clean, tol = expected(p, mask=mask)
    page, row = int(p.table[0, 2]), 40 % 16
    p.value_pages[page, 1, row, 9], p.value_pages[page, 1, row, 10] = math.nan, math.inf
    out = run(pkg, p, mask=mask).cpu()
    assert out[1::2, 0, 2:, 9].isnan().all() and (out[1::2, 0, 2:, 10] == math.inf).all()
    out[1::2, 0, 2:, 9:11], clean[1::2, 0, 2:, 9:11] = 0, 0
    assert_within(out, clean, tol)


@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
def test_masks_of_few_keys_and_of_one_term(pkg, device, dtype):
    """A mask that ends within the shared pages, and one term for all keys."""
    p = problem(device, _behind(160, [16, 40, 16]), shared=10, dtype=dtype, seed=10)  # rows for every position below
    for keys in (2, 16, 100, 160, 161, 176):
        mask = torch.ones(3, 1, 1, keys, dtype=torch.bool, device=device)
        p.positions = torch.tensor([keys - 1, keys // 2, keys], device=device)
        out = run(pkg, p, mask=mask)
        assert (out[2] == 0).all()
        assert_within(out, *expected(p, mask=mask))
    p.positions = torch.tensor([164, 199, 160], device=device)
    one = torch.tensor([True, False, True], device=device)[:, None, None, None]
    out = run(pkg, p, mask=one)
    assert (out[1] == 0).all()
    assert_within(out, *expected(p, mask=one.expand(3, 1, 1, p.table.shape[1] * 16)))


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('below', [5.0, 40.0, 80.0])
def test_infinite_shared_values_under_small_weights_show(pkg, device, dtype, below):
    p = problem(device, _behind(320, [40] * 10), shared=20, q_heads=4, kv_heads=2, dtype=dtype, seed=11)
    p.query.zero_()
    p.query[..., 0] = 8.0
    p.key_pages.nan_to_num_(0.0).zero_()
    p.key_pages[p.table[0, :20].long(), :, 3, 0] = below * 128 ** 0.5 / 8.0
    clean, tol = expected(p)
    assert_within(run(pkg, p), clean, tol)
    p.value_pages[int(p.table[0, 0]), 0, 4, 17] = math.inf
    p.value_pages[int(p.table[0, 19]), 0, 0, 18] = -math.inf
    p.value_pages[int(p.table[0, 7]), 0, 0, 19] = math.nan
    out = run(pkg, p).cpu()
    assert (out[:, 0, :2, 17] == math.inf).all() and (out[:, 0, :2, 18] == -math.inf).all() and out[:, 0, :2, 19].isnan().all()
    out[:, 0, :2, 17:20], clean[:, 0, :2, 17:20] = 0, 0
    assert_within(out, clean, tol)


def test_shared_pages_outside_the_pool_do_not_exist(pkg, device):
    p = problem(device, _behind(320, [5, 40, 1, 17]), shared=20, seed=12)
    p.table[:, 3], p.table[:, 7], p.table[2, 20] = -1, 2 ** 31 - 1, -5
    assert_within(run(pkg, p), *expected(p))
    p.table[:, :20] = -1
    assert_within(run(pkg, p), *expected(p))


@pytest.mark.parametrize('dtype,width', [(BF16, 128), (F16, 64), (F32, 128)], ids=str)
@pytest.mark.parametrize('prefix,batch', [(64, 40), (2048, 5), (2048, 40)])
def test_by_the_librarys_choice_and_never(pkg, device, dtype, width, prefix, batch):
    """Short and long prefixes, on either side of where the library reads them once."""
    p = problem(device, _behind(prefix, [b % 50 for b in range(batch)]), shared=prefix // 16, dtype=dtype, width=width, seed=13)
    never = run(pkg, p, read_once=False)
    want = expected(p)
    assert_within(never, *want)
    assert torch.equal(never, pkg.paged_attention(p.query, p.key_pages, p.value_pages, p.table, p.positions))
    chosen = run(pkg, p, read_once=None)
    assert_within(chosen, *want)
    assert torch.equal(chosen, never) or torch.equal(chosen, run(pkg, p))


@pytest.mark.parametrize('held', HELD, ids=str)
@pytest.mark.parametrize('dtype,width', [(BF16, 128), (F16, 64), (F32, 128)], ids=str)
@pytest.mark.parametrize('batch', [3, 40])
def test_pools_of_8_bits(pkg, device, held, dtype, width, batch):
    p = problem(device, _behind(480, [b % 50 for b in range(batch)]), shared=20, page=24, held=held, dtype=dtype, width=width, seed=14)
    assert_within(run(pkg, p), *expected(p))


def test_out_strides_scales_and_the_query_itself(pkg, device):
    p = problem(device, _behind(320, [5, 40, 1, 17, 200]), shared=20, seed=15)
    want = run(pkg, p)
    out = torch.zeros(5, 1, 40, 130, device=device, dtype=BF16)[:, :, 3:35:2, 1:129]
    assert run(pkg, p, out=out) is out and torch.equal(out, want)
    assert_within(run(pkg, p, scale=0.3), *expected(p, scale=0.3))
    assert run(pkg, p, out=p.query) is p.query and torch.equal(p.query, want)


@pytest.mark.parametrize('batch', [6, 40])
def test_captured_and_replayed(pkg, device, batch):
    """Two graphs, replayed in turn as positions change, with eager calls between."""
    problems = [problem(device, _behind(640, [(b * k) % 90 + 1 for b in range(batch)]), shared=20, page=32, seed=16 + k) for k in (1, 2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for p in problems:
        run(pkg, p)
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            outs.append(run(pkg, p))
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(graph)
    for n in range(4):
        for p, graph, out in zip(problems, graphs, outs):
            p.positions -= n
            p.query.normal_()
            graph.replay()
            eager = run(pkg, p)
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
            assert_within(out, *expected(p))


def test_on_two_streams_at_once(pkg, device):
    problems = [problem(device, _behind(1600, [(b * k) % 90 + 1 for b in range(30)]), shared=50, page=32, seed=20 + k) for k in (1, 2)]
    want = [run(pkg, p) for p in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    outs = [[], []]
    for _ in range(10):
        for p, stream, out in zip(problems, streams, outs):
            with torch.cuda.stream(stream):
                out.append(run(pkg, p))
    torch.cuda.synchronize()
    for w, out in zip(want, outs):
        assert all(torch.equal(w, o) for o in out)


def test_shared_pages_past_four_gigabytes(pkg, device):
    pages = (1 << 32) // (8 * 16 * 128 * 2) + 16
    near = problem(device, _behind(128, [5, 20, 1]), shared=8, seed=30)
    pools = [torch.empty(pages, 8, 16, 128, dtype=BF16, device=device) for _ in range(2)]
    for pool, given in zip(pools, (near.key_pages, near.value_pages)):
        pool[-given.shape[0]:] = given
    table = torch.where(near.table < 0, near.table, near.table + pages - near.key_pages.shape[0])
    out = pkg.paged_attention(near.query, *pools, table, near.positions, shared_pages=8, read_once=True)
    assert torch.equal(out, run(pkg, near))
    assert_within(out, *expected(near))


@pytest.mark.parametrize('dtype,width,heads', [(BF16, 128, (16, 8)), (F16, 64, (20, 2)), (F32, 128, (4, 4))], ids=str)
@pytest.mark.parametrize('masked', [False, True])
def test_such_values_before_long_requests(pkg, device, dtype, width, heads, masked):
    """Launches for requests of thousands of own keys that have to take the prefix as well."""
    lengths = [5000, 3000, 2048, 100, 2600, 0, 2049, 4100] * 3
    p = problem(device, lengths, shared=64, page=32, dtype=dtype, width=width, q_heads=heads[0], kv_heads=heads[1], seed=31)
    mask = None
    if masked:
        mask = torch.ones(len(lengths), 1, 1, p.table.shape[1] * 32, dtype=torch.bool, device=device)
        mask[::5, ..., 90:140] = False
    clean, tol = expected(p, mask=mask)
    p.value_pages[int(p.table[0, 4]), 0, 1, 9] = math.nan  # key 129
    out = run(pkg, p, mask=mask).cpu()
    group = slice(0, heads[0] // heads[1])
    for b, n in enumerate(lengths):
        if n > 129 and not (masked and b % 5 == 0):
            assert out[b, 0, group, 9].isnan().all()
            out[b, 0, group, 9], clean[b, 0, group, 9] = 0, 0
    assert_within(out, clean, tol)
