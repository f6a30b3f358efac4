"""``paged_attention`` over shared pages where what the launch ahead of the requests' own keys does on its own shows: the bits
of its weights, how long it may be, and whose row of the table it goes by."""
import pytest
import torch

from tests._paged import assert_within, attention64
from tests._paged_more import HELD, expected, problem, run

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=str)
@pytest.mark.parametrize('width', [64, 128])
@pytest.mark.parametrize('batch', [5, 40])
@pytest.mark.parametrize('masked', [False, True])
def test_weights_keep_the_bits_that_outputs_show(pkg, device, dtype, width, batch, masked):
    """Every second key scores a little more than the others and has a value of 1, the others -1: what is left of the values is the
    difference of weights next to each other, which weights of the type's own bits get wrong by a sixth.

    The scores are sums of one product, so that ``attention64``'s bound is small.  To it comes what two parts leave of a weight:
    half a step each, 2^-16 of it in bf16, times A = sum_j w_j |v_j| = 1; in fp16 2^-22 (which the bound holds), and of weights
    that are 2^8 times as large half of the smallest number, 2^-25, for each of 320 keys."""
    p = problem(device, [321 + b % 7 for b in range(batch)], shared=20, dtype=dtype, width=width, seed=40)
    p.query.zero_()
    p.query[..., 0] = 0.01 + 0.004 * torch.arange(batch, device=device)[:, None, None] % 0.05
    sign = torch.tensor([1.0, -1.0], device=device).repeat(8)[None, None, :, None]
    p.key_pages.copy_(sign.expand(p.key_pages.shape))
    p.value_pages.copy_(sign.expand(p.value_pages.shape))
    mask = torch.ones(batch, 1, 1, p.table.shape[1] * 16, dtype=torch.bool, device=device) if masked else None
    want, tol = attention64(p.query, p.key_pages, p.value_pages, p.table, p.positions, mask=mask)
    tol += {BF16: 2.0 ** -16, F16: 320 * 2.0 ** -33, F32: 0.0}[dtype]
    assert_within(run(pkg, p, mask=mask), want, tol)


@pytest.mark.parametrize('odd', [False, True])
def test_prefixes_past_two_to_the_25_keys(pkg, device, odd):
    """One page over and over, and at the end one whose key outweighs all others; a value after the request's end that is not finite
    leaves all of them to the request's one workgroup."""
    page, entries = 512, 65600  # (own keys that a workgroup has to itself)
    pools = [torch.zeros(3, 1, page, 128, dtype=BF16, device=device) for _ in range(2)]
    pools[0][1, 0, 7, 0] = 42.5  # a score of 30 over those of 3.4e7 others
    pools[1][1, 0, 7] = torch.randn(128, device=device)
    pools[1][1, 0, -1] = float('inf') if odd else 3.0
    table = torch.zeros(2, entries + 1, dtype=torch.int32, device=device)
    table[:, entries - 1], table[:, entries] = 1, 2
    query = torch.zeros(2, 1, 1, 128, dtype=BF16, device=device)
    query[..., 0] = 8
    positions = torch.tensor([entries * page - 2, -1], device=device)
    out = pkg.paged_attention(query, *pools, table, positions, shared_pages=entries, read_once=True)
    want = pools[1][1, 0, 7].float()
    assert ((out[0, 0, 0].float() - want).abs() <= want.abs() * (2.0 ** -8 + 1e-5)).all() and (out[1] == 0).all()


@pytest.mark.parametrize('dtype,width,heads', [(BF16, 128, (16, 8)), (F16, 64, (20, 2)), (F32, 64, (3, 3))], ids=str)
@pytest.mark.parametrize('batch,retired', [(5, [0]), (5, [0, 1, 2, 3]), (40, [0, 1, 17, 39]), (40, range(40)), (700, range(650))],
                         ids=['0', 'all but one', 'some', 'all', 'past a workgroup'])
@pytest.mark.parametrize('masked', [False, True])
def test_rows_that_requests_have_left(pkg, device, dtype, width, heads, batch, retired, masked):
    """Rows of -1, the first one's too, as the page table of an arena has them: they attend nothing, and no other loses a key."""
    p = problem(device, [321 + 5 * b % 60 for b in range(batch)], shared=20, q_heads=heads[0], kv_heads=heads[1], dtype=dtype, width=width,
                seed=41)
    retired = list(retired)
    p.table[retired] = -1
    mask = torch.ones(batch, 1, 1, p.table.shape[1] * 16, dtype=torch.bool, device=device) if masked else None
    want = expected(p, mask=mask)
    for positions in (p.positions.clone(), p.positions.clone().index_fill(0, torch.tensor(retired, device=device), -1)):
        p.positions = positions
        out = run(pkg, p, mask=mask)
        assert (out[retired] == 0).all()
        assert_within(out, *want)


def test_a_captured_launch_of_which_requests_retire(pkg, device):
    """Through the table's contents alone, one after the other, a value that is not finite in between."""
    p = problem(device, [1300 + b % 70 for b in range(30)], shared=80, seed=42)
    run(pkg, p)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = run(pkg, p)
    torch.cuda.current_stream().wait_stream(side)
    for b in (0, 7, 1, 2):
        p.table[b] = -1
        p.query.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(pkg, p))
        assert_within(out, *expected(p))
    place = int(p.table[-1, 3]), 0, 5, 6
    kept = p.value_pages[place].item()
    p.value_pages[place] = float('inf')
    graph.replay()
    torch.cuda.synchronize()
    assert (out[:3] == 0).all() and (out[3:7, 0, :2, 6] == float('inf')).all()
    p.value_pages[place] = kept
    graph.replay()
    torch.cuda.synchronize()
    assert_within(out, *expected(p))


@pytest.mark.parametrize('held', HELD, ids=str)
@pytest.mark.parametrize('dtype,width', [(BF16, 128), (F16, 64), (F32, 128)], ids=str)
@pytest.mark.parametrize('batch', [3, 40])
def test_pools_of_8_bits_are_read_by_each_request(pkg, device, held, dtype, width, batch):
    """To the bound that they have without shared pages, and to the same bits."""
    p = problem(device, [481 + b % 50 for b in range(batch)], shared=20, page=24, held=held, dtype=dtype, width=width, seed=43)
    out = run(pkg, p)
    p.shared = 0
    assert torch.equal(out, run(pkg, p))
    assert_within(out, *expected(p))


@pytest.mark.parametrize('page,prefix,heads', [(1, 9000, (16, 1)), (1, 3000, (8, 4)), (2, 9000, (4, 1)), (3, 12000, (16, 1))], ids=str)
@pytest.mark.parametrize('dtype', [BF16, F32], ids=str)
@pytest.mark.parametrize('masked', [False, True])
def test_parts_that_end_with_the_pages_that_a_workgroup_knows(pkg, device, page, prefix, heads, dtype, masked):
    """Pages of few rows: 1022 of them hold fewer keys than a part would have otherwise, so that there are more parts."""
    p = problem(device, [prefix + 1 + b for b in range(3)], shared=prefix // page, page=page, q_heads=heads[0], kv_heads=heads[1], dtype=dtype,
                seed=44)
    mask = None
    if masked:
        mask = torch.rand(3, 1, 1, p.table.shape[1] * page, generator=torch.Generator().manual_seed(45)).to(device) < 0.8
    assert_within(run(pkg, p, mask=mask), *expected(p, mask=mask))


@pytest.mark.parametrize('dtype,width', [(BF16, 128), (F16, 64), (F32, 64)], ids=str)
@pytest.mark.parametrize('batch', [5, 40])
@pytest.mark.parametrize('odd', [float('nan'), float('inf')])
def test_queries_that_are_not_finite_stay_with_their_requests(pkg, device, dtype, width, batch, odd):
    p = problem(device, [650 + b % 30 for b in range(batch)], shared=40, dtype=dtype, width=width, seed=46)
    p.query[2, 0, 3, 5] = odd
    out = run(pkg, p).cpu()
    assert out[2, 0, 3].isnan().all()
    p.query[2, 0, 3] = 0
    want, tol = expected(p)
    out[2, 0, 3], want[2, 0, 3] = 0, 0
    assert_within(out, want, tol)
