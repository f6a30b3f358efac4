"""Steps of ``PackedAttention`` over a ``PagedCache`` that are refused, or take an unusual mask."""
import math

import pytest
import torch

from tests._paged import assert_within, expected, problem, run
from tests._talker import Talker

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _layer(pkg, device, table_width=4):
    model = Talker(layers=1, hidden=256, seed=3, dtype=BF16).to(device).eval()
    pkg.install_packed_attention(model, native_gqa=True, text_only_rope=True, triton_talker_rope=True)
    arena = pkg.PagedArena(model, pages=9, page_size=16)
    arena.packed.normal_()
    table = arena.page_table([arena.allocate(3), arena.allocate(3)], width=table_width)
    return model, arena, pkg.PagedCache(arena, table, torch.tensor([40, 20], device=device))


def _step(model, cache, hidden, mask):
    tables = model.rotary_emb(hidden, cache.positions.expand(3, -1)[..., None])
    with torch.inference_mode():
        return model.layers[0](hidden, attention_mask=mask, past_key_values=cache, position_embeddings=tables)[0]


@pytest.mark.parametrize('shape,dtype', [((2, 1, 1, 65), BF16), ((2, 1, 1, 64), torch.float64), ((2, 16, 1, 64), BF16),
                                         ((3, 1, 1, 64), BF16), ((2, 64), BF16), ((2, 1, 1, 1), BF16),
                                         ((2, 1, 1, 1), torch.bool), ((1, 1, 1, 1), torch.float32)], ids=str)
def test_a_refused_step_leaves_the_pages(pkg, device, shape, dtype):
    model, arena, cache = _layer(pkg, device)
    before = arena.packed.clone()
    with pytest.raises(ValueError):
        _step(model, cache, torch.randn(2, 1, 256, device=device, dtype=BF16), torch.zeros(shape, dtype=dtype, device=device))
    torch.cuda.synchronize(device)
    same = torch.equal(arena.packed, before)
    assert same


@pytest.mark.parametrize('dtype,width', [(BF16, 128), (torch.float16, 64), (torch.float32, 64)], ids=str)
@pytest.mark.parametrize('kind', [torch.bool, BF16, torch.float32], ids=str)
@pytest.mark.parametrize('table_width', [None, 300])
def test_a_mask_of_one_term_is_for_all_keys(pkg, device, dtype, width, kind, table_width):
    """SDPA's meaning of a last dimension of 1: a request is shown all of its keys, or none."""
    p = problem(device, [1, 40, 300, 17, 0], width=width, dtype=dtype, seed=40, table_width=table_width)
    ctx = p.table.shape[1] * p.page
    shown = torch.tensor([True, True, True, False, True], device=device)[:, None, None, None]
    mask = shown if kind == torch.bool else torch.where(shown, 1.5, -math.inf).to(kind)
    out = run(pkg, p, mask=mask)
    assert (out[3] == 0).all() and (out[4] == 0).all()
    assert_within(out, *expected(p, mask=mask.expand(5, 1, 1, ctx)))
    for one in (mask[:1], mask[0, 0, 0], mask[:1].expand(5, 1, 1, 1)):
        assert_within(run(pkg, p, mask=one), *expected(p, mask=one.expand(5, 1, 1, ctx)))


@pytest.mark.parametrize('dtype', [BF16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize('heads', [(16, 8), (20, 1)], ids=str)
@pytest.mark.parametrize('lengths', [[100, 3, 0, 333], [9000, 17, 4000]], ids=['short', 'cut'])
def test_the_output_may_be_the_query(pkg, device, dtype, heads, lengths):
    p = problem(device, lengths, q_heads=heads[0], kv_heads=heads[1], dtype=dtype, seed=41)
    want = run(pkg, p)
    assert run(pkg, p, out=p.query) is p.query
    assert torch.equal(p.query, want)


@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('below', [5.0, 23.0, 25.0, 40.0, 80.0])
@pytest.mark.parametrize('dtype', [BF16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize('lengths', [[100, 40], [5000, 2000]], ids=['short', 'cut'])
def test_infinite_values_under_small_weights_show(pkg, device, dtype, lengths, below, masked):
    """An attended infinity is an infinity of the output down to float32's smallest weights (e^-87), and NaN a
    NaN; other elements keep their values.  All scores are 0 but those of row 3 of every page, ``below`` higher:
    each stage of a wave has the maximum."""
    p = problem(device, lengths, q_heads=4, kv_heads=2, dtype=dtype, seed=42)
    p.query.zero_()
    p.query[..., 0] = 8.0
    for b, n in enumerate(lengths):
        at = p.table[b, :-(-n // 16)].long()
        p.key_pages[at] = 0
        p.key_pages[at, :, 3, 0] = below * 128 ** 0.5 / 8.0
    mask = torch.zeros(2, 1, 1, p.table.shape[1] * 16, device=device) if masked else None
    clean, tol = expected(p, mask=mask)
    assert_within(run(pkg, p, mask=mask), clean, tol)
    first, last = int(p.table[0, 0]), int(p.table[0, (lengths[0] - 1) // 16])
    p.value_pages[first, 0, 4, 17] = math.inf
    p.value_pages[last, 0, 0, 18] = -math.inf
    p.value_pages[first, 0, 5, 19] = math.inf
    p.value_pages[last, 0, 1, 19] = -math.inf
    p.value_pages[last, 0, 2, 20] = math.nan
    out = run(pkg, p, mask=mask).cpu()
    for h in (0, 1):
        assert out[0, 0, h, 17] == math.inf and out[0, 0, h, 18] == -math.inf and out[0, 0, h, 19:21].isnan().all()
        out[0, 0, h, 17:21], clean[0, 0, h, 17:21] = 0, 0
    assert_within(out, clean, tol)


@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('dtype,width', [(BF16, 128), (torch.float16, 128), (torch.float16, 64), (torch.float32, 64)], ids=str)
@pytest.mark.parametrize('lengths', [[100, 40], [5000, 2000]], ids=['short', 'cut'])
def test_an_attended_key_that_is_nan_shows(pkg, device, dtype, width, lengths, masked):
    """Its score is NaN, and with it all of its head's outputs; other heads and requests keep their values."""
    p = problem(device, lengths, q_heads=4, kv_heads=2, width=width, dtype=dtype, seed=43)
    mask = torch.zeros(2, 1, 1, p.table.shape[1] * 16, device=device) if masked else None
    clean, tol = expected(p, mask=mask)
    p.key_pages[int(p.table[0, (lengths[0] - 1) // 16]), 1, 2, 9] = math.nan
    out = run(pkg, p, mask=mask).cpu()
    assert out[0, 0, 2:].isnan().all()
    out[0, 0, 2:], clean[0, 0, 2:] = 0, 0
    assert_within(out, clean, tol)
