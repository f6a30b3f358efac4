"""What the paged cache's wrappers check and pass on, without a GPU: the device check is taken as
passed, and launches are recorded instead of made."""
import importlib
import random
from contextlib import contextmanager
from types import SimpleNamespace

import pytest
import torch

BF16 = torch.bfloat16


@pytest.fixture
def launches(pkg, monkeypatch):
    """The calls that would have been launched: ('write',) or ('attend', argument structure)."""
    lib, seen = pkg._lib, []
    paged = importlib.import_module(pkg.__name__ + '.paged')
    real = lib.packed

    @contextmanager
    def on_device(index):
        yield 0

    def packed(name):
        if name != 'q3t_paged_attention':
            return real(name)
        return lambda args, stream: seen.append(('attend', lib.PagedArgs.from_buffer_copy(args))) or 0

    monkeypatch.setattr(lib, 'gpu_index', lambda *tensors: 0)
    monkeypatch.setattr(lib, 'on_device', on_device)
    monkeypatch.setattr(lib, 'packed', packed)
    monkeypatch.setattr(lib, 'launch', lambda name, *rest: seen.append(('write',)))
    monkeypatch.setattr(paged, 'workspace', lambda device, size, stream: torch.empty(size, dtype=torch.uint8))
    return seen


def _tensors(batch=2, q_heads=16, kv_heads=8, width=128, page=16, pages=9, table=4, dtype=BF16):
    return dict(query=torch.zeros(batch, 1, q_heads, width, dtype=dtype),
                key_pages=torch.zeros(pages, kv_heads, page, width, dtype=dtype),
                value_pages=torch.zeros(pages, kv_heads, page, width, dtype=dtype),
                page_table=torch.zeros(batch, table, dtype=torch.int32), positions=torch.zeros(batch, dtype=torch.int64))


def _cache(pkg, batch=2, width=128, table=4):
    module = torch.nn.Linear(2, 2).bfloat16()
    reference = SimpleNamespace(parameters=module.parameters, layers=[None],
                                config=SimpleNamespace(num_key_value_heads=8, head_dim=width))
    arena = pkg.PagedArena(reference, pages=9, page_size=16)
    return pkg.PagedCache(arena, torch.zeros(batch, table, dtype=torch.int32), torch.zeros(batch, dtype=torch.int64))


def _step(cache, batch=2, width=128, **kwargs):
    rows = torch.zeros(batch, 8, 1, width, dtype=BF16)
    return cache.step(torch.zeros(batch, 1, 16, width, dtype=BF16), rows, rows, 0, **kwargs)


def test_a_step_writes_and_then_attends(pkg, launches):
    out = _step(_cache(pkg), scale=0.25)
    assert out.shape == (2, 1, 16, 128)
    assert [call[0] for call in launches] == ['write', 'attend']
    assert launches[1][1].scale == 0.25 and launches[1][1].ctx == 64


@pytest.mark.parametrize('mask', [
    torch.zeros(2, 1, 1, 65, dtype=BF16), torch.zeros(2, 1, 1, 64, dtype=torch.float64), torch.zeros(2, 1, 1, 64, dtype=torch.int64),
    torch.zeros(2, 16, 1, 64, dtype=BF16), torch.zeros(3, 1, 1, 64, dtype=BF16), torch.zeros(2, 64, dtype=BF16), (0.0,) * 64,
    torch.zeros(2, 1, 1, 0, dtype=BF16),
], ids=['long', 'float64', 'int64', 'heads', 'batch', 'rows', 'tuple', 'none'])
def test_a_refused_step_writes_nothing(pkg, launches, mask):
    with pytest.raises(ValueError):
        _step(_cache(pkg), mask=mask)
    assert launches == []


def test_a_step_under_a_mask_of_far_rows_writes_nothing(pkg, launches):
    """Rows of a mask 2^32 elements apart (memory that is never touched)."""
    mask = torch.empty((1 << 32) + 64, dtype=torch.bool).as_strided((2, 1, 1, 64), (1 << 32, 1, 1, 1))
    with pytest.raises(ValueError):
        _step(_cache(pkg), mask=mask)
    assert launches == []


def test_a_step_of_unsupported_sizes_writes_nothing(pkg, launches):
    with pytest.raises(ValueError):
        _step(_cache(pkg, width=96), width=96)
    with pytest.raises(ValueError):  # rows of two tokens
        _cache(pkg).step(torch.zeros(2, 2, 16, 128, dtype=BF16), *[torch.zeros(2, 8, 2, 128, dtype=BF16)] * 2, 0)
    assert launches == []


@pytest.mark.parametrize('shape', [(2, 1, 1, 1), (1, 1, 1, 1), (1, 1), (1,)], ids=str)
@pytest.mark.parametrize('dtype', [torch.bool, BF16, torch.float32], ids=str)
def test_a_mask_of_one_term_is_for_all_keys(pkg, launches, shape, dtype):
    pkg.paged_attention(**_tensors(), mask=torch.ones(shape, dtype=dtype))
    a = launches[0][1]
    assert a.ctx == 64 and a.mask and a.mask_stride_t == 0 and a.mask_stride_b == (1 if shape[0] == 2 else 0)


def test_a_mask_of_several_keys_bounds_them(pkg, launches):
    pkg.paged_attention(**_tensors(), mask=torch.ones(2, 1, 1, 2, dtype=torch.bool))
    pkg.paged_attention(**_tensors(), mask=torch.ones(2, 1, 1, 64, dtype=torch.bool))
    pkg.paged_attention(**_tensors())
    assert [call[1].ctx for call in launches] == [2, 64, 64]
    assert launches[0][1].mask_stride_t == launches[1][1].mask_stride_t == 1


@pytest.mark.parametrize('dtype', [torch.bool, BF16], ids=str)
def test_a_step_refuses_a_mask_of_one_key(pkg, launches, dtype):
    for shape in ((2, 1, 1, 1), (1, 1, 1, 1), (1,)):
        with pytest.raises(ValueError, match='key dimension'):
            _step(_cache(pkg), mask=torch.ones(shape, dtype=dtype))
    assert launches == []


def test_a_step_over_one_key_takes_its_mask(pkg, launches):
    cache = _cache(pkg)
    cache.arena.page_size = 1
    cache.arena.keys, cache.arena.values = [[torch.zeros(9, 8, 1, 128, dtype=BF16)] for _ in range(2)]
    cache.page_table = torch.zeros(2, 1, dtype=torch.int32)
    _step(cache, mask=torch.ones(2, 1, 1, 1, dtype=torch.bool))
    assert [call[0] for call in launches] == ['write', 'attend'] and launches[1][1].ctx == 1


@pytest.mark.parametrize('implementation', ['eager', 'sdpa'])
def test_masks_that_transformers_builds_are_refused(pkg, launches, implementation):
    from transformers import Qwen3Config
    from transformers.masking_utils import create_causal_mask
    config = Qwen3Config(hidden_size=256, num_attention_heads=2, num_key_value_heads=1, head_dim=128, num_hidden_layers=1)
    config._attn_implementation = implementation
    cache = _cache(pkg)
    padded = torch.ones(2, 40, dtype=torch.int64)
    padded[0, :7] = 0
    mask = create_causal_mask(config=config, inputs_embeds=torch.zeros(2, 1, 256, dtype=BF16), attention_mask=padded,
                              past_key_values=cache, position_ids=torch.tensor([[39], [39]]))
    assert mask is not None
    with pytest.raises(ValueError):
        _step(cache, mask=mask)
    assert launches == []


def test_overlapping_rows_are_told_from_others(pkg):
    overlap = importlib.import_module(pkg.__name__ + '.paged')._rows_overlap
    rng, found = random.Random(0), [0, 0]
    for _ in range(20000):
        row, counts = rng.randrange(1, 6), [rng.randrange(1, 6) for _ in range(2)]
        strides = [rng.choice([0, rng.randrange(0, 12), rng.randrange(0, 60)]) for _ in range(2)]
        places = [i * strides[0] + j * strides[1] + e for i in range(counts[0]) for j in range(counts[1]) for e in range(row)]
        want = len(set(places)) < len(places)
        assert overlap(row, counts[0], strides[0], counts[1], strides[1]) == want, (row, counts, strides)
        found[want] += 1
    assert min(found) > 1000


@pytest.mark.parametrize('strides,refused', [
    ((2048, 128), False), ((128, 256), False), ((4096, 256), False), ((2048 + 64, 128), False), ((128, 384), False),
    ((192, 384), False), ((0, 128), True), ((2048, 0), True), ((2048, 64), True), ((1024, 128), True), ((64, 256), True),
    ((2047, 128), True), ((384, 192), True),
], ids=str)
def test_outputs_whose_rows_share_memory_are_refused(pkg, launches, strides, refused):
    out = torch.zeros(20000, dtype=BF16).as_strided((2, 1, 16, 128), (strides[0], 128, strides[1], 1))
    if refused:
        with pytest.raises(ValueError, match='share memory'):
            pkg.paged_attention(**_tensors(), out=out)
        assert launches == []
    else:
        assert pkg.paged_attention(**_tensors(), out=out) is out and len(launches) == 1


def test_outputs_over_other_rows_of_the_query_are_refused(pkg, launches):
    room = torch.zeros(2, 1, 40, 128, dtype=BF16)
    call = _tensors()
    call['query'] = room[:, :, 8:24]
    for out in (room[:, :, 7:23], room[:, :, 9:25], room[:, :, :16], room[:, :, 23:39], room.view(-1)[8 * 128:][:4096].view(2, 1, 16, 128)):
        with pytest.raises(ValueError, match='query itself'):
            pkg.paged_attention(**call, out=out)
    assert launches == []
    for out in (room[:, :, 8:24], room[:, :, 24:], torch.zeros(2, 1, 16, 128, dtype=BF16)):
        assert pkg.paged_attention(**call, out=out) is out
    one = _tensors(batch=1)
    view = one['query'].as_strided((1, 1, 16, 128), (7, 11, 128, 1))  # strides of single entries mean nothing
    assert pkg.paged_attention(**one, out=view) is view
    assert len(launches) == 4


def test_empty_tensors_share_no_memory(pkg, launches):
    """Empty tensors have one address, null: calls in place on them do nothing."""
    query, key = torch.zeros(3, 5, 16, 128), torch.zeros(3, 5, 8, 128)
    for at in ((slice(0), slice(None)), (slice(None), slice(0))):
        q, k = query[at], key[at]
        positions = torch.zeros(3, *q.shape[:2], dtype=torch.int64)
        out = pkg.rotary_axes(q, k, positions, (24, 20, 20), inv_freq=torch.ones(64), inplace=True)
        assert out[0] is q and out[1] is k
    call = _tensors(batch=0)
    for out in (torch.zeros(0, 1, 16, 128, dtype=BF16), torch.zeros(5, 1, 32, 128, dtype=BF16)[:0, :, :16]):
        assert pkg.paged_attention(**call, out=out) is out
    assert launches == []
