"""Pools of 8 bits, rows read out of pages and shared pages without a GPU: the refusals of the wrappers and of the C
entry points before anything is launched, and the arena's accounting of shared pages."""
import ctypes
import importlib
from contextlib import contextmanager
from types import SimpleNamespace

import pytest
import torch

from tests.test_boundary import _c_layout

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.mark.parametrize('name,cls', [('q3t_paged_read_args', 'PagedReadArgs'), ('q3t_paged_scales', 'PagedScales')])
def test_struct_layouts_match_the_header(pkg, tmp_path, name, cls):
    struct = getattr(pkg._lib, cls)
    fields = [f for f, _ in struct._fields_]
    c = _c_layout(name, fields, tmp_path)
    assert c == [ctypes.sizeof(struct)] + [getattr(struct, f).offset for f in fields]


@pytest.fixture
def launches(pkg, monkeypatch):
    """The entry points that would have been called, with their arguments."""
    lib, seen = pkg._lib, []
    paged = importlib.import_module(pkg.__name__ + '.paged')
    real = lib.packed

    @contextmanager
    def on_device(index):
        yield 0

    def packed(name):
        if name.startswith('q3t_paged_workspace'):
            return real(name)
        return lambda *args: seen.append((name, *args)) or 0

    monkeypatch.setattr(lib, 'gpu_index', lambda *tensors: 0)
    monkeypatch.setattr(lib, 'on_device', on_device)
    monkeypatch.setattr(lib, 'packed', packed)
    monkeypatch.setattr(paged, 'workspace', lambda device, size, stream: torch.empty(size, dtype=torch.uint8))
    return seen


def _pools(dtype=torch.int8, width=128, pages=9, heads=8, page=16):
    return [torch.zeros(pages, heads, page, width, dtype=dtype) for _ in range(2)]


def _scales(pages=9, heads=8, page=16):
    return tuple(torch.ones(pages, heads, page) for _ in range(2))


def _attend(pkg, batch=2, table=4, pools=None, dtype=BF16, **kwargs):
    pools = _pools() if pools is None else pools
    return pkg.paged_attention(torch.zeros(batch, 1, 16, pools[0].shape[3], dtype=dtype), *pools, torch.zeros(batch, table, dtype=torch.int32),
                               torch.zeros(batch, dtype=torch.int64), **kwargs)


def _write(pkg, pools, dtype=BF16, **kwargs):
    rows = torch.zeros(2, 8, 3, pools[0].shape[3], dtype=dtype)
    pkg.paged_write(rows, rows, *pools, torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), **kwargs)


def _read(pkg, pools, tokens=3, **kwargs):
    return pkg.paged_read(*pools, torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), tokens, **kwargs)


def test_entry_points_by_the_pools(pkg, launches):
    for held in (torch.int8, E4M3):
        _attend(pkg, pools=_pools(held), scales=_scales())
        _write(pkg, _pools(held), scales=_scales())
        keys, values = _read(pkg, _pools(held), scales=_scales())
        assert keys.dtype == values.dtype == BF16 and keys.shape == values.shape == (2, 8, 3, 128)
    _attend(pkg, pools=_pools(BF16))
    _attend(pkg, pools=_pools(BF16), shared_pages=2)
    _write(pkg, _pools(BF16))
    assert _read(pkg, _pools(F32))[0].dtype == F32
    assert [call[0] for call in launches] == ['q3t_paged_attention_with', 'q3t_paged_write_quantized', 'q3t_paged_read'] * 2 + \
        ['q3t_paged_attention', 'q3t_paged_attention_with', 'q3t_paged_write', 'q3t_paged_read']
    formats = [pkg._lib.PagedScales.from_buffer_copy(call[-2 if n else 2]).format for call, n in
               ((launches[1], 1), (launches[4], 1))]
    assert formats == [pkg._lib.Q3T_I8, pkg._lib.Q3T_E4M3]
    assert launches[2][2] is not None and launches[-1][2] is None


@pytest.mark.parametrize('pools,scales', [
    (_pools(), None), (_pools(E4M3), None), (_pools(BF16), _scales()), (_pools(torch.uint8), _scales()),
    (_pools(torch.float8_e5m2), _scales()), ([_pools()[0], _pools(E4M3)[0]], _scales()),
    (_pools(), _scales(pages=8)), (_pools(), _scales(page=1)), (_pools(), tuple(x.double() for x in _scales())),
    (_pools(), tuple(x[..., None] for x in _scales())), (_pools(F32), None),
], ids=['int8', 'e4m3', 'bf16 with scales', 'uint8', 'e5m2', 'two types', 'pages', 'rows', 'float64', 'four dims', 'float32'])
def test_pools_and_scales_that_do_not_fit_are_refused(pkg, launches, pools, scales):
    calls = [lambda: _attend(pkg, pools=pools, scales=scales), lambda: _write(pkg, pools, scales=scales)]
    if pools[0].dtype != F32:
        calls.append(lambda: _read(pkg, pools, scales=scales))
    for call in calls:
        with pytest.raises(ValueError):
            call()
    assert launches == []


@pytest.mark.parametrize('shared', [-1, 5, True, 1.0, None, '2'], ids=repr)
def test_shared_pages_outside_the_table_are_refused(pkg, launches, shared):
    with pytest.raises(ValueError):
        _attend(pkg, pools=_pools(BF16), shared_pages=shared)
    assert launches == []


@pytest.mark.parametrize('once', [2, 'yes', 0.5], ids=repr)
def test_other_ways_to_read_are_refused(pkg, launches, once):
    with pytest.raises(ValueError):
        _attend(pkg, pools=_pools(BF16), shared_pages=2, read_once=once)
    assert launches == []


def test_ways_to_read_are_passed_on(pkg, launches):
    for once in (None, True, False):
        _attend(pkg, pools=_pools(BF16), shared_pages=2, read_once=once)
    assert [pkg._lib.PagedArgs.from_buffer_copy(call[1]).reserved for call in launches] == [0, 1, 2]


def test_the_last_row_is_left_to_the_requests(pkg, launches):
    """Of pages that are all shared, and under a mask that ends within them."""
    _attend(pkg, pools=_pools(BF16), shared_pages=4)
    _attend(pkg, pools=_pools(BF16), shared_pages=4, mask=torch.ones(2, 1, 1, 33, dtype=torch.bool))
    _attend(pkg, pools=_pools(BF16), shared_pages=2, mask=torch.ones(2, 1, 1, 33, dtype=torch.bool))
    _attend(pkg, pools=_pools(BF16), shared_pages=2, mask=torch.ones(2, 1, 1, 32, dtype=torch.bool))
    _attend(pkg, pools=_pools(BF16), shared_pages=2, mask=torch.ones(2, 1, 1, 7, dtype=torch.bool))
    assert [call[3] for call in launches] == [3, 2, 2, 1, 0]


@pytest.mark.parametrize('tokens', [-1, 1.0, True, None], ids=repr)
def test_tokens_that_are_no_number_of_rows_are_refused(pkg, launches, tokens):
    with pytest.raises(ValueError):
        _read(pkg, _pools(BF16), tokens=tokens)
    assert launches == []


def test_outputs_of_a_read_that_do_not_fit_are_refused(pkg, launches):
    x = torch.zeros(2, 8, 3, 128, dtype=BF16)
    for out in ((x, x), (x, x[:, :, :2]), (x, x.float()), (x.transpose(2, 3).contiguous().transpose(2, 3), x.clone()),
                (x[:1].expand(2, 8, 3, 128), x.clone())):
        with pytest.raises(ValueError):
            _read(pkg, _pools(BF16), out=out)
    for bad in (dict(dtype=torch.float64), dict(dtype=F32), dict(lengths=torch.zeros(2)), dict(lengths=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            _read(pkg, _pools(BF16), **bad)
    assert launches == []
    out = (x, x.clone())
    assert all(a is b for a, b in zip(_read(pkg, _pools(BF16), out=out), out))
    assert _read(pkg, _pools(BF16), tokens=0)[0].shape == (2, 8, 0, 128)
    assert len(launches) == 1


def _args(pkg, cls, **changes):
    a = getattr(pkg._lib, cls)()
    if cls == 'PagedArgs':
        a.batch, a.q_heads, a.kv_heads, a.head_dim, a.dtype, a.ctx, a.scale = 2, 16, 8, 128, 0, 64, 0.1
        a.query = a.out = 4096
        a.q_stride_b, a.q_stride_h, a.o_stride_b, a.o_stride_h = 2048, 128, 2048, 128
    else:
        a.batch, a.heads, a.tokens, a.width = 2, 8, 5, 128
        a.keys = a.values = 4096
        a.k_stride_b, a.k_stride_h, a.k_stride_t = 5120, 640, 128
        a.v_stride_b, a.v_stride_h, a.v_stride_t = 5120, 640, 128
    if cls == 'PagedWriteArgs':
        a.elem_size = 2
    a.key_pages = a.value_pages = a.page_table = a.positions = 4096
    a.kp_stride_p, a.kp_stride_h, a.kp_stride_t = 8 * 16 * 128, 16 * 128, 128
    a.vp_stride_p, a.vp_stride_h, a.vp_stride_t = 8 * 16 * 128, 16 * 128, 128
    a.pages, a.page_size, a.table_width, a.table_stride_b = 10, 16, 4, 4
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def _c_scales(pkg, **changes):
    s = pkg._lib.PagedScales()
    s.format, s.key_scales, s.value_scales = pkg._lib.Q3T_I8, 4096, 4096
    s.ks_stride_p, s.ks_stride_h, s.ks_stride_t = 128, 16, 1
    s.vs_stride_p, s.vs_stride_h, s.vs_stride_t = 128, 16, 1
    for name, value in changes.items():
        setattr(s, name, value)
    return s


BAD = [dict(page_size=0), dict(pages=0), dict(table_width=0), dict(key_pages=0), dict(page_table=0), dict(positions=0),
       dict(positions=4100), dict(page_table=4098), dict(key_pages=4104), dict(kp_stride_t=116), dict(vp_stride_p=1), dict(pages=1 << 31)]


@pytest.mark.parametrize('bad', BAD + [dict(tokens=-1), dict(heads=0), dict(batch=-1), dict(width=96), dict(keys=0), dict(lengths=2)], ids=str)
def test_the_c_entry_points_refuse_rows(pkg, bad):
    lib, scales = pkg.library(), _c_scales(pkg)
    assert lib.q3t_paged_write_quantized(_args(pkg, 'PagedWriteArgs', **bad), 0, scales, None) < 0
    assert lib.q3t_paged_read(_args(pkg, 'PagedReadArgs', **bad), scales, None) < 0


@pytest.mark.parametrize('bad', [dict(format=0), dict(format=7), dict(key_scales=0), dict(value_scales=4098)], ids=str)
def test_the_c_entry_points_refuse_scales(pkg, bad):
    lib, scales = pkg.library(), _c_scales(pkg, **bad)
    assert lib.q3t_paged_write_quantized(_args(pkg, 'PagedWriteArgs'), 0, scales, None) < 0
    assert lib.q3t_paged_read(_args(pkg, 'PagedReadArgs'), scales, None) < 0
    a = _args(pkg, 'PagedArgs', workspace=1 << 20, workspace_bytes=1 << 40)
    assert lib.q3t_paged_attention_with(a, scales, 0, None) < 0


def test_the_c_entry_points_refuse_types(pkg):
    lib, scales = pkg.library(), _c_scales(pkg)
    assert lib.q3t_paged_write_quantized(None, 0, scales, None) == -1
    assert lib.q3t_paged_write_quantized(_args(pkg, 'PagedWriteArgs'), 0, None, None) == -1
    assert lib.q3t_paged_write_quantized(_args(pkg, 'PagedWriteArgs'), 2, scales, None) == -1
    assert lib.q3t_paged_write_quantized(_args(pkg, 'PagedWriteArgs'), 3, scales, None) == -2
    assert lib.q3t_paged_read(None, None, None) == -1
    assert lib.q3t_paged_read(_args(pkg, 'PagedReadArgs', dtype=4), None, None) == -2
    assert lib.q3t_paged_read(_args(pkg, 'PagedReadArgs', batch=0), scales, None) == 0
    assert lib.q3t_paged_write_quantized(_args(pkg, 'PagedWriteArgs', tokens=0), 0, scales, None) == 0


@pytest.mark.parametrize('bad', BAD + [dict(ctx=65), dict(ctx=0), dict(head_dim=96), dict(dtype=3), dict(q_heads=12), dict(query=0), dict(out=0),
                                       dict(query=4104), dict(q_stride_h=4), dict(workspace=0), dict(workspace_bytes=8), dict(mask=4096, mask_dtype=9),
                                       dict(o_stride_b=-1), dict(reserved=3), dict(reserved=-1)], ids=str)
@pytest.mark.parametrize('held,shared', [(True, 0), (False, 2), (True, 2)])
def test_the_c_entry_point_refuses_attention(pkg, bad, held, shared):
    a = _args(pkg, 'PagedArgs', **{**dict(workspace=1 << 20, workspace_bytes=1 << 40), **bad})
    assert pkg.library().q3t_paged_attention_with(a, _c_scales(pkg) if held else None, shared, None) < 0


def test_the_c_entry_point_refuses_shared_pages(pkg):
    lib = pkg.library()
    for shared in (-1, 4, 5, 1 << 40):
        a = _args(pkg, 'PagedArgs', workspace=1 << 20, workspace_bytes=1 << 40)
        assert lib.q3t_paged_attention_with(a, None, shared, None) == -1
        assert lib.q3t_paged_workspace_bytes_with(a, None, shared) == -1
    small, large = (lib.q3t_paged_workspace_bytes_with(_args(pkg, 'PagedArgs', reserved=way), None, 3) for way in (2, 1))
    assert 0 < small < large
    assert lib.q3t_paged_workspace_bytes_with(_args(pkg, 'PagedArgs'), _c_scales(pkg), 3) > 0
    assert lib.q3t_paged_workspace_bytes_with(None, None, 0) == -1


@pytest.mark.parametrize('way', [0, 1, 2])
def test_attention_without_requests_is_none(pkg, way):
    lib, a = pkg.library(), _args(pkg, 'PagedArgs', batch=0, reserved=way)
    for held in (None, _c_scales(pkg)):
        assert lib.q3t_paged_workspace_bytes_with(a, held, 2) >= 0
        assert lib.q3t_paged_attention_with(a, held, 2, None) == 0


@pytest.mark.parametrize('bad', [dict(heads=(1 << 32) + 8), dict(tokens=(1 << 32) + 5), dict(heads=1 << 40, tokens=0)], ids=str)
def test_the_c_entry_points_refuse_counts_past_32_bits(pkg, bad):
    lib, scales = pkg.library(), _c_scales(pkg)
    expected = 0 if bad.get('tokens') == 0 else -2
    assert lib.q3t_paged_write_quantized(_args(pkg, 'PagedWriteArgs', **bad), 0, scales, None) == expected
    assert lib.q3t_paged_read(_args(pkg, 'PagedReadArgs', **bad), scales, None) == expected
    assert lib.q3t_paged_read(_args(pkg, 'PagedReadArgs', **bad), None, None) == expected


# ---- the arena -------------------------------------------------------------------------------

def _arena(pkg, **kwargs):
    module = torch.nn.Linear(2, 2).bfloat16()
    reference = SimpleNamespace(parameters=module.parameters, layers=[None, None],
                                config=SimpleNamespace(num_key_value_heads=8, head_dim=128))
    return pkg.PagedArena(reference, pages=9, page_size=16, **kwargs)


def test_shared_pages_are_released_as_often_as_they_were_taken(pkg):
    arena = _arena(pkg)
    prompt = arena.allocate(3)
    assert arena.share(prompt) == prompt and arena.share(prompt[:1]) == prompt[:1]
    own = arena.allocate(2)
    assert arena.free_pages == 4
    arena.release(prompt + own)
    assert arena.free_pages == 6
    arena.release(prompt)
    assert arena.free_pages == 8
    with pytest.raises(ValueError):
        arena.release(prompt)
    assert arena.free_pages == 8
    arena.release(prompt[:1])
    assert arena.free_pages == 9 and sorted(arena.allocate(9)) == list(range(9))
    for bad in ([3, 3], [9], [-1]):
        with pytest.raises(ValueError):
            arena.share(bad)
    arena.release(range(9))
    with pytest.raises(ValueError):
        arena.share([0])
    assert arena.free_pages == 9


def test_arenas_of_8_bits(pkg):
    for held in (torch.int8, E4M3):
        arena = _arena(pkg, dtype=held)
        assert arena.packed.dtype == held and arena.packed_scales.shape == (4, 9, 8, 16)
        keys, values = arena.scales[1]
        assert keys.data_ptr() == arena.packed_scales[1].data_ptr() and values.data_ptr() == arena.packed_scales[3].data_ptr()
    assert _arena(pkg).scales == [None, None] and _arena(pkg, dtype=BF16).packed.dtype == BF16
    for bad in (torch.float16, torch.uint8, torch.float8_e5m2):
        with pytest.raises(ValueError):
            _arena(pkg, dtype=bad)


@pytest.mark.parametrize('held', [None, torch.int8, E4M3], ids=str)
def test_a_step_and_its_prompts_follow_the_arena(pkg, launches, held):
    arena = _arena(pkg, dtype=held)
    table = torch.zeros(2, 4, dtype=torch.int32)
    cache = pkg.PagedCache(arena, table, torch.zeros(2, dtype=torch.int64), shared_pages=2)
    rows = torch.zeros(2, 8, 1, 128, dtype=BF16)
    cache.step(torch.zeros(2, 1, 16, 128, dtype=BF16), rows, rows, 1)
    layer = SimpleNamespace(keys=torch.zeros(2, 8, 5, 128, dtype=BF16), values=torch.zeros(2, 8, 5, 128, dtype=BF16))
    arena.load(table, SimpleNamespace(layers=[layer, layer]), torch.zeros(2, dtype=torch.int32))
    assert arena.read(table, 5).shape == (4, 2, 8, 5, 128)
    write = 'q3t_paged_write' if held is None else 'q3t_paged_write_quantized'
    assert [call[0] for call in launches] == [write, 'q3t_paged_attention_with', write, write, 'q3t_paged_read', 'q3t_paged_read']
    assert launches[1][3] == 2 and (launches[1][2] is None) == (held is None)


def test_a_refused_step_writes_nothing(pkg, launches):
    arena = _arena(pkg, dtype=torch.int8)
    rows = torch.zeros(2, 8, 1, 128, dtype=BF16)
    cache = pkg.PagedCache(arena, torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), shared_pages=5)
    with pytest.raises(ValueError):
        cache.step(torch.zeros(2, 1, 16, 128, dtype=BF16), rows, rows, 0)
    assert launches == []
