"""The paged cache and the several-axes rotary without a GPU: refusals of the wrappers and of the
C entry points, before anything is launched, the index arithmetic compiled by the host compiler,
and the arena's page accounting."""
import ctypes
import importlib
import random
import subprocess
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from tests.test_boundary import _c_layout

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / 'qwen3-tts-rsi-engine_amd' / 'csrc'


@pytest.mark.parametrize('name,cls', [('q3t_paged_write_args', 'PagedWriteArgs'), ('q3t_paged_args', 'PagedArgs'),
                                      ('q3t_rotary_axes_args', 'RotaryAxesArgs')])
def test_struct_layouts_match_the_header(pkg, tmp_path, name, cls):
    struct = getattr(pkg._lib, cls)
    fields = [f for f, _ in struct._fields_]
    c = _c_layout(name, fields, tmp_path)
    assert c == [ctypes.sizeof(struct)] + [getattr(struct, f).offset for f in fields]


@pytest.fixture(scope='module')
def index(tmp_path_factory):
    """csrc/paged_index.hpp built by g++ alone."""
    where = tmp_path_factory.mktemp('index')
    (where / 'index.cpp').write_text(f'''
#include "{CSRC / 'paged_index.hpp'}"
extern "C" uint32_t quotient(uint32_t n, uint32_t d) {{ return q3t::divide(n, q3t::divisor(d)); }}
extern "C" void share_out(uint32_t pairs, uint32_t stages, uint32_t pieces, uint32_t least, uint32_t cost, uint32_t workgroups, uint32_t *out) {{
    const q3t::Sharing s = q3t::sharing(pairs, stages, pieces, least, cost, q3t::divisor(workgroups));
    out[0] = s.unit; out[1] = s.cost; out[2] = s.share; out[3] = s.total;
}}
static q3t::Sharing of(const uint32_t *s) {{ return {{s[0], s[1], s[2], s[3]}}; }}
extern "C" uint32_t places(uint32_t stages, const uint32_t *sharing) {{ return q3t::places(stages, of(sharing)); }}
static void put(const q3t::Cursor &c, uint32_t *cursor) {{
    const uint32_t after[5] = {{c.x, c.left, c.b, c.head, c.off}};
    for (int i = 0; i < 5; ++i) cursor[i] = after[i];
}}
extern "C" void end_pair(uint32_t *cursor, uint32_t length, uint32_t heads) {{
    q3t::Cursor c = {{cursor[0], cursor[1], cursor[2], cursor[3], cursor[4]}};
    q3t::end_pair(c, length, heads);
    put(c, cursor);
}}
extern "C" void next_run(uint32_t *cursor, uint32_t stages, uint32_t heads, const uint32_t *sharing, uint32_t *out) {{
    q3t::Cursor c = {{cursor[0], cursor[1], cursor[2], cursor[3], cursor[4]}};
    const q3t::Run r = q3t::next_run(c, stages, heads, of(sharing));
    put(c, cursor);
    const uint32_t run[7] = {{r.b, r.head, r.lo, r.hi, r.first, r.parts, r.begins}};
    for (int i = 0; i < 7; ++i) out[i] = run[i];
}}
''')
    subprocess.run(['g++', '-std=c++17', '-O2', '-shared', '-fPIC', '-fsanitize=undefined', '-fno-sanitize-recover',
                    str(where / 'index.cpp'), '-o', str(where / 'index.so')], check=True)
    lib = ctypes.CDLL(str(where / 'index.so'))
    lib.quotient.argtypes, lib.quotient.restype = [ctypes.c_uint32] * 2, ctypes.c_uint32
    return lib


def test_division(index):
    rng = random.Random(0)
    top = 2 ** 31 - 1
    divisors = list(range(1, 130)) + [2 ** k + e for k in range(2, 31) for e in (-1, 0, 1)] + [top - 1, top]
    for d in divisors + [rng.randrange(1, top) for _ in range(200)]:
        for n in [0, 1, d - 1, d, min(d + 1, top), 2 * d - 1 if 2 * d - 1 <= top else top, top // d * d, max(top // d * d - 1, 0), top] + \
                 [rng.randrange(0, top) for _ in range(20)]:
            assert index.quotient(n, d) == n // d, (n, d)


@pytest.mark.parametrize('seed', range(80))
def test_shares_cover_every_pair_once(index, seed):
    """Every workgroup's runs, together: each stage of each pair exactly once, in one run per share,
    parts numbered from the pair's first share, at most two unfinished states a workgroup and no slot
    of them twice."""
    rng = random.Random(seed)
    heads, workgroups, least = rng.choice([1, 2, 3, 8]), rng.choice([1, 3, 16, 64, 512]), rng.choice([1, 4, 8])
    cost = rng.choice([0, 1, 3, 7])
    stages = [rng.choice([1, 1, 2, 3, rng.randrange(1, 17), rng.randrange(1, 900)]) for _ in range(rng.choice([1, 2, 7, 40]))]
    u32 = ctypes.c_uint32
    sharing = (u32 * 4)()
    index.share_out(len(stages) * heads, sum(stages) * heads, sum(-(-r // least) for r in stages) * heads, least, cost, workgroups, sharing)
    unit, extra, share, total = sharing
    length = [index.places(r, sharing) for r in stages]
    assert total == heads * sum(length) and share * workgroups >= total and share >= 1
    covered, parts, slots = {}, {}, set()
    for w in range(workgroups):
        x = w * share
        if x >= total:
            continue
        off, b = x, 0
        while off >= length[b] * heads:
            off -= length[b] * heads
            b += 1
        cursor = (u32 * 5)(x, min(share, total - x), b, off // length[b], off % length[b])
        if cursor[4] >= stages[b]:
            index.end_pair(cursor, length[b], heads)
        unfinished = 0
        while cursor[1]:
            out = (u32 * 7)()
            index.next_run(cursor, stages[cursor[2]], heads, sharing, out)
            rb, head, lo, hi, first, count, begins = out
            assert lo < hi <= stages[rb]
            for r in range(lo, hi):
                assert (rb, head, r) not in covered
                covered[rb, head, r] = w
            if count == 1:
                first = w
            assert begins == (lo == 0) and first <= w < first + count
            assert parts.setdefault((rb, head), (first, count)) == (first, count)
            assert (w == first) == bool(begins)
            if count > 1:
                unfinished += 1
                slot = 2 * w + begins
                assert slot not in slots
                slots.add(slot)
        assert unfinished <= 2
    assert len(covered) == heads * sum(stages)
    for (rb, head), (first, count) in parts.items():
        assert {covered[rb, head, r] for r in range(stages[rb])} == set(range(first, first + count))


def _attend_args(pkg, **changes):
    a = pkg._lib.PagedArgs()
    a.batch, a.q_heads, a.kv_heads, a.head_dim, a.dtype, a.ctx, a.scale = 2, 16, 8, 128, 0, 64, 0.1
    a.query = a.key_pages = a.value_pages = a.page_table = a.positions = a.out = 4096
    a.q_stride_b, a.q_stride_h, a.o_stride_b, a.o_stride_h = 2048, 128, 2048, 128
    a.kp_stride_p, a.kp_stride_h, a.kp_stride_t = 8 * 16 * 128, 16 * 128, 128
    a.vp_stride_p, a.vp_stride_h, a.vp_stride_t = 8 * 16 * 128, 16 * 128, 128
    a.pages, a.page_size, a.table_width, a.table_stride_b = 10, 16, 4, 4
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize('changes,status', [
    (dict(batch=-1), -1), (dict(q_heads=0), -1), (dict(kv_heads=0), -1), (dict(q_heads=12), -1), (dict(ctx=0), -1),
    (dict(ctx=65), -1), (dict(pages=0), -1), (dict(page_size=0), -1), (dict(table_width=0), -1),
    (dict(head_dim=96), -2), (dict(head_dim=256), -2), (dict(dtype=3), -2), (dict(dtype=7), -2), (dict(pages=1 << 31), -2),
    (dict(ctx=1 << 30, table_width=1 << 30), -2), (dict(page_size=1 << 31), -2), (dict(table_width=1 << 31), -2),
    (dict(batch=1 << 17), -2), (dict(batch=1 << 16, q_heads=32, kv_heads=2), -2),
    (dict(query=None), -1), (dict(key_pages=None), -1), (dict(value_pages=None), -1), (dict(page_table=None), -1),
    (dict(positions=None), -1), (dict(out=None), -1), (dict(key_pages=4104), -1), (dict(value_pages=4100), -1),
    (dict(query=4098), -1), (dict(kp_stride_t=132), -1), (dict(vp_stride_h=4), -1), (dict(kp_stride_p=1), -1),
    (dict(q_stride_b=2), -1), (dict(page_table=4097), -1), (dict(positions=4100), -1), (dict(out=4097), -1),
    (dict(mask=4096, mask_dtype=4), -1), (dict(mask=4096, mask_dtype=-1), -1),
])
def test_attention_entry_refuses(pkg, changes, status):
    lib = pkg.library()
    a = _attend_args(pkg, workspace=4096, workspace_bytes=1 << 40, **changes)
    assert lib.q3t_paged_attention(a, None) == status
    assert lib.q3t_paged_attention(None, None) == -1


def test_empty_calls_launch_nothing(pkg):
    lib = pkg.library()
    assert lib.q3t_paged_attention(_attend_args(pkg, batch=0, query=None, out=None), None) == 0
    a = pkg._lib.PagedWriteArgs()
    a.batch, a.heads, a.tokens, a.width, a.elem_size, a.pages, a.page_size, a.table_width = 0, 1, 1, 64, 2, 1, 1, 1
    assert lib.q3t_paged_write(a, None) == 0
    a.batch, a.tokens = 3, 0
    assert lib.q3t_paged_write(a, None) == 0
    r = pkg._lib.RotaryAxesArgs()
    r.batch, r.tokens, r.q_heads, r.k_heads, r.width, r.dtype, r.axes = 0, 5, 1, 0, 64, 0, 1
    r.sections[0] = 32
    assert lib.q3t_rotary_axes(r, None) == 0


@pytest.mark.parametrize('changes,status', [
    (dict(batch=-1), -1), (dict(heads=0), -1), (dict(tokens=-1), -1), (dict(width=0), -1), (dict(pages=0), -1),
    (dict(page_size=0), -1), (dict(table_width=0), -1), (dict(elem_size=1), -2), (dict(elem_size=8), -2),
    (dict(keys=None), -1), (dict(values=None), -1), (dict(key_pages=None), -1), (dict(value_pages=None), -1),
    (dict(page_table=None), -1), (dict(positions=None), -1), (dict(keys=4097), -1), (dict(positions=4100), -1),
    (dict(lengths=4098), -1), (dict(pages=1 << 31), -2), (dict(table_width=1 << 28, page_size=16), -2),
    (dict(tokens=1 << 31), -2), (dict(heads=1 << 31), -2), (dict(width=1 << 21), -2), (dict(batch=1 << 31), -2),
])
def test_write_entry_refuses(pkg, changes, status):
    a = pkg._lib.PagedWriteArgs()
    a.batch, a.heads, a.tokens, a.width, a.elem_size, a.pages, a.page_size, a.table_width = 2, 8, 1, 128, 2, 10, 16, 4
    a.keys = a.values = a.key_pages = a.value_pages = a.page_table = a.positions = 4096
    for name, value in changes.items():
        setattr(a, name, value)
    lib = pkg.library()
    assert lib.q3t_paged_write(a, None) == status
    assert lib.q3t_paged_write(None, None) == -1


@pytest.mark.parametrize('changes,status', [
    (dict(batch=-1), -1), (dict(tokens=-1), -1), (dict(q_heads=0), -1), (dict(k_heads=-1), -1), (dict(axes=0), -1),
    (dict(axes=5), -1), (dict(sections=(0, 0, 0, 0)), -1), (dict(sections=(-1, 9, 0, 0)), -1),
    (dict(sections=(40, 20, 20, 0)), -1), (dict(sections=(1 << 40, 0, 0, 0)), -1), (dict(dtype=3), -2), (dict(width=1), -1),
    (dict(width=1 << 17), -2), (dict(q_heads=1 << 17), -2), (dict(batch=1 << 40), -2), (dict(tokens=1 << 62), -2),
    (dict(width=2048, sections=(600, 0, 0, 0)), -2), (dict(query=None), -1), (dict(q_out=None), -1), (dict(key=None), -1),
    (dict(k_out=None), -1), (dict(turns=None), -1), (dict(positions=None), -1), (dict(query=4097), -1),
    (dict(positions=4100), -1), (dict(turns=4100), -1), (dict(width=65536, q_heads=65536, sections=(1, 0, 0, 0), query=4098), -2),
])
def test_rotary_entry_refuses(pkg, changes, status):
    a = pkg._lib.RotaryAxesArgs()
    a.batch, a.tokens, a.q_heads, a.k_heads, a.width, a.dtype, a.axes = 2, 3, 16, 8, 128, 0, 3
    a.sections[0], a.sections[1], a.sections[2] = 24, 20, 20
    a.query = a.key = a.q_out = a.k_out = a.turns = a.positions = 4096
    for name, value in changes.items():
        setattr(a, name, (ctypes.c_int64 * 4)(*value) if name == 'sections' else value)
    lib = pkg.library()
    assert lib.q3t_rotary_axes(a, None) == status
    assert lib.q3t_rotary_axes(None, None) == -1


def _tensors(batch=2, q_heads=16, kv_heads=8, width=128, page=16, pages=9, table=4, dtype=torch.bfloat16):
    return dict(query=torch.zeros(batch, 1, q_heads, width, dtype=dtype),
                key_pages=torch.zeros(pages, kv_heads, page, width, dtype=dtype),
                value_pages=torch.zeros(pages, kv_heads, page, width, dtype=dtype),
                page_table=torch.zeros(batch, table, dtype=torch.int32), positions=torch.zeros(batch, dtype=torch.int64))


@pytest.mark.parametrize('change', [
    dict(query=torch.zeros(2, 2, 16, 128, dtype=torch.bfloat16)), dict(query=torch.zeros(2, 16, 128, dtype=torch.bfloat16)),
    dict(query=torch.zeros(2, 1, 12, 128, dtype=torch.bfloat16)), dict(query=torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)),
    dict(query=torch.zeros(2, 1, 16, 128)), dict(query=torch.zeros(2, 1, 16, 256, dtype=torch.bfloat16)[..., ::2]),
    dict(query=torch.zeros(3, 1, 16, 128, dtype=torch.bfloat16)),
    dict(value_pages=torch.zeros(9, 8, 8, 128, dtype=torch.bfloat16)), dict(value_pages=torch.zeros(9, 8, 16, 128)),
    dict(key_pages=torch.zeros(9, 8, 128, 16, dtype=torch.bfloat16).transpose(2, 3)),
    dict(page_table=torch.zeros(2, 4, dtype=torch.int64)), dict(page_table=torch.zeros(8, dtype=torch.int32)),
    dict(page_table=torch.zeros(2, 0, dtype=torch.int32)), dict(page_table=torch.zeros(2, 8, dtype=torch.int32)[:, ::2]),
    dict(positions=torch.zeros(2, dtype=torch.int32)), dict(positions=torch.zeros(2, 1, dtype=torch.int64)),
    dict(positions=torch.zeros(4, dtype=torch.int64)[::2]), dict(),  # the last: CPU tensors
])
def test_attention_wrapper_refuses(pkg, change):
    with pytest.raises(ValueError):
        pkg.paged_attention(**{**_tensors(), **change})


@pytest.mark.parametrize('change', [
    dict(values=torch.zeros(2, 8, 3, 128, dtype=torch.bfloat16)), dict(keys=torch.zeros(2, 8, 128, dtype=torch.bfloat16)),
    dict(keys=torch.zeros(2, 8, 1, 128), values=torch.zeros(2, 8, 1, 128)),
    dict(keys=torch.zeros(2, 8, 1, 64, dtype=torch.bfloat16), values=torch.zeros(2, 8, 1, 64, dtype=torch.bfloat16)),
    dict(keys=torch.zeros(2, 4, 1, 128, dtype=torch.bfloat16), values=torch.zeros(2, 4, 1, 128, dtype=torch.bfloat16)),
    dict(key_pages=torch.zeros(9, 8, 16, 128)), dict(page_table=torch.zeros(3, 4, dtype=torch.int32)),
    dict(positions=torch.zeros(3, dtype=torch.int64)), dict(),
])
def test_write_wrapper_refuses(pkg, change):
    t = _tensors()
    del t['query']
    rows = torch.zeros(2, 8, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        pkg.paged_write(**{**t, 'keys': rows, 'values': rows, **change})


@pytest.mark.parametrize('change', [
    dict(query=torch.zeros(2, 16, 128)), dict(key=torch.zeros(2, 4, 8, 128)), dict(key=torch.zeros(2, 3, 8, 64)),
    dict(key=torch.zeros(2, 3, 8, 128).half()), dict(query=torch.zeros(2, 3, 16, 128).double(), key=None),
    dict(sections=()), dict(sections=(1, 1, 1, 1, 1)), dict(sections=(0, 0, 0)), dict(sections=(40, 20, 20)),
    dict(sections=(-1, 3, 3)), dict(sections=(2.0, 3, 3)), dict(positions=torch.zeros(2, 2, 3, dtype=torch.int64)),
    dict(positions=torch.zeros(3, 2, 3, dtype=torch.int32)), dict(inv_freq=torch.ones(63)), dict(),
])
def test_rotary_wrapper_refuses(pkg, change):
    call = dict(query=torch.zeros(2, 3, 16, 128), key=torch.zeros(2, 3, 8, 128),
                positions=torch.zeros(3, 2, 3, dtype=torch.int64), sections=(24, 20, 20))
    with pytest.raises(ValueError):
        pkg.rotary_axes(**{**call, **change})


def _reference(layers=2):
    module = torch.nn.Linear(2, 2).bfloat16()
    config = SimpleNamespace(num_key_value_heads=8, head_dim=128)
    return SimpleNamespace(parameters=module.parameters, config=config, layers=[None] * layers)


def test_arena_hands_out_every_page_once(pkg):
    arena = pkg.PagedArena(_reference(), pages=7, page_size=16)
    assert arena.packed.shape == (4, 7, 8, 16, 128) and arena.free_pages == 7
    assert [arena.pages_for(n) for n in (0, 1, 16, 17, 160)] == [0, 1, 1, 2, 10]
    first, second = arena.allocate(4), arena.allocate(3)
    assert sorted(first + second) == list(range(7)) and arena.free_pages == 0
    with pytest.raises(ValueError):
        arena.allocate(1)
    for bad in ([first[0], first[0]], [99], [first[0], -1]):
        with pytest.raises(ValueError):
            arena.release(bad)
    assert arena.free_pages == 0
    arena.release(first)
    with pytest.raises(ValueError):
        arena.release(first[:1])
    with pytest.raises(ValueError):
        arena.allocate(5)
    with pytest.raises(ValueError):
        arena.allocate(-1)
    assert sorted(arena.allocate(4)) == sorted(first)
    table = arena.page_table([second, [], first[:2]])
    assert table.dtype == torch.int32 and table.tolist() == [second, [-1] * 3, first[:2] + [-1]]
    assert arena.page_table([[]]).tolist() == [[-1]] and arena.page_table([], width=2).shape == (0, 2)
    assert arena.page_table([[3]], width=4).tolist() == [[3, -1, -1, -1]]
    with pytest.raises(ValueError):
        arena.page_table([first], width=3)
    for bad in (dict(pages=0), dict(pages=3, page_size=0)):
        with pytest.raises(ValueError):
            pkg.PagedArena(_reference(), **bad)


def test_a_prefill_cache_of_other_layers_is_refused(pkg):
    arena = pkg.PagedArena(_reference(), pages=4)
    rows = torch.zeros(1, 8, 3, 128, dtype=torch.bfloat16)
    cache = SimpleNamespace(layers=[SimpleNamespace(keys=rows, values=rows)])
    with pytest.raises(ValueError, match='layers'):
        arena.load(arena.page_table([[0]]), cache, torch.tensor([3], dtype=torch.int32))


def _places(t):
    return torch.arange(100000).as_strided(t.shape, t.stride(), t.storage_offset()).flatten().tolist()


@pytest.mark.parametrize('seed', range(20))
def test_rows_that_share_memory_are_found(pkg, seed):
    """No overlap is missed, whatever the strides."""
    share = importlib.import_module(pkg.__name__ + '.rotary')._share_memory
    rng = torch.Generator().manual_seed(seed)
    memory = torch.zeros(20000, dtype=torch.float16)
    number = lambda low, high: int(torch.randint(low, high + 1, (1,), generator=rng))
    apart = 0
    for _ in range(300):
        width, strides = number(1, 4), [number(0, 40) for _ in range(3)]
        views = []
        for _ in range(2):
            shape = [number(1, 3) for _ in range(3)]
            if number(0, 2) == 0:
                strides = [number(0, 40) for _ in range(3)]
            views.append(memory.as_strided(shape + [width], strides + [1], number(0, 60)))
        x, y = views
        for t in views:
            if len(set(_places(t))) < t.numel():
                assert share(t)
        if set(_places(x)) & set(_places(y)):
            assert share(x, y)
        elif not share(x, y):
            apart += 1
    assert apart > 30  # some were told apart


def test_rows_of_one_projection_do_not_share_memory(pkg):
    share = importlib.import_module(pkg.__name__ + '.rotary')._share_memory
    fused = torch.zeros(3, 5, 28, 16)
    per_head = torch.zeros(3, 5, 8, 3, 16)
    bnsd = torch.zeros(3, 24, 5, 16).transpose(1, 2)
    for q, k in ((fused[:, :, :16], fused[:, :, 16:24]), (fused[:, :, 8:24], fused[:, :, :8]), (fused[:1, :, :16], fused[:1, :, 16:20]),
                 (fused[:, :1, :16], fused[:, :1, 27:]), (per_head[:, :, :, 0], per_head[:, :, :, 1]),
                 (per_head[:, :, :, 2], per_head[:, :, :, 0]), (bnsd[:, :, :16], bnsd[:, :, 16:]), (fused, bnsd),
                 (fused[..., :8], fused[..., 8:])):
        assert not share(q) and not share(k) and not share(q, k) and not share(k, q)
    for q, k in ((fused, fused), (fused[:, :, :16], fused[:, :, 15:24]), (fused[..., :8], fused[..., 4:12]), (fused, fused[1:])):
        assert share(q, k) and share(k, q)
    assert share(fused[:, :, :1].expand(3, 5, 4, 16)) and share(torch.zeros(200).as_strided((1, 4, 4, 16), (0, 16, 15, 1)))
