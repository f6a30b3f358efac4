"""Shared pages of the paged cache without a GPU: what launches of any length have for their work, which calls are refused, and
which way the library reads."""
import ctypes
import subprocess
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

CSRC = Path(__file__).resolve().parents[1] / 'qwen3-tts-rsi-engine_amd' / 'csrc'


@pytest.fixture(scope='module')
def whole_pair(tmp_path_factory):
    """The run of a workgroup that has a pair to itself: (head, lo, hi, parts, begins, places left)."""
    where = tmp_path_factory.mktemp('whole')
    (where / 'whole.cpp').write_text(f'''
#include "{CSRC / 'paged_index.hpp'}"
extern "C" void run(uint32_t b, uint32_t head, uint32_t stages, uint32_t heads, uint32_t *out) {{
    q3t::Cursor at = q3t::whole_pair_at(b, head);
    const q3t::Run r = q3t::next_run(at, stages, heads, q3t::whole_pair());
    const uint32_t all[7] = {{r.b, r.head, r.lo, r.hi, r.parts, r.begins, at.left}};
    for (int i = 0; i < 7; ++i) out[i] = all[i];
}}
''')
    subprocess.run(['g++', '-std=c++17', '-O2', '-shared', '-fPIC', '-fsanitize=undefined', '-fno-sanitize-recover',
                    str(where / 'whole.cpp'), '-o', str(where / 'whole.so')], check=True)
    lib = ctypes.CDLL(str(where / 'whole.so'))

    def run(*args):
        out = (ctypes.c_uint32 * 7)()
        lib.run(*args, out)
        return list(out)
    return run


@pytest.mark.parametrize('keys', [1, 16, 17, 1024, (1 << 25) - 16, 1 << 25, (1 << 25) + 1, 34_000_000, (1 << 30) - 1])
def test_a_workgroup_of_one_pair_has_all_of_its_stages(whole_pair, keys):
    """Of 16 keys each, up to the longest request that the entry points take."""
    stages = -(-keys // 16)
    for b, head, heads in ((0, 0, 1), (0, 1, 8), (31, 7, 8)):
        assert whole_pair(b, head, stages, heads) == [b, head, 0, stages, 1, 1, 0]


def _args(pkg, **changes):
    a = pkg._lib.PagedArgs()
    a.batch, a.q_heads, a.kv_heads, a.head_dim, a.dtype, a.scale = 2, 16, 8, 128, pkg._lib.Q3T_BF16, 0.1
    a.pages, a.page_size, a.table_width, a.table_stride_b, a.ctx = 10, 16, 4, 4, 64
    for name, value in changes.items():
        setattr(a, name, value)
    a.ctx = changes.get('ctx', a.table_width * a.page_size)
    return a


def _bytes(pkg, shared, **changes):
    return pkg.library().q3t_paged_workspace_bytes_with(_args(pkg, **changes), None, shared)


@pytest.mark.parametrize('dtype,width', [('Q3T_BF16', 128), ('Q3T_F16', 128), ('Q3T_F32', 64), ('Q3T_F32', 128), ('Q3T_BF16', 64)])
@pytest.mark.parametrize('once', ['Q3T_SHARE_AUTO', 'Q3T_SHARE_ALWAYS', 'Q3T_SHARE_NEVER'])
def test_calls_of_too_many_stages_are_refused_however_much_is_shared(pkg, dtype, width, once):
    """Stages are counted in 30 bits, those of the requests' shared keys too, which they may have to attend each for itself."""
    ways = {'Q3T_SHARE_AUTO': 0, 'Q3T_SHARE_ALWAYS': 1, 'Q3T_SHARE_NEVER': 2}
    keys = 32 if dtype != 'Q3T_F32' and width == 64 else 16  # of a stage
    sizes = dict(batch=64512, q_heads=1, kv_heads=1, head_dim=width, dtype=getattr(pkg._lib, dtype), page_size=512, reserved=ways[once])
    most = (1 << 30) // 64512  # stages of a request
    fits, not_ = ((most - 40) * keys // 512, (most + 40) * keys // 512)
    for entries, good in ((fits, True), (not_, False)):
        for shared in (0, 1, entries - 1):
            assert (_bytes(pkg, shared, table_width=entries, table_stride_b=entries, **sizes) >= 0) == good


# (requests, keys shared, page, query heads, KV heads, width, type, masked, read once), and us read once / request by request
CHOICES = [
    ((8, 512, 16, 16, 8, 128, 'Q3T_BF16', False, False), '16.9 / 12.1'),
    ((8, 4096, 16, 16, 8, 128, 'Q3T_BF16', False, True), '19.7 / 24.5'),
    ((64, 4096, 16, 16, 8, 128, 'Q3T_BF16', False, True), '32.3 / 108'),
    ((64, 4096, 16, 16, 8, 128, 'Q3T_F32', False, True), '70.5 / 260'),
    ((128, 16384, 64, 32, 8, 128, 'Q3T_BF16', False, True), '103 / 965'),
    ((64, 512, 16, 16, 8, 128, 'Q3T_BF16', True, False), '47.2 / 33.2'),
    ((64, 4096, 16, 16, 8, 128, 'Q3T_BF16', True, True), '49.6 / 121'),
    ((21, 792, 24, 12, 12, 64, 'Q3T_F32', True, True), '24.2 / 29.0'),
    ((16, 4096, 16, 40, 2, 128, 'Q3T_F32', False, False), '98.6 / 49.2'),
    ((16, 4096, 16, 40, 2, 128, 'Q3T_F16', False, False), '33.9 / 26.1'),
    ((16, 4096, 16, 40, 2, 64, 'Q3T_F32', False, False), '40.5 / 29.0'),
    ((26, 13568, 32, 8, 1, 128, 'Q3T_F32', True, False), '217 / 68'),
    ((97, 2048, 256, 16, 1, 128, 'Q3T_BF16', False, False), '34.6 / 24.2'),
    ((64, 4096, 1, 16, 8, 128, 'Q3T_BF16', False, True), '39.3 / 126'),
    ((10, 389, 1, 64, 8, 128, 'Q3T_F32', False, False), '28.6 / 16.3'),
]


@pytest.mark.parametrize('case,times', CHOICES, ids=[str(c[0][:-1]) for c in CHOICES])
def test_the_library_chooses_what_is_quicker(pkg, case, times):
    """By the workspace that it asks for, which reading once needs more of."""
    batch, keys, page, q_heads, kv_heads, width, dtype, masked, once = case
    shared = keys // page
    sizes = dict(batch=batch, q_heads=q_heads, kv_heads=kv_heads, head_dim=width, dtype=getattr(pkg._lib, dtype), page_size=page,
                 pages=shared + 64 * batch, table_width=shared + 64)
    if masked:
        sizes.update(mask=4096, mask_dtype=pkg._lib.Q3T_BOOL, mask_stride_b=keys + 64 * page, mask_stride_t=1)
    chosen, always, never = (_bytes(pkg, shared, reserved=way, **sizes) for way in (0, 1, 2))
    assert 0 < never and 0 < always and never != always
    assert chosen == (always if once else never)


@pytest.mark.parametrize('held', [torch.int8, torch.float8_e4m3fn], ids=str)
def test_arenas_of_8_bits_for_other_widths_are_refused(pkg, held):
    """When they are made, not at the first row."""
    module = torch.nn.Linear(2, 2).bfloat16()

    def arena(width, **kwargs):
        config = SimpleNamespace(num_key_value_heads=8, head_dim=width)
        return pkg.PagedArena(SimpleNamespace(parameters=module.parameters, layers=[None], config=config), pages=3, **kwargs)
    for width in (32, 96, 256):
        with pytest.raises(ValueError):
            arena(width, dtype=held)
        assert arena(width).packed.shape[-1] == width
    for width in (64, 128):
        assert arena(width, dtype=held).packed.shape[-1] == width
