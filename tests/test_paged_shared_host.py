"""Shared pages of the paged cache without a GPU: what launches of any length have for their work."""
import ctypes
import subprocess
from pathlib import Path

import pytest

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
