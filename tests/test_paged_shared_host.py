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
