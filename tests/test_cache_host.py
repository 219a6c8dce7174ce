"""The key/value cache's and the log probabilities' entry points without a
device: refusals come back as codes and touch nothing; the blocks' code layouts
place every value once."""
import ctypes
import os
import subprocess

import pytest

from pixelina_amd import _lib, build

CSRC = os.path.join(os.path.dirname(_lib.LIBRARY), "csrc")


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIBRARY):
        build.build()
    return _lib.load()


def test_entry_points_without_a_session(lib):
    state, h = _lib.ERR_STATE, ctypes.c_void_p(77)
    assert lib.pixhip_cache_create(None, 1, 1, 64, 32, ctypes.byref(h)) == state
    assert lib.pixhip_cache_append(None, None, 0, None, None, 1, 0, None) == state
    assert lib.pixhip_cache_truncate(None, None, 0, 0) == state
    assert lib.pixhip_cache_copy(None, None, None) == state
    assert lib.pixhip_cache_evict(None, None, 0, 1, 1, None) == state
    assert lib.pixhip_cache_read(None, None, 0, 0, 1, None, None, None) == state
    assert lib.pixhip_cache_attention(None, None, 0, None, 1, 1, 0, 1, 0, 1.0, None) == state
    assert lib.pixhip_log_probs(None, None, 1, 10, 0, None, None, None, 0, None, None) == state
    assert b"session" in lib.pixhip_last_error()
    assert lib.pixhip_cache_length(None, 0, ctypes.byref(ctypes.c_size_t())) == _lib.ERR_ARGUMENT
    lib.pixhip_cache_destroy(None, None)  # no-op


def test_code_layouts_place_every_value_once(tmp_path):
    source, program = tmp_path / "layout.cpp", tmp_path / "layout"
    source.write_text("""
#include <cstdio>
#include <vector>
#include "pixhip_internal.h"
int main()
{
    for (int D : {64,128})
        for (int value = 0; value < 2; value++) {
            std::vector<int> seen(32 * D,0);
            for (int t = 0; t < 32; t++)
                for (int d = 0; d < D; d++) {
                    const int o = value? pixhip::cache_v_offset(t,d) : pixhip::cache_k_offset(t,d,D);
                    if (o < 0 || o >= 32 * D || seen[o]++) return 1;
                    if (!value && o != pixhip::cache_k_offset(t,d & ~15,D) + (d & 15)) return 2;  // 16 dims of a token are one piece
                    if (value && o != pixhip::cache_v_offset(0,d) + t) return 3;                  // a dim's tokens are one row
                }
        }
    std::puts("ok");
    return 0;
}
""")
    subprocess.run([build._hipcc(), "-x", "hip", "--cuda-host-only", "-std=c++17", "-I", CSRC, str(source), "-o", str(program)], check=True)
    assert subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout == "ok\n"
