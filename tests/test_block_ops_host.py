"""The entry points of a block's residual norm, head rotation and adapters without a
device: refusals come back as codes and touch nothing; the wide form of a head's
rotation places every value of a head once."""
import ctypes
import os
import struct
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
    assert lib.pixhip_residual_norm_quantize(None, 0, None, None, 1, 4, None, None, None, None) == state
    assert lib.pixhip_split_heads(None, None, None, None, 1, 0, 1, 1, 64, None, None, None, None) == state
    assert lib.pixhip_cache_append_rotated(None, None, 0, None, None, None, 1, 0, 1, None, None, None) == state
    assert lib.pixhip_adapter_create(None, 0, None, None, 1, 4, 4, ctypes.byref(h)) == state
    assert lib.pixhip_adapters(None, None, 0, None, 1, 0, None, None, 4, 0) == state
    assert b"session" in lib.pixhip_last_error()
    assert lib.pixhip_model_adapter(None, None, b"a", b"b", ctypes.byref(h)) == _lib.ERR_ARGUMENT
    assert lib.pixhip_adapter_shape(None, None, None, None, None) == _lib.ERR_ARGUMENT
    lib.pixhip_adapter_destroy(None, None)  # no-op


def test_workspace_without_a_session(lib):
    assert lib.pixhip_adapters_reserve(None, 1, 1, 16) == _lib.ERR_STATE


def test_structures_have_the_header_s_layout(tmp_path):
    source, program = tmp_path / "layout.c", tmp_path / "layout"
    structures = {"pixhip_residual_norm": _lib.ResidualNorm, "pixhip_rotation": _lib.Rotation, "pixhip_adapter_range": _lib.AdapterRange}
    lines = [f'printf("%zu {n} {f} %zu\\n", sizeof({n}), offsetof({n}, {f}));' for n, s in structures.items() for f, _ in s._fields_]
    source.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"pixhip.h\"\nint main(void)\n{\n" + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(build.ROOT, "include"), str(source), "-o", str(program)], check=True)
    for line in subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.splitlines():
        size, name, field, offset = line.split()
        s = structures[name]
        assert ctypes.sizeof(s) == int(size) and getattr(s, field).offset == int(offset), line
    # as Session.adapters packs a range
    r = _lib.AdapterRange(3, 5, 77, 0.5)
    assert struct.pack("QQQf4x", 3, 5, 77, 0.5) == bytes(r)


def test_wide_heads_place_every_value_once():
    """turn_quads of csrc/heads_device.h, restated: for every head and rotary size that the wide forms take."""
    for dim in range(4, 129, 4):
        for rotary in range(0, dim + 1, 8):
            for adjacent in (False, True):
                seen = []
                for lane in range(16):
                    if adjacent:
                        quads = (8 * lane, 8 * lane + 4)
                    elif lane < rotary // 8:
                        quads = (4 * lane, rotary // 2 + 4 * lane)
                    else:
                        quads = (rotary + 8 * (lane - rotary // 8),) * 2
                        quads = (quads[0], quads[0] + 4)
                    seen += [q for q in quads if q < dim]
                assert sorted(seen) == list(range(0, dim, 4)), (dim, rotary, adjacent)
