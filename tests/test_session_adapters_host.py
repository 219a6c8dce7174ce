"""Session.adapters without a device: the ranges that reach pixhip_adapters, and the
ones that are refused before."""
import struct
import types

import pytest

from pixelina_amd import _lib
from pixelina_amd.session import Session


@pytest.fixture
def call():
    """Session.adapters of given ranges: the structures that the library is called with."""
    def adapters(ranges):
        seen = []
        lib = types.SimpleNamespace(pixhip_adapters=lambda handle, packed, count, *rest: seen.append((packed, count)))
        Session.adapters(types.SimpleNamespace(lib=lib, handle=None), ranges, None, 8, None, 4)
        packed, count = seen[0]
        return [(r.begin, r.end, r.adapter, r.scale) for r in (_lib.AdapterRange * count).from_buffer_copy(packed)]
    return adapters


def test_ranges(call):
    assert call([(0, 3, 77, 0.5), (3, 8, 78, -1)]) == [(0, 3, 77, 0.5), (3, 8, 78, -1.0)]
    assert call([(0, 3, None, 0.5), (3, 8, 78, -1)]) == [(0, 3, None, 0.5), (3, 8, 78, -1.0)]  # None: no adapter


@pytest.mark.parametrize("ranges", [[(0, 3, 77, None)], [(0, 3, None, None)], [(None, 3, 77, 1.0)], [(0, None, 77, 1.0)], [(0, 3, None, 1.0), (3, None, 77, 1.0)],
                                    [(0, 3, 77)], [(-1, 3, 77, 1.0)], [(0, 3, "a", 1.0)]])
def test_a_missing_bound_or_scale_is_not_taken_as_0(call, ranges):
    with pytest.raises((struct.error, ValueError)):
        call(ranges)


def test_ending_what_is_no_adapter():
    lib = _lib.load()
    for handle in (0x1000, 0x7f0000001000):
        lib.pixhip_adapter_destroy(None, handle)
