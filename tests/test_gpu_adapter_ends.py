"""An adapter's memory goes back to the session that made it, whoever ends it."""
import ctypes

import numpy as np
import pytest

from gpu_helpers import new_session
from pixelina_amd import _lib
from test_gpu_adapters import F32, Adapter, check, data, definition, run

pytestmark = pytest.mark.gpu


def free_bytes(lib):
    free, total = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
    return free.value


@pytest.mark.parametrize("how", ["own session", "another session", "no session"])
def test_memory_returns(how):
    rank, inner, rows = 256, 32768, 32  # 48 MB, from matrices of 32 MB
    down, up = np.ones((rank, inner), np.float32), np.ones((rows, rank), np.float32)
    owner, other = new_session(), new_session()
    by = {"own session": owner.handle, "another session": other.handle, "no session": None}[how]
    try:
        held = []
        for _ in range(6):
            h = owner.adapter(F32, down.ctypes.data, up.ctypes.data, rank, inner, rows)
            owner.synchronize()
            held.append(free_bytes(owner.lib))
            owner.lib.pixhip_adapter_destroy(by, h)
            owner.lib.pixhip_adapter_destroy(by, h)  # (again: nothing)
        assert held[0] - held[-1] < 48 << 20, held
        # the session goes on, with another adapter
        rng, x, base = data(1, 9, 40, 30)
        a = Adapter(owner, rng, F32, 5, 40, 30)
        check(run(owner, x, base, [(0, 9, a, 1.0)], 30), definition(x, base, [(0, 9, a, 1.0)]))
    finally:
        owner.close()
    # ended with its session
    other.adapter_destroy(a.h)
    other.lib.pixhip_adapter_destroy(None, a.h)
    other.close()


def test_destroyed_among_others():
    """Each of a session's adapters, first, last and between, ended through another session; the rest serve on."""
    s, other = new_session(), new_session()
    rng, x, base = data(2, 12, 33, 20)
    adapters = [Adapter(s, rng, _lib.F16, 3 + i, 33, 20) for i in range(5)]
    for gone in (2, 4, 0):
        other.adapter_destroy(adapters[gone].h)
        adapters[gone] = None
        left = [a for a in adapters if a]
        ranges = [(3 * i, 3 * i + 3, a, 1.0) for i, a in enumerate(left)]
        check(run(s, x, base, ranges, 20), definition(x, base, ranges))
    other.close()
    s.close()
