"""A convolution captured with its image in pinned memory: replays read the image where
it is, as it is then, and leave the buffers that were made after the capture alone."""
import ctypes

import numpy as np
import pytest

from gpu_helpers import TOL, Pinned, new_session, row_rel_error
from oracle_lib import conv2d, oracle
from pixelina_amd import _lib

pytestmark = pytest.mark.gpu

F32 = 0


@pytest.mark.parametrize("wd,ht,cin,cout", [(17, 9, 16, 24), (24, 20, 256, 64)])
def test_captured_convolution(wd, ht, cin, cout):
    rng = np.random.default_rng(cin)
    w = (rng.standard_normal((cout, cin * 9)) / np.sqrt(cin * 9)).astype(np.float32)
    raw = w.view(np.uint8).reshape(-1)
    s = new_session()
    lib, stream, graph, ready = s.lib, ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    try:
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, stream), "set_stream")
        x = rng.standard_normal((wd * ht, cin)).astype(np.float32)
        h, hx, yb = s.conv_weight("w", raw, F32, 3, 3, cin, cout), Pinned(s, x), s.alloc(wd * ht * cout * 4)
        _lib.check(s.conv2d(h, hx.p.value, wd, ht, yb.ptr), "conv2d")
        s.synchronize()
        assert lib.hipStreamBeginCapture(stream, 1) == 0
        code = s.conv2d(h, hx.p.value, wd, ht, yb.ptr)
        assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0 and code == _lib.OK
        assert lib.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)) == 0
        mine = [s.to_device(np.full(x.size, 9.0, np.float32)) for _ in range(2)]
        for i in range(3):
            print(f"replay {i}", flush=True)
            x = rng.standard_normal((wd * ht, cin)).astype(np.float32)
            ctypes.memmove(hx.p, x.ctypes.data, x.nbytes)
            assert lib.hipGraphLaunch(ready, stream) == 0
            y = yb.download(np.float32, wd * ht * cout).reshape(-1, cout)
            assert row_rel_error(y, conv2d(oracle(), x, wd, ht, w, 3, 3)).max() <= TOL
            assert all((b.download(np.float32, x.size) == 9).all() for b in mine)
        s.synchronize()
        assert lib.hipGraphExecDestroy(ready) == 0 and lib.hipGraphDestroy(graph) == 0
        hx.free()
        _lib.check(lib.pixhip_session_set_stream(s.handle, None), "set_stream")
        assert lib.hipStreamDestroy(stream) == 0
    finally:
        s.close()
