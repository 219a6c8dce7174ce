"""pixhip_log_probs against 64 bits, within a bound counted from its own roundings.

S = sum of e^(x - m) is an fp32 sum of positive terms: a lane adds 16 of its row's
logits per step (8192 logits of a workgroup, or of a piece), then 9 joins, then
those of the pieces.  R = 16 steps + 9 + pieces roundings of 2^-24 bound its relative
error; each term brings 2^-22 (the exponential and its argument's scaling) and the
rounding of its argument, together 2^-23 E|x - m| with E the mean over the
distribution.  So with u = 2^-24
  log p        u (2 |x_i - m| + 2 log S + R + 4 + 2 E|x - m|)
  entropy      u (2 log S + (R + 8) (1 + E|x - m|) + 2 E(x - m)^2)
where the entropy's own sum has the same roundings relative to E|x - m|.
"""
import ctypes

import numpy as np
import pytest

from gpu_helpers import new_session
from pixelina_amd import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


def bounds(x, ids, pieces):
    """(log p of ids, entropy, their bounds) in 64 bits."""
    x = x.astype(np.float64)
    d = x - x.max(axis=1, keepdims=True)
    total = np.exp(d).sum(axis=1)
    p = np.exp(d) / total[:, None]
    first, second = (p * np.abs(d)).sum(axis=1), (p * d * d).sum(axis=1)
    steps = -(-x.shape[1] // 8192)
    r = 16 * -(-steps // pieces) + 9 + pieces
    own = d[np.arange(len(x)), ids]
    lp, h = own - np.log(total), np.log(total) + first
    return lp, h, U * (2 * np.abs(own) + 2 * np.log(total) + r + 4 + 2 * first), U * (2 * np.log(total) + (r + 8) * (1 + first) + 2 * second)


def check(lp, en, x, ids, pieces):
    want_lp, want_en, lp_bound, en_bound = bounds(x, ids, pieces)
    print(f"  of the bounds {(np.abs(lp - want_lp) / lp_bound).max():.2f} {(np.abs(en - want_en) / en_bound).max():.2f}", flush=True)
    assert (np.abs(lp - want_lp) <= lp_bound).all() and (np.abs(en - want_en) <= en_bound).all()


@pytest.mark.parametrize("rows,vocab,top", [(3, 500, 0), (40, 1000, 5), (5, 8192, 64), (600, 3001, 1), (1, 151936, 20), (2, 40003, 0), (520, 20000, 3)])
@pytest.mark.parametrize("spread", [0.0, 0.01, 1.0, 4.0, 30.0])
def test_within_the_roundings(sess, rows, vocab, top, spread):
    """From all tokens alike to one that takes all."""
    rng = np.random.default_rng(rows + vocab)
    x = (spread * rng.standard_normal((rows, vocab)) - 3).astype(np.float32)
    ids = rng.integers(0, vocab, rows).astype(np.int32)
    ids[::2] = x[::2].argmax(axis=1)
    print(f"rows={rows} vocab={vocab} top={top} spread={spread}", flush=True)
    xb, ib, lb, eb, tb, tl = sess.to_device(x), sess.to_device(ids), sess.alloc(4 * rows), sess.alloc(4 * rows), sess.alloc(4 * rows * 64), sess.alloc(4 * rows * 64)
    _lib.check(sess.log_probs(xb.ptr, rows, vocab, ib.ptr, lb.ptr, eb.ptr, top, tb.ptr if top else None, tl.ptr if top else None), "log_probs")
    # as many pieces as a row has steps, while the launch stays at 512 workgroups
    check(lb.download(np.float32, rows), eb.download(np.float32, rows), x, ids, max(1, min(-(-vocab // 8192), 512 // rows)))
    for b in (xb, ib, lb, eb, tb, tl):
        b.free()


def test_captured_row(sess):
    """Captured, a row is one workgroup's: the same definition within the roundings of its longer sums."""
    rng = np.random.default_rng(6)
    x, ids = (3 * rng.standard_normal((1, 151936))).astype(np.float32), np.array([99], np.int32)
    s = new_session()
    lib, stream, graph, ready = s.lib, ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    try:
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, stream), "set_stream")
        xb, ib, lb, eb = s.to_device(x), s.to_device(ids), s.alloc(4), s.alloc(4)
        s.synchronize()
        assert lib.hipStreamBeginCapture(stream, 1) == 0
        code = s.log_probs(xb.ptr, 1, 151936, ib.ptr, lb.ptr, eb.ptr)
        assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0 and code == _lib.OK
        assert lib.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)) == 0
        for i in range(3):
            x = (3 * rng.standard_normal((1, 151936))).astype(np.float32)
            xb.upload(x)
            assert lib.hipGraphLaunch(ready, stream) == 0
            check(lb.download(np.float32, 1), eb.download(np.float32, 1), x, ids, 1)
        s.synchronize()
        assert lib.hipGraphExecDestroy(ready) == 0 and lib.hipGraphDestroy(graph) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, None), "set_stream")
        assert lib.hipStreamDestroy(stream) == 0
    finally:
        s.close()
