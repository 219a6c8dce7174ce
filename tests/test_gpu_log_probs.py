"""pixhip_log_probs through the C ABI against the definition in 64 bits (numpy).

The bound.  The shifted logit x - m and log S are rounded to 2^-24 of their
magnitudes, S and the entropy's sum are fp32 sums of at most 2^18 terms, added up
in pieces: with the rounding of each exp (two of its steps, 2^-23), the
argument's own rounding |x - m| 2^-24 and at most 256 roundings of the sums, a
log probability is off by
  2^-23 (|x_i - m| + log S) + 2^-15
and the entropy by 2^-14 (1 + entropy).
"""
import ctypes

import numpy as np
import pytest

from gpu_helpers import Pinned, new_session
from pixelina_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


def call(sess, x, ids, top, vocab=None, want_entropy=True):
    rows, ld = x.shape
    vocab = vocab or ld
    xb = sess.to_device(x)
    ib = sess.to_device(ids) if ids is not None else None
    lp, en = sess.to_device(np.full(rows + 4, 7.0, np.float32)), sess.to_device(np.full(rows + 4, 7.0, np.float32))
    ti, tl = sess.to_device(np.full(rows * top + 4, -7, np.int32)), sess.to_device(np.full(rows * top + 4, 7.0, np.float32))
    _lib.check(sess.log_probs(xb.ptr, rows, vocab, ib.ptr if ib else None, lp.ptr if ib else None, en.ptr if want_entropy else None, top,
                              ti.ptr if top else None, tl.ptr if top else None, ld if ld != vocab else 0), "log_probs")
    out = [lp.download(np.float32, rows + 4), en.download(np.float32, rows + 4), ti.download(np.int32, rows * top + 4), tl.download(np.float32, rows * top + 4)]
    for a, n, fill in zip(out, (rows, rows, rows * top, rows * top), (7.0, 7.0, -7, 7.0)):
        assert (a[n:] == fill).all()  # nothing behind the last row
    if ib is None:
        assert (out[0] == 7.0).all()
    for b in (xb, ib, lp, en, ti, tl):
        if b:
            b.free()
    return out[0][:rows], out[1][:rows], out[2][:rows * top].reshape(rows, top), out[3][:rows * top].reshape(rows, top)


def exact(x):
    x = x.astype(np.float64)
    m = x.max(axis=1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        s = np.where(np.isneginf(x), -np.inf, x - np.where(np.isneginf(m), 0, m))
        total = np.exp(s).sum(axis=1, keepdims=True)
        logp = s - np.where(total > 0, np.log(total), 0)
        p = np.exp(logp)
        h = -np.where(p > 0, p * np.where(p > 0, logp, 0), 0).sum(axis=1)
    return logp, h, s, np.where(total > 0, np.log(total), 0)


def order_of(x, top):
    """The `top` first by value, NaN lowest, equal ones by the lower index (-0 equals 0)."""
    key = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    key = np.stack([np.lexsort((np.arange(x.shape[1]), -key[r], np.isnan(x[r]))) for r in range(x.shape[0])])
    return key[:, :top]


def check(sess, x, ids, top, vocab=None):
    vocab = vocab or x.shape[1]
    lp, en, ti, tl = call(sess, x, ids, top, vocab)
    v = x[:, :vocab]
    logp, h, s, norm = exact(v)
    bound = 2.0 ** -23 * (np.where(np.isfinite(s), np.abs(s), 0) + np.abs(norm)) + 2.0 ** -15
    r = np.arange(x.shape[0])

    def close(got, want, b):
        inf = ~np.isfinite(want)
        assert np.array_equal(got[inf], want[inf].astype(np.float32))
        if (~inf).any():
            print(f"  of the bound {(np.abs(got[~inf] - want[~inf]) / b[~inf]).max():.3f}", flush=True)
        assert (np.abs(got[~inf] - want[~inf]) <= b[~inf]).all()

    close(lp, logp[r, ids], bound[r, ids])
    close(en, h, 2.0 ** -14 * (1 + h))
    if top:
        want = order_of(v, top)
        assert np.array_equal(ti, want)
        close(tl, np.take_along_axis(logp, want, 1), np.take_along_axis(bound, want, 1))
    return lp, en, ti, tl


@pytest.mark.parametrize("rows,vocab,top,pad", [
    (1, 1, 1, 0), (1, 2, 2, 3), (3, 7, 7, 0), (1, 63, 5, 1), (2, 64, 64, 0), (5, 65, 3, 2), (1, 1000, 20, 0), (4, 1024, 64, 0), (7, 4097, 1, 5),
    (1, 8191, 40, 0), (1, 32000, 64, 0), (3, 32003, 20, 1), (1, 151936, 20, 0), (1, 151936, 0, 0), (2, 151935, 64, 3), (64, 5000, 10, 0), (300, 2049, 5, 7),
    (700, 33, 33, 0), (20, 40001, 7, 0),
])
def test_against_the_definition(sess, rows, vocab, top, pad):
    rng = np.random.default_rng(rows * 17 + vocab + top)
    x = (3 * rng.standard_normal((rows, vocab + pad))).astype(np.float32)
    x[:, vocab:] = np.nan  # not part of the rows
    if vocab > 50:
        x[:, rng.integers(0, vocab, vocab // 50)] = -np.inf
        x[np.arange(rows), rng.integers(0, vocab, rows)] = 25
    print(f"rows={rows} vocab={vocab} top={top} pad={pad}", flush=True)
    ids = rng.integers(0, vocab, rows).astype(np.int32)
    first = check(sess, x, ids, top, vocab)
    for a, b in zip(call(sess, x, ids, top, vocab), first):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32)), "repeats differ"


@pytest.mark.parametrize("vocab", [64, 1000, 5000, 151936])
def test_equal_logits(sess, vocab):
    """All equal; two values alternating; few distinct values; -0 and 0: alternatives by the lower index."""
    rng = np.random.default_rng(vocab)
    x = np.zeros((5, vocab), np.float32)
    x[1, 1::2] = 1
    x[2] = rng.integers(0, 3, vocab)
    x[3, ::3] = -0.0
    x[4] = np.where(np.arange(vocab) >= vocab - 10, 2.0, -5.0)
    check(sess, x, np.array([0, 1, 5, 3, vocab - 1], np.int32), 64)
    check(sess, x[:1], np.array([vocab - 1], np.int32), 3)


@pytest.mark.parametrize("vocab", [70, 3000, 100000])
def test_values_at_the_edges(sess, vocab):
    """Rows of -Inf alone, all but one, the type's largest and lowest values, logits far apart, subnormals."""
    x = np.full((6, vocab), -np.inf, np.float32)
    x[1, vocab - 1] = 3
    x[2] = -3.4028235e38
    x[3] = np.linspace(-3e38, 3e38, vocab, dtype=np.float32)
    x[4] = np.linspace(-200, 200, vocab, dtype=np.float32)
    x[5] = np.float32(1e-41) * np.arange(vocab)
    lp, en, ti, _ = check(sess, x, np.array([0, vocab - 1, 3, vocab - 1, 0, 7], np.int32), 20)
    assert np.isneginf(lp[0]) and en[0] == 0 and lp[1] == 0 and en[1] == 0 and np.array_equal(ti[0], np.arange(20))


@pytest.mark.parametrize("vocab", [70, 3000, 100000])
def test_not_a_number(sess, vocab):
    """NaN or +Inf in a row: NaN for it and for no other row; alternatives still in order, NaN lowest."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((4, vocab)).astype(np.float32)
    clean = call(sess, x, np.array([1, 2, 3, 4], np.int32), 30)
    bad = x.copy()
    bad[0, vocab // 2] = np.nan
    bad[2, 5] = np.inf
    bad[3, :] = np.nan
    lp, en, ti, tl = call(sess, bad, np.array([1, 2, 3, 4], np.int32), 30)
    for r in (0, 2, 3):
        assert np.isnan(lp[r]) and np.isnan(en[r])
    assert lp[1] == clean[0][1] and en[1] == clean[1][1] and np.array_equal(tl[1], clean[3][1])
    assert np.array_equal(ti, order_of(bad, 30))


def test_ids_outside_the_vocabulary(sess):
    x = np.random.default_rng(1).standard_normal((6, 999)).astype(np.float32)
    ids = np.array([-1, 0, 998, 999, 2 ** 31 - 1, -2 ** 31], np.int32)
    lp, _, _, _ = call(sess, x, ids, 0)
    logp = exact(x)[0]
    assert np.isnan(lp[[0, 3, 4, 5]]).all() and abs(lp[1] - logp[1, 0]) < 1e-4 and abs(lp[2] - logp[2, 998]) < 1e-4


def test_parts_wanted(sess):
    """Each output alone is what it is among the others; ids and logits from host memory; a misaligned row."""
    rng = np.random.default_rng(2)
    x, ids = rng.standard_normal((3, 20001)).astype(np.float32), np.array([5, 20000, 0], np.int32)
    lp, en, ti, tl = call(sess, x, ids, 9)
    assert np.array_equal(call(sess, x, ids, 0, want_entropy=False)[0], lp)
    assert np.array_equal(call(sess, x, None, 0)[1], en)
    only = call(sess, x, None, 9, want_entropy=False)
    assert np.array_equal(only[2], ti) and np.array_equal(only[3], tl)
    out = sess.alloc(64)
    _lib.check(sess.log_probs(x.ctypes.data, 3, 20001, ids.ctypes.data, out.ptr), "log_probs")
    assert np.array_equal(out.download(np.float32, 3), lp)
    hx, hi, ho = Pinned(sess, x), Pinned(sess, ids), Pinned(sess, np.zeros(3, np.float32))
    _lib.check(sess.log_probs(hx.p.value, 3, 20001, hi.p.value, ho.p.value), "log_probs")
    sess.synchronize()
    assert np.array_equal(ho.read(np.float32, (3,)), lp)
    for p in (hx, hi, ho):
        p.free()
    odd = sess.alloc(x.nbytes + 12)
    odd.upload(x, 12)
    _lib.check(sess.log_probs(odd.ptr + 12, 3, 20001, ids.ctypes.data, out.ptr), "log_probs")
    assert np.abs(out.download(np.float32, 3) - lp).max() <= 2.0 ** -15
    odd.free()
    out.free()


def test_refusals(sess):
    arg = _lib.ERR_ARGUMENT
    x, ids, out, many = sess.alloc(4 * 1000), sess.to_device(np.zeros(4, np.int32)), sess.alloc(1024), sess.alloc(4096)
    f = sess.log_probs
    assert f(None, 1, 1000, ids.ptr, out.ptr) == arg and f(x.ptr, 0, 1000, ids.ptr, out.ptr) == arg and f(x.ptr, 1, 0, ids.ptr, out.ptr) == arg
    assert f(x.ptr, 1, 1000, None, out.ptr) == arg and f(x.ptr, 1, 1000, ids.ptr, None) == arg and f(x.ptr, 1, 1000, None, None) == arg
    assert f(x.ptr, 1, 1000, ids.ptr, out.ptr, None, 65, many.ptr, many.ptr) == arg and f(x.ptr, 1, 8, ids.ptr, out.ptr, None, 9, many.ptr, many.ptr) == arg
    assert f(x.ptr, 1, 1000, ids.ptr, out.ptr, None, 3, None, many.ptr) == arg and f(x.ptr, 1, 1000, ids.ptr, out.ptr, None, 3, many.ptr, None) == arg
    assert f(x.ptr, 2, 500, ids.ptr, out.ptr, ld=499) == arg and f(x.ptr, 100, 500, ids.ptr, out.ptr) == arg
    assert f(x.ptr + 2, 1, 100, ids.ptr, out.ptr) == arg and f(x.ptr, 1, 1 << 31, ids.ptr, out.ptr) == arg
    host = np.zeros(4, np.float32)
    assert f(x.ptr, 1, 1000, ids.ptr, host.ctypes.data) == arg
    for b in (x, ids, out, many):
        b.free()


def test_captured_call(sess):
    """One long row (cut into pieces where that is not captured) replayed with larger eager calls between."""
    rng = np.random.default_rng(4)
    x, ids = rng.standard_normal((1, 151936)).astype(np.float32), np.array([77], np.int32)
    want = call(sess, x, ids, 20)
    s = new_session()
    lib, stream, graph, ready = s.lib, ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    try:
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, stream), "set_stream")
        xb, ib, lp, en, ti, tl = s.to_device(x), s.to_device(ids), s.alloc(4), s.alloc(4), s.alloc(80), s.alloc(80)
        s.synchronize()
        assert lib.hipStreamBeginCapture(stream, 1) == 0
        rc = s.log_probs(xb.ptr, 1, 151936, ib.ptr, lp.ptr, en.ptr, 20, ti.ptr, tl.ptr)
        assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0 and rc == _lib.OK
        assert lib.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)) == 0
        for i in range(4):
            print(f"replay {i}", flush=True)
            assert lib.hipGraphLaunch(ready, stream) == 0
            assert np.array_equal(ti.download(np.int32, 20), want[2][0])
            assert abs(lp.download(np.float32, 1)[0] - want[0][0]) <= 2.0 ** -14 and abs(en.download(np.float32, 1)[0] - want[1][0]) <= 2.0 ** -10
            big = rng.standard_normal((i + 2, 151936)).astype(np.float32)
            check(s, big, np.arange(i + 2, dtype=np.int32), 64)
        s.synchronize()
        assert lib.hipGraphExecDestroy(ready) == 0 and lib.hipGraphDestroy(graph) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, None), "set_stream")
        assert lib.hipStreamDestroy(stream) == 0
    finally:
        s.close()
