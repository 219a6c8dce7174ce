"""Low-rank adapters (pixhip_adapter_*, pixhip_adapters) through the C ABI against
base + scale * up (down x) in 64 bits.

The bound.  With u = 2^-23 (a step of fp32, whichever way a matrix instruction
rounds): a sum of K products, each exact to u, is off by at most (K + 8) u sum|terms|,
the scaled part t by that and a step, and an output by
  |scale| sum_j |U_j| ((K + 9) u T_j) + (rank + 8) u |scale| sum_j |U_j t_j| + u |y|
with T_j = sum_k |D_jk x_k|.  Sums of a few exact products are checked bit for bit.
"""
import ctypes

import numpy as np
import pytest

from gpu_helpers import Pinned, new_session
from pixelina_amd import _lib

pytestmark = pytest.mark.gpu

F32, F16, BF16 = _lib.F32, _lib.F16, _lib.BF16
U = 2.0 ** -23
GUARD = 32


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


def stored(a, wtype):
    """(raw array, values) of a matrix in the given type."""
    a = np.ascontiguousarray(a, np.float32)
    if wtype == F32:
        return a, a
    if wtype == F16:
        h = a.astype(np.float16)
        return h, h.astype(np.float32)
    b = a.view(np.uint32)
    b = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return b, (b.astype(np.uint32) << 16).view(np.float32)


class Adapter:
    def __init__(self, sess, rng, wtype, rank, inner, rows, down=None, up=None):
        raw_d, self.down = stored(rng.standard_normal((rank, inner)) / np.sqrt(inner) if down is None else down, wtype)
        raw_u, self.up = stored(rng.standard_normal((rows, rank)) * 0.3 if up is None else up, wtype)
        self.sess, self.h = sess, sess.adapter(wtype, raw_d.ctypes.data, raw_u.ctypes.data, rank, inner, rows)

    def free(self):
        self.sess.adapter_destroy(self.h)


def definition(x, base, ranges):
    """(y, bound) in 64 bits; ranges [(begin, end, Adapter or None, scale)]."""
    x, y = x.astype(np.float64), base.astype(np.float64)
    bound = np.zeros_like(y)
    for b, e, a, scale in ranges:
        if a is None:
            continue
        scale = np.float64(np.float32(scale))
        d, up = a.down.astype(np.float64), a.up.astype(np.float64)
        t, big = x[b:e] @ d.T, np.abs(x[b:e]) @ np.abs(d).T
        inner, rank = d.shape[1], d.shape[0]
        y[b:e] += scale * (t @ up.T)
        bound[b:e] += abs(scale) * (((inner + 9) * U * big + (rank + 8) * U * np.abs(t)) @ np.abs(up).T) + 2 * U * np.abs(y[b:e])
    return y, bound + 2 * U * np.abs(y) + 1e-37


def place(sess, a, ld=None, shift=0):
    """Rows of `a`, `ld` values apart, NaN between and behind them: (buffer, address)."""
    ld = ld or a.shape[1]
    flat = np.full((a.shape[0], ld), np.nan, np.float32)
    flat[:, :a.shape[1]] = a
    b = sess.alloc(flat.nbytes + 4 * GUARD + 32)
    b.upload(np.concatenate([flat.reshape(-1), np.full(GUARD, np.nan, np.float32)]), shift)
    return b, b.ptr + shift


def fetch(b, rows, cols, ld=None, shift=0):
    """The rows; what lies between and behind them has to be what place put there."""
    ld = ld or cols
    a = b.download(np.float32, rows * ld + GUARD, shift)
    assert np.isnan(a[rows * ld:]).all()
    a = a[:rows * ld].reshape(rows, ld)
    assert np.isnan(a[:, cols:]).all()
    return a[:, :cols]


def run(sess, x, base, ranges, rows, mode="apart", ldx=0, ldy=0, shift=0):
    cols = x.shape[0]
    xb, xp = place(sess, x, ldx, shift)
    bb, bp = place(sess, base, ldy, shift)
    yb, yp = (bb, bp) if mode == "in place" else place(sess, np.full((cols, rows), 7.0, np.float32), ldy, shift)
    calls = [(b, e, a.h if a else None, s) for b, e, a, s in ranges]
    _lib.check(sess.adapters(calls, xp, cols, yp, rows, None if mode == "zero" else bp, ldx, ldy), "adapters")
    y = fetch(yb, cols, rows, ldy, shift)
    for b in {xb, bb, yb}:
        b.free()
    return y


def check(y, want):
    assert (np.abs(y - want[0]) <= want[1]).all()


def data(seed, cols, inner, rows):
    rng = np.random.default_rng(seed)
    return rng, rng.standard_normal((cols, inner)).astype(np.float32) * np.exp(rng.standard_normal(inner)).astype(np.float32), \
        rng.standard_normal((cols, rows)).astype(np.float32)


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("rank,inner,rows,cols", [
    (1, 1, 1, 1), (3, 5, 7, 2), (4, 33, 31, 16), (15, 64, 32, 17), (16, 100, 129, 1), (17, 257, 64, 5), (32, 96, 1000, 33), (33, 300, 65, 40), (48, 128, 40, 3),
    (64, 4096, 96, 7), (100, 36, 260, 18), (255, 70, 50, 4), (256, 256, 512, 2), (8, 1500, 3001, 300), (24, 512, 1024, 700)])
def test_one_adapter(sess, wtype, rank, inner, rows, cols):
    rng, x, base = data(rank + inner, cols, inner, rows)
    a = Adapter(sess, rng, wtype, rank, inner, rows)
    ranges = [(0, cols, a, 0.75)]
    want = definition(x, base, ranges)
    first = run(sess, x, base, ranges, rows)
    check(first, want)
    for kw in ({"mode": "in place"}, {"shift": 4}, {"ldx": inner + 3, "ldy": rows + 5}, {"ldx": inner + 4 - inner % 4, "ldy": rows + 8 - rows % 4, "mode": "in place"}):
        assert np.array_equal(run(sess, x, base, ranges, rows, **kw).view(np.uint32), first.view(np.uint32))
    check(run(sess, x, base, ranges, rows, mode="zero"), definition(x, np.zeros_like(base), ranges))
    a.free()


@pytest.mark.parametrize("wtype,rank,inner,rows,cols", [(BF16, 20, 200, 7400, 4500), (F32, 130, 333, 1001, 4200), (F16, 70, 96, 7300, 4700)])
def test_many_rows(sess, wtype, rank, inner, rows, cols):
    """Several requests of unequal length, whose tiles the forms for many rows take in twos and fours."""
    rng, x, base = data(rank, cols, inner, rows)
    a, b = Adapter(sess, rng, wtype, rank, inner, rows), Adapter(sess, rng, wtype, 5, inner, rows)
    ranges = [(0, 37, b, 1.0), (37, 2100, a, 0.5), (2111, cols - 3, a, -1.0), (cols - 3, cols, b, 2.0)]
    want = definition(x, base, ranges)
    for mode in ("apart", "in place"):
        check(run(sess, x, base, ranges, rows, mode), want)
    a.free()
    b.free()


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
def test_exact_products(sess, wtype):
    """Selections: every value of x comes through whole, all 24 bits of it, times the weight's."""
    inner, rank, rows, cols = 70, 40, 90, 20
    rng, x, _ = data(7, cols, inner, rows)
    x *= np.exp2(rng.integers(-40, 40, x.shape)).astype(np.float32)
    pick, place_at = rng.permutation(inner)[:rank], rng.permutation(rows)[:rank]
    down, up = np.zeros((rank, inner), np.float32), np.zeros((rows, rank), np.float32)
    down[np.arange(rank), pick], up[place_at, np.arange(rank)] = 1, 1
    a = Adapter(sess, rng, wtype, rank, inner, rows, down, up)
    want = np.zeros((cols, rows), np.float32)
    want[:, place_at] = x[:, pick]
    assert np.array_equal(run(sess, x, want * 0, [(0, cols, a, 1.0)], rows, mode="zero"), want)
    a.free()
    # a weight of all the bits its type holds: within the 2^-23 that the planes left out leave
    down[np.arange(rank), pick] = rng.uniform(0.5, 2, rank)
    a = Adapter(sess, rng, wtype, rank, inner, rows, down, up)
    want = np.zeros((cols, rows))
    want[:, place_at] = x[:, pick].astype(np.float64) * a.down[np.arange(rank), pick]
    assert (np.abs(run(sess, x, base=np.zeros((cols, rows), np.float32), ranges=[(0, cols, a, 1.0)], rows=rows) - want) <= 2.5 * U * np.abs(want)).all()
    a.free()


@pytest.mark.parametrize("cols", [5, 64, 512, 513, 1500])
def test_many_requests(sess, cols):
    """Adapters of all types and several ranks, shared, out of order, with gaps, empty ranges and rows of none."""
    inner, rows = 260, 333
    rng, x, base = data(cols, cols, inner, rows)
    adapters = [Adapter(sess, rng, t, r, inner, rows) for t, r in ((F32, 5), (F16, 16), (BF16, 64), (BF16, 8), (F16, 70), (F32, 33))]
    cuts = np.sort(rng.choice(np.arange(1, cols), min(cols - 1, 40), replace=False))
    cuts = [0, *(int(c) for c in cuts), cols]
    ranges = []
    for i, (b, e) in enumerate(zip(cuts, cuts[1:])):
        if i % 7 == 3:
            continue  # of no range
        ranges.append((b, e, None if i % 7 == 5 else adapters[i % 6], [1.0, -0.5, 2.0][i % 3]))
    ranges += [(0, 0, adapters[0], 1.0), (cols, cols, None, 1.0)]
    want = definition(x, base, ranges)
    for order in (ranges, ranges[::-1]):
        for mode in ("apart", "in place"):
            y = run(sess, x, base, order, rows, mode)
            check(y, want)
            for b, e, a, _ in ranges:
                assert a or np.array_equal(y[b:e].view(np.uint32), base[b:e].view(np.uint32))
    # a row's result does not depend on the others of the call
    b, e, a, s = next(r for r in ranges if r[2])
    alone = run(sess, x[b:e], base[b:e], [(0, e - b, a, s)], rows)
    assert np.array_equal(alone.view(np.uint32), run(sess, x, base, ranges, rows)[b:e].view(np.uint32))
    for a in adapters:
        a.free()


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("rank,inner,rows,cols", [(16, 640, 96, 1), (9, 801, 70, 3), (32, 1021, 333, 18), (16, 1024, 1000, 64), (5, 2048, 31, 2), (64, 512, 40, 5)])
def test_single_rows(sess, wtype, rank, inner, rows, cols):
    """A request per row, of inner sizes about those that one launch takes."""
    rng, x, base = data(rank + inner, cols, inner, rows)
    adapters = [Adapter(sess, rng, wtype, max(1, rank - i), inner, rows) for i in range(3)]
    ranges = [(c, c + 1, adapters[c % 3], 1.0 + c) for c in range(cols)]
    want = definition(x, base, ranges)
    first = run(sess, x, base, ranges, rows)
    check(first, want)
    for kw in ({"mode": "in place"}, {"shift": 4}, {"ldx": inner + 3, "ldy": rows + 5}):
        assert np.array_equal(run(sess, x, base, ranges, rows, **kw).view(np.uint32), first.view(np.uint32))
    for a in adapters:
        a.free()


def test_more_adapters_than_a_launch_takes(sess):
    inner, rows, cols = 64, 40, 150
    rng, x, base = data(3, cols, inner, rows)
    adapters = [Adapter(sess, rng, (F32, F16, BF16)[i % 3], 1 + i % 20, inner, rows) for i in range(cols)]
    ranges = [(i, i + 1, adapters[(i * 37) % cols], 1.0 + i) for i in range(cols)]
    check(run(sess, x, base, ranges, rows), definition(x, base, ranges))
    for a in adapters:
        a.free()


def test_adapters_add_up(sess):
    inner, rows, cols = 128, 200, 45
    rng, x, base = data(9, cols, inner, rows)
    a, b, c = (Adapter(sess, rng, t, 12, inner, rows) for t in (BF16, F32, F16))
    ranges = [(0, cols, a, 0.5), (10, 30, b, 1.0), (20, cols, c, -2.0), (0, 15, a, 1.5)]
    for mode in ("apart", "in place"):
        check(run(sess, x, base, ranges, rows, mode), definition(x, base, ranges))
    for z in (a, b, c):
        z.free()


def test_no_ranges(sess):
    _, x, base = data(1, 9, 8, 21)
    assert np.array_equal(run(sess, x, base, [], 21), base) and np.array_equal(run(sess, x, base, [], 21, "in place"), base)
    assert (run(sess, x, base, [(0, 9, None, 1.0)], 21, "zero") == 0).all()


def test_rows_that_are_not_finite_stay_alone(sess):
    inner, rows, cols = 100, 70, 20
    rng, x, base = data(4, cols, inner, rows)
    for wtype in (F32, F16, BF16):
        a = Adapter(sess, rng, wtype, 20, inner, rows)
        bad = x.copy()
        bad[3, 50], bad[17, 99] = np.nan, -np.inf
        y, want = run(sess, bad, base, [(0, cols, a, 1.0)], rows), definition(x, base, [(0, cols, a, 1.0)])
        good = [r for r in range(cols) if r not in (3, 17)]
        assert np.isnan(y[[3, 17]]).all() and (np.abs(y - want[0]) <= want[1])[good].all()
        a.free()
    # base passes as it is
    a, odd = Adapter(sess, rng, F32, 4, inner, rows), base.copy()
    odd[1, 2], odd[2, 3], odd[5, 0] = np.nan, np.inf, -0.0
    y = run(sess, x, odd, [(0, 5, a, 1.0)], rows)
    assert np.isnan(y[1, 2]) and y[2, 3] == np.inf and np.isfinite(np.delete(y[:5].reshape(-1), [72, 143])).all()
    assert np.signbit(y[5, 0]) and y[5, 0] == 0
    y = run(sess, x, base, [(0, 5, a, np.nan), (5, cols, a, 0.0), (2, 4, a, np.nan)], rows)
    assert np.isnan(y[:5]).all() and np.array_equal(y[5:], base[5:])
    a.free()


def test_host_operands_and_device_matrices(sess):
    inner, rows, cols, rank = 96, 64, 10, 8
    rng, x, base = data(12, cols, inner, rows)
    raw_d, raw_u = (stored(rng.standard_normal(s), F16)[0] for s in ((rank, inner), (rows, rank)))
    db, ub = sess.to_device(raw_d), sess.to_device(raw_u)
    pd, pu = Pinned(sess, raw_d), Pinned(sess, raw_u)
    got = []
    px, pb, py = Pinned(sess, x), Pinned(sess, base), Pinned(sess, base)
    yb = sess.alloc(base.nbytes)
    for d, u in ((raw_d.ctypes.data, raw_u.ctypes.data), (db.ptr, ub.ptr), (pd.p.value, pu.p.value)):
        h = sess.adapter(F16, d, u, rank, inner, rows)
        for xp, bp in ((x.ctypes.data, base.ctypes.data), (px.p.value, pb.p.value)):
            _lib.check(sess.adapters([(0, cols, h, 1.0)], xp, cols, yb.ptr, rows, bp), "adapters")
            got.append(yb.download(np.uint32, base.size))
        _lib.check(sess.adapters([(0, cols, h, 1.0)], px.p.value, cols, py.p.value, rows, pb.p.value), "pinned output")
        sess.synchronize()
        got.append(py.read(np.uint32, base.size))
        sess.adapter_destroy(h)
    assert all(np.array_equal(g, got[0]) for g in got)
    for b in (db, ub, pd, pu, px, pb, py, yb):
        b.free()


def test_sizes_beyond_a_buffer(sess):
    rng = np.random.default_rng(3)
    a = Adapter(sess, rng, F32, 2, 8, 8)
    b = sess.alloc(4096)
    w = np.ones(64, np.float32)
    for inner, rows in ((1 << 24, 8), (8, 1 << 24)):
        h = ctypes.c_void_p()
        assert sess.lib.pixhip_adapter_create(sess.handle, F32, w.ctypes.data, w.ctypes.data, 2, inner, rows, ctypes.byref(h)) == _lib.ERR_ARGUMENT
    for ldx, ldy in ((1 << 24, 0), (0, 1 << 24), (1 << 62, 0), (0, 1 << 62)):
        assert sess.adapters([(0, 2, a.h, 1.0)], b.ptr, 2, b.ptr + 1024, 8, None, ldx, ldy) == _lib.ERR_ARGUMENT
    b.free()
    a.free()


def test_from_a_model_file(sess, tmp_path):
    import model_files
    inner, rows, cols, rank = 48, 36, 6, 4
    rng, x, base = data(2, cols, inner, rows)
    down, up = stored(rng.standard_normal((rank, inner)), BF16), stored(rng.standard_normal((rows, rank)), BF16)
    path = tmp_path / "adapter.safetensors"
    path.write_bytes(model_files.safetensors([("a.down", "BF16", down[0].shape, down[0].tobytes()), ("a.up", "BF16", up[0].shape, up[0].tobytes()),
                                              ("a.odd", "F32", (rows, rank), up[1].tobytes())]))
    model, h = ctypes.c_void_p(), ctypes.c_void_p()
    _lib.check(sess.lib.pixhip_model_open(str(path).encode(), 1, ctypes.byref(model)), "open")
    call = sess.lib.pixhip_model_adapter
    assert call(sess.handle, model, b"a.up", b"a.down", ctypes.byref(h)) == _lib.ERR_ARGUMENT
    assert call(sess.handle, model, b"a.down", b"a.odd", ctypes.byref(h)) == _lib.ERR_ARGUMENT
    assert call(sess.handle, model, b"a.down", b"none", ctypes.byref(h)) == _lib.ERR_ARGUMENT
    _lib.check(call(sess.handle, model, b"a.down", b"a.up", ctypes.byref(h)), "adapter")
    sess.lib.pixhip_model_close(model)
    t, sizes = ctypes.c_uint32(), [ctypes.c_size_t() for _ in range(3)]
    _lib.check(sess.lib.pixhip_adapter_shape(h, ctypes.byref(t), *(ctypes.byref(z) for z in sizes)), "shape")
    assert (t.value, *(z.value for z in sizes)) == (BF16, rank, inner, rows)

    class Held:
        pass
    a = Held()
    a.h, a.down, a.up = h.value, down[1], up[1]
    check(run(sess, x, base, [(0, cols, a, 1.0)], rows), definition(x, base, [(0, cols, a, 1.0)]))
    sess.adapter_destroy(h.value)


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("power", [-118, -126, -140, 100])
def test_values_at_the_ends_of_the_range(sess, wtype, power):
    """Planes, products and sums below fp32's least normal value may be lost, 2^-126 of each:
    K values of x, 6 K products and K + 1 sums before `up`, the same of rank values behind it."""
    inner, rank, rows, cols = 96, 20, 70, 19
    rng, x, _ = data(8, cols, inner, rows)
    x = np.ldexp(x, power).astype(np.float32)
    base = np.zeros((cols, rows), np.float32)
    a = Adapter(sess, rng, wtype, rank, inner, rows)
    want, bound = definition(x, base, [(0, cols, a, 1.0)])
    lost = (np.abs(a.down).sum(axis=1).astype(np.float64) + 8 * inner + 1) * 2.0 ** -126
    bound = bound - 1e-37 + np.abs(a.up).astype(np.float64) @ lost + (np.abs(a.up).sum(axis=1).astype(np.float64) + 8 * rank + 1) * 2.0 ** -126
    check(run(sess, x, base, [(0, cols, a, 1.0)], rows, "zero"), (want, bound))
    a.free()


def test_two_sessions(sess):
    """Calls of two sessions, queued in turn on their streams, each with its own workspace."""
    inner, rows, cols = 2100, 700, 50
    rng, x, base = data(12, cols, inner, rows)
    other = new_session()
    try:
        calls = []
        for s in (sess, other):
            a = Adapter(s, rng, BF16, 24, inner, rows)
            calls.append((s, a, s.to_device(x), s.to_device(base), [s.alloc(base.nbytes) for _ in range(6)]))
        for i in range(6):
            for s, a, xb, bb, ys in calls:
                _lib.check(s.adapters([(0, cols, a.h, 1.0 + i)], xb.ptr, cols, ys[i].ptr, rows, bb.ptr), "adapters")
        for s, a, xb, bb, ys in calls:
            for i in range(6):
                check(ys[i].download(np.float32, base.size).reshape(base.shape), definition(x, base, [(0, cols, a, 1.0 + i)]))
            for b in (xb, bb, *ys):
                b.free()
            a.free()
    finally:
        other.close()


def test_captured(sess):
    """Two graphs of one adapter, replayed in turn with eager calls between them."""
    inner, rows, cols = 300, 520, 37
    rng, x, base = data(6, cols, inner, rows)
    s = new_session()
    lib, stream = s.lib, ctypes.c_void_p()
    try:
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, stream), "set_stream")
        adapters = [Adapter(s, rng, t, r, inner, rows) for t, r in ((BF16, 16), (F16, 40))]
        xb, bb = s.to_device(x), s.to_device(base)
        graphs = []
        for ranges in ([(0, 20, adapters[0].h, 1.0), (20, cols, adapters[1].h, 0.5)], [(i, i + 1, adapters[i % 2].h, 2.0) for i in range(cols)]):
            yb, graph, ready = s.alloc(base.nbytes), ctypes.c_void_p(), ctypes.c_void_p()
            _lib.check(s.adapters(ranges, xb.ptr, cols, yb.ptr, rows, bb.ptr), "eager")
            eager = yb.download(np.float32, base.size)
            assert lib.hipStreamBeginCapture(stream, 1) == 0
            code = s.adapters(ranges, xb.ptr, cols, yb.ptr, rows, bb.ptr)
            h = ctypes.c_void_p()
            refused = lib.pixhip_adapter_create(s.handle, F32, x.ctypes.data, x.ctypes.data, 1, 4, 4, ctypes.byref(h))
            assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0 and code == _lib.OK and refused == _lib.ERR_STATE
            assert lib.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)) == 0
            graphs.append((ranges, yb, graph, ready, eager))
        for i in range(3):
            for ranges, yb, _, ready, eager in graphs:
                yb.upload(np.full(base.size, float(i), np.float32))
                assert lib.hipGraphLaunch(ready, stream) == 0
                got = yb.download(np.float32, base.size).reshape(base.shape)
                own = [(b, e, next(a for a in adapters if a.h == h), sc) for b, e, h, sc in ranges]
                check(got, definition(x, base, own))
                check(eager.reshape(base.shape), definition(x, base, own))
                _lib.check(s.adapters(graphs[0][0], xb.ptr, cols, yb.ptr, rows, bb.ptr), "other work")
        s.synchronize()
        for _, _, graph, ready, _ in graphs:
            assert lib.hipGraphExecDestroy(ready) == 0 and lib.hipGraphDestroy(graph) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, None), "set_stream")
        assert lib.hipStreamDestroy(stream) == 0
    finally:
        s.close()


def test_captured_with_a_workspace(sess):
    """Graphs whose calls have a workspace of their own give what calls outside of them give, bit for bit, with
    calls outside between their replays and the workspace made larger after their capture."""
    s = new_session()
    lib, stream = s.lib, ctypes.c_void_p()
    try:
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, stream), "set_stream")
        graphs = []
        for t, rank, inner, rows, cols in ((F16, 64, 3840, 1030, 1), (F32, 100, 2049, 300, 20), (BF16, 16, 1500, 520, 600)):
            rng, x, base = data(rank, cols, inner, rows)
            adapters = [Adapter(s, rng, t, r, inner, rows) for r in (rank, 5)]
            ranges = [(0, (cols + 1) // 2, adapters[0].h, 0.5), (cols - cols // 3, cols, adapters[1].h, 2.0)]
            want = definition(x, base, [(b, e, next(a for a in adapters if a.h == h), sc) for b, e, h, sc in ranges])
            xb, bb, yb, graph, ready = s.to_device(x), s.to_device(base), s.alloc(base.nbytes), ctypes.c_void_p(), ctypes.c_void_p()
            _lib.check(s.adapters(ranges, xb.ptr, cols, yb.ptr, rows, bb.ptr), "eager")
            eager = yb.download(np.float32, base.size)
            _lib.check(s.adapters_reserve(cols, len(ranges), rank), "reserve")
            assert lib.hipStreamBeginCapture(stream, 1) == 0
            code, refused = s.adapters(ranges, xb.ptr, cols, yb.ptr, rows, bb.ptr), s.adapters_reserve(1, 1, 1)
            assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0 and code == _lib.OK and refused == _lib.ERR_STATE
            assert lib.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)) == 0
            graphs.append((ranges, xb, bb, yb, graph, ready, eager, want, cols, rows))
        for i in range(3):
            for ranges, xb, bb, yb, _, ready, eager, want, cols, rows in graphs:
                yb.upload(np.full(eager.size, float(i), np.float32))
                assert lib.hipGraphLaunch(ready, stream) == 0
                got = yb.download(np.float32, eager.size)
                assert np.array_equal(got.view(np.uint32), eager.view(np.uint32))
                check(got.reshape(want[0].shape), want)
                _lib.check(s.adapters(ranges, xb.ptr, cols, yb.ptr, rows, bb.ptr), "other work")
        for code in (s.adapters_reserve(0, 1, 16), s.adapters_reserve(1, 0, 16), s.adapters_reserve(1, 1, 0), s.adapters_reserve(1, 1, 257)):
            assert code == _lib.ERR_ARGUMENT
        s.synchronize()
        for *_, graph, ready, _, _, _, _ in graphs:
            assert lib.hipGraphExecDestroy(ready) == 0 and lib.hipGraphDestroy(graph) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, None), "set_stream")
        assert lib.hipStreamDestroy(stream) == 0
    finally:
        s.close()


def test_refusals(sess):
    inner, rows, cols = 16, 24, 6
    rng, x, base = data(5, cols, inner, rows)
    arg, h, lib = _lib.ERR_ARGUMENT, ctypes.c_void_p(77), sess.lib
    m = np.zeros(4096, np.float32)

    def create(wtype=F32, down=m.ctypes.data, up=m.ctypes.data, rank=4, inner=inner, rows=rows):
        return lib.pixhip_adapter_create(sess.handle, wtype, down, up, rank, inner, rows, ctypes.byref(h))
    assert create(8) == _lib.ERR_UNSUPPORTED and create(rank=257) == _lib.ERR_UNSUPPORTED and not h.value
    for bad in ({"down": None}, {"up": None}, {"rank": 0}, {"inner": 0}, {"rows": 0}, {"inner": 1 << 31}, {"rows": 1 << 62}, {"down": m.ctypes.data + 2}):
        assert create(**bad) == arg, bad
    assert lib.pixhip_adapter_create(sess.handle, F32, m.ctypes.data, m.ctypes.data, 4, inner, rows, None) == arg
    dev = sess.to_device(m[:8])
    assert create(down=dev.ptr, rank=40) == arg  # past the allocation (of 256 bytes, whole)
    a, other = Adapter(sess, rng, F32, 3, inner, rows), Adapter(sess, rng, F32, 3, inner + 1, rows)
    foreign_session = new_session()
    foreign = Adapter(foreign_session, rng, F32, 3, inner, rows)
    xb, bb, yb = sess.to_device(x), sess.to_device(base), sess.to_device(base)
    call, one = sess.adapters, [(0, cols, a.h, 1.0)]
    assert call(one, xb.ptr, 0, yb.ptr, rows, bb.ptr) == arg and call(one, xb.ptr, cols, yb.ptr, 0, bb.ptr) == arg
    assert call(one, None, cols, yb.ptr, rows, bb.ptr) == arg and call(one, xb.ptr, cols, None, rows, bb.ptr) == arg
    assert call([(0, cols + 1, a.h, 1.0)], xb.ptr, cols, yb.ptr, rows, bb.ptr) == arg and call([(3, 2, a.h, 1.0)], xb.ptr, cols, yb.ptr, rows, bb.ptr) == arg
    assert call(one, xb.ptr, cols, yb.ptr, rows + 1, bb.ptr) == arg
    assert call([(0, 2, a.h, 1.0), (2, 4, other.h, 1.0)], xb.ptr, cols, yb.ptr, rows, bb.ptr) == arg
    assert call([(0, 2, foreign.h, 1.0)], xb.ptr, cols, yb.ptr, rows, bb.ptr) == arg
    assert call(one, xb.ptr, cols, yb.ptr, rows, bb.ptr, ldx=inner - 1) == arg and call(one, xb.ptr, cols, yb.ptr, rows, bb.ptr, ldy=rows - 1) == arg
    assert call(one, xb.ptr + 2, cols, yb.ptr, rows, bb.ptr) == arg and call(one, yb.ptr, cols, yb.ptr, rows, bb.ptr) == arg
    assert call(one, xb.ptr, 1 << 20, yb.ptr, rows, bb.ptr) == arg and call(one, xb.ptr, cols, yb.ptr, rows, bb.ptr, ldy=1 << 61) == arg
    assert call(one, xb.ptr, cols, base.ctypes.data, rows, bb.ptr) == arg  # pageable output
    assert lib.pixhip_adapters(sess.handle, None, 1, xb.ptr, cols, 0, bb.ptr, yb.ptr, rows, 0) == arg
    assert np.array_equal(yb.download(np.float32, base.size), base.reshape(-1))
    foreign_session.close()
    for b in (a, other, xb, bb, yb, dev):
        b.free()
