"""pixhip_residual_norm_quantize through the C ABI: against the calls that it stands
for (bit for bit, quantized activations included) and against its formula in 64 bits.

The bound of the second.  With u = 2^-24 (half a step of fp32): the added term b' *
tanh(gate) * scale is rounded at most 7 times (x - mean, 1 / sqrt, two products, tanh,
two products), the sum once:  dx = 7 u |add| + u |x'|.  y is rounded at most 6 times,
and takes over x's errors directly, through the mean and through the mean square:
  dy = 7 u |y| + inverse |w (1 + m)| (dx + max dx) + |y| inverse max dx.
Both are taken 1 % larger for the second order.
"""
import ctypes

import numpy as np
import pytest

from gpu_helpers import Pinned, new_session
from pixelina_amd import Q5_K, Q8_0, _lib, synth

pytestmark = pytest.mark.gpu

NONE, RMS, LAYER = _lib.NORM_NONE, _lib.NORM_RMS, _lib.NORM_LAYER
RESIDUAL = 9
GUARD = 16


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


def inputs(rows, inner, seed=0):
    rng = np.random.default_rng(1000 * rows + inner + seed)
    n = lambda *shape: rng.standard_normal(shape).astype(np.float32)  # noqa: E731
    return {"x": 4 * n(rows, inner) * np.exp(n(inner)), "branch": 0.7 * n(rows, inner) + np.float32(0.1), "post_weight": 1 + 0.2 * n(inner),
            "pre_weight": 1 + 0.2 * n(inner), "gate": n(2, inner), "modulation": 0.5 * n(2, inner)}


def norm64(x, how, weight, eps):
    if how == NONE:
        return x, np.zeros(x.shape[:-1] + (1,)), weight
    x = x - x.mean(axis=-1, keepdims=True) if how == LAYER else x
    inverse = 1 / np.sqrt((x * x).mean(axis=-1, keepdims=True) + np.float64(np.float32(eps)))
    return x * inverse * weight, inverse, weight


def definition(t, post, pre, gate, modulation, split, scale, eps=1e-5):
    """(x', bound, y, bound) in 64 bits."""
    d = {k: v.astype(np.float64) for k, v in t.items()}
    before = (np.arange(t["x"].shape[0]) < split).astype(int)
    add = norm64(d["branch"], post, d["post_weight"], eps)[0] * np.float64(np.float32(scale))
    if gate:
        add = add * np.tanh(d["gate"])[before]
    u = 2.0 ** -24
    x = d["x"] + add
    dx = 1.01 * (7 * u * np.abs(add) + u * np.abs(x)) + 1e-44
    if pre == NONE:
        return x, dx, None, None
    y, inverse, w = norm64(x, pre, d["pre_weight"], eps)
    f = 1 + d["modulation"][before] if modulation else np.ones_like(x)
    worst = dx.max(axis=-1, keepdims=True)
    dy = 1.01 * (7 * u * np.abs(y * f) + inverse * np.abs(w * f) * (dx + worst) + np.abs(y * f) * inverse * worst) + 1e-44
    return x, dx, y * f, dy


class Call:
    """One call's tensors in device memory, `shift` bytes off a 16-byte boundary, guards behind the outputs."""

    def __init__(self, sess, t, shift=0):
        self.sess, self.shift, self.bufs = sess, shift, []
        self.rows, self.inner = t["x"].shape
        self.p = {k: self.place(v) for k, v in t.items()}
        self.out, self.y = self.place(np.full(t["x"].size + GUARD, 7.0, np.float32)), self.place(np.full(t["x"].size + GUARD, 7.0, np.float32))

    def place(self, a):
        b = self.sess.alloc(a.nbytes + 64)
        b.upload(np.ascontiguousarray(a), self.shift)
        self.bufs.append(b)
        return b.ptr + self.shift

    def get(self, ptr):
        b = next(b for b in self.bufs if b.ptr == ptr - self.shift)
        n = self.rows * self.inner
        a = b.download(np.float32, n + GUARD, self.shift)
        assert (a[n:] == 7).all()
        return a[:n].reshape(self.rows, self.inner)

    def run(self, post=NONE, pre=RMS, gate=False, modulation=False, split=0, scale=1.0, wtype=0, eps=1e-5, out=None, y=None, want_y=True, blocks=None,
            x=None, branch=None):
        row = 4 * self.inner
        return self.sess.residual_norm_quantize(
            wtype, x or self.p["x"], branch or self.p["branch"], self.rows, self.inner, out or self.out, (y or self.y) if pre and want_y else None, blocks,
            post=post, post_weight_ptr=self.p["post_weight"] if post else None, post_eps=eps, gate_ptr=self.p["gate"] if gate else None, scale=scale,
            pre=pre, pre_weight_ptr=self.p["pre_weight"] if pre else None, pre_eps=eps, modulation_ptr=self.p["modulation"] if modulation else None,
            target_begin=split, gate_before_ptr=self.p["gate"] + row if gate else None,
            modulation_before_ptr=self.p["modulation"] + row if modulation else None)

    def free(self):
        for b in self.bufs:
            b.free()


def bits(a):
    return np.ascontiguousarray(a).view(np.uint32)


SHAPES = [(1, 1), (3, 2), (2, 5), (7, 63), (5, 64), (33, 255), (4, 256), (3, 257), (17, 1023), (2, 1024), (129, 1538), (1, 4096), (3, 4097), (2, 8191),
          (2, 8193), (1, 20001), (2, 10240)]


@pytest.mark.parametrize("post,pre", [(NONE, RMS), (RMS, RMS), (LAYER, LAYER), (NONE, LAYER), (RMS, NONE), (NONE, NONE)])
@pytest.mark.parametrize("rows,inner", SHAPES)
def test_formula(sess, rows, inner, post, pre):
    t = inputs(rows, inner)
    for gate, modulation, split, scale, shift in ((True, True, 0, 1.0, 0), (True, True, (rows + 1) // 2, 0.22, 4), (False, False, 0, 1.0, 0),
                                                  (False, True, rows, 1.0, 0)):
        c = Call(sess, t, shift)
        modulation = modulation and pre != NONE
        _lib.check(c.run(post, pre, gate, modulation, split, scale), "residual_norm_quantize")
        x, dx, y, dy = definition(t, post, pre, gate, modulation, split, scale)
        assert (np.abs(c.get(c.out) - x) <= dx).all()
        if pre:
            assert (np.abs(c.get(c.y) - y) <= dy).all()
        else:
            assert (c.get(c.y) == 7).all()
        c.free()


@pytest.mark.parametrize("rows,inner", [(300, 4096), (257, 3844), (1100, 1024), (600, 2048), (515, 1028), (3, 6144), (65, 8192), (9, 8196), (2, 20480), (3, 16384)])
def test_rows_on_both_sides(sess, rows, inner):
    """The forms of each row length, with rows before target_begin at every place in a workgroup's runs."""
    t = inputs(rows, inner, 7)
    c = Call(sess, t)
    for split in (1, rows // 2, rows - 1):
        for post, pre, gate, modulation in ((RMS, RMS, True, True), (NONE, LAYER, True, False), (LAYER, RMS, False, True)):
            _lib.check(c.run(post, pre, gate, modulation, split, 1.5), "residual_norm_quantize")
            x, dx, y, dy = definition(t, post, pre, gate, modulation, split, 1.5)
            assert (np.abs(c.get(c.out) - x) <= dx).all() and (np.abs(c.get(c.y) - y) <= dy).all()
    c.free()


@pytest.mark.parametrize("rows,inner", [(300, 4093), (5, 4095), (1100, 1021), (600, 2046), (515, 1029), (3, 6143), (65, 8190), (9, 8199), (5, 10243), (2, 20479),
                                        (3, 20480), (3, 20483), (2, 20484)])
def test_odd_rows_on_both_sides(sess, rows, inner):
    """Rows of any size, off a 16-byte boundary, in the forms of each length; a layer norm on either side."""
    t = inputs(rows, inner, 17)
    c = Call(sess, t, 4)
    for split in (1, rows // 2, rows):
        for post, pre, gate, modulation in ((RMS, LAYER, True, True), (LAYER, LAYER, False, True), (LAYER, RMS, True, False)):
            _lib.check(c.run(post, pre, gate, modulation, split, 0.5), "residual_norm_quantize")
            x, dx, y, dy = definition(t, post, pre, gate, modulation, split, 0.5)
            assert (np.abs(c.get(c.out) - x) <= dx).all() and (np.abs(c.get(c.y) - y) <= dy).all()
    c.free()


def test_host_operands(sess):
    """Inputs and vectors in pageable and in pinned memory, outputs in pinned memory."""
    rows, inner = 21, 260
    t = inputs(rows, inner, 3)
    x, dx, y, dy = definition(t, RMS, RMS, True, True, 8, 1.0)
    c = Call(sess, t)
    pinned = {k: Pinned(sess, v) for k, v in t.items()}
    outs = [Pinned(sess, np.zeros((rows, inner), np.float32)) for _ in range(2)]
    for place in ({k: v.ctypes.data for k, v in t.items()}, {k: v.p.value for k, v in pinned.items()}):
        c.p = place
        _lib.check(c.run(RMS, RMS, True, True, 8), "host inputs")
        assert (np.abs(c.get(c.out) - x) <= dx).all() and (np.abs(c.get(c.y) - y) <= dy).all()
        _lib.check(c.run(RMS, RMS, True, True, 8, out=outs[0].p.value, y=outs[1].p.value), "host inputs and outputs")
        sess.synchronize()
        assert (np.abs(outs[0].read(np.float32, x.shape) - x) <= dx).all() and (np.abs(outs[1].read(np.float32, x.shape) - y) <= dy).all()
    host = np.zeros((rows, inner), np.float32)
    assert c.run(RMS, RMS, out=host.ctypes.data) == _lib.ERR_ARGUMENT and c.run(RMS, RMS, y=host.ctypes.data) == _lib.ERR_ARGUMENT
    for b in (*pinned.values(), *outs, c):
        b.free()


def composed(c, post, pre, gate, modulation, wtype, blocks):
    """The calls it stands for: (x', y, blocks)."""
    s, rows, inner, p = c.sess, c.rows, c.inner, c.p
    b = p["branch"]
    if post:
        b = c.place(np.zeros((rows, inner), np.float32))
        _lib.check(s.norm_quantize(0, p["branch"], rows, inner, p["post_weight"], 1e-5, post == LAYER, None, b), "norm")
    x = c.place(np.full(rows * inner + GUARD, 7.0, np.float32))
    s.copy_device(x, p["x"], 4 * rows * inner)
    _lib.check(s.pointwise_ex(RESIDUAL, x, b, p["gate"] if gate else None, rows, inner), "residual")
    y = c.place(np.full(rows * inner + GUARD, 7.0, np.float32))
    _lib.check(s.norm_quantize(wtype, x, rows, inner, p["pre_weight"], 1e-5, pre == LAYER, p["modulation"] if modulation else None, y, blocks), "norm")
    return c.get(x), c.get(y)


@pytest.mark.parametrize("post,pre,gate,modulation", [(RMS, RMS, True, True), (NONE, RMS, False, False), (LAYER, LAYER, True, True), (NONE, LAYER, True, False)])
@pytest.mark.parametrize("rows,inner", [(1, 3840), (4608, 256), (70, 3840), (9, 4096), (5, 544), (3, 10240), (2, 20480)])
def test_the_calls_it_stands_for(sess, rows, inner, post, pre, gate, modulation):
    t = inputs(rows, inner, 5)
    for wtype, size, block in ((0, 4, 1), (Q8_0, 34, 32), (Q5_K, 292, 256)):
        if inner % block:
            continue
        c = Call(sess, t)
        count = rows * inner // block * size if wtype else 4
        mine, theirs = sess.to_device(np.full(count + 64, 9, np.uint8)), sess.to_device(np.full(count + 64, 9, np.uint8))
        x, y = composed(c, post, pre, gate, modulation, wtype, theirs.ptr if wtype else None)
        _lib.check(c.run(post, pre, gate, modulation, wtype=wtype, blocks=mine.ptr if wtype else None), "residual_norm_quantize")
        assert np.array_equal(bits(c.get(c.out)), bits(x)) and np.array_equal(bits(c.get(c.y)), bits(y))
        assert np.array_equal(mine.download(np.uint8, count + 64), theirs.download(np.uint8, count + 64))
        for b in (mine, theirs):
            b.free()
        c.free()


@pytest.mark.parametrize("wtype,rows,inner", [(Q8_0, 37, 544), (Q5_K, 37, 512), (Q8_0, 1, 4096), (Q5_K, 300, 3840)])
def test_activations_for_the_next_layers(sess, wtype, rows, inner):
    """What MULTIPLY reads afterwards is what pixhip_norm_quantize leaves."""
    t, n = inputs(rows, inner, 9), 160
    w = (np.random.default_rng(3).standard_normal((n, inner)) * 0.05).astype(np.float32)
    from oracle_lib import oracle, quantize
    packed = quantize(oracle(), "orc", w, "q8_0") if wtype == Q8_0 else synth.pack_q5_K(w)
    h = sess.weight(f"residual:{wtype}:{inner}", packed, wtype, inner, n)
    got = []
    for composition in (False, True):
        c = Call(sess, t)
        if composition:
            composed(c, RMS, RMS, True, True, wtype, None)
        else:
            _lib.check(c.run(RMS, RMS, True, True, wtype=wtype, want_y=False), "residual_norm_quantize")
            assert (c.get(c.y) == 7).all()
        y = sess.alloc(4 * rows * n)
        _lib.check(sess.matmul_stage(h, None, rows, y.ptr, _lib.STAGE_MULTIPLY), "multiply")
        got.append(y.download(np.uint32, rows * n))
        y.free()
        c.free()
    assert np.array_equal(*got)


@pytest.mark.parametrize("rows,inner,post,pre", [(5, 544, LAYER, LAYER), (3, 8224, NONE, LAYER), (2, 10272, LAYER, RMS), (2, 20512, LAYER, LAYER), (300, 1056, LAYER, LAYER)])
def test_layer_norms_of_padded_rows(sess, rows, inner, post, pre):
    """Q8_0 activations whose rows end inside a chunk of 256 values, their tensors on and off a 16-byte boundary."""
    t = inputs(rows, inner, 19)
    n = 96
    w = (np.random.default_rng(4).standard_normal((n, inner)) * 0.05).astype(np.float32)
    from oracle_lib import oracle, quantize
    h = sess.weight(f"layer:{inner}", quantize(oracle(), "orc", w, "q8_0"), Q8_0, inner, n)
    got = []
    for composition, shift in ((True, 0), (False, 0), (False, 4)):
        c = Call(sess, t, shift)
        if composition:
            composed(c, post, pre, True, True, Q8_0, None)
        else:
            _lib.check(c.run(post, pre, True, True, wtype=Q8_0, want_y=False), "residual_norm_quantize")
        y = sess.alloc(4 * rows * n)
        _lib.check(sess.matmul_stage(h, None, rows, y.ptr, _lib.STAGE_MULTIPLY), "multiply")
        got.append(y.download(np.uint32, rows * n))
        y.free()
        c.free()
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


def test_in_place(sess):
    for rows, inner in ((5, 1000), (700, 256), (3, 8500)):
        t = inputs(rows, inner, 2)
        c = Call(sess, t)
        _lib.check(c.run(RMS, RMS, True, True), "apart")
        x, y = c.get(c.out), c.get(c.y)
        c.free()
        for out, norm in (("x", None), ("branch", None), (None, "x"), (None, "branch"), ("x", "branch"), ("branch", "x")):
            t2 = {k: np.concatenate([v.reshape(-1), np.full(GUARD, 7, np.float32)]) if k in ("x", "branch") else v for k, v in t.items()}
            c = Call(sess, t)
            for k in ("x", "branch"):
                c.p[k] = c.place(t2[k])
            _lib.check(c.run(RMS, RMS, True, True, out=c.p[out] if out else None, y=c.p[norm] if norm else None), "in place")
            assert np.array_equal(bits(c.get(c.p[out] if out else c.out)), bits(x))
            assert np.array_equal(bits(c.get(c.p[norm] if norm else c.y)), bits(y))
            c.free()


def test_rows_that_are_not_finite_stay_alone(sess):
    t = inputs(9, 700, 4)
    t["x"][2, 5], t["branch"][4, 699], t["branch"][7, 0] = np.nan, np.inf, np.nan
    c = Call(sess, t)
    _lib.check(c.run(LAYER, RMS, True, True), "residual_norm_quantize")
    x, dx, y, dy = definition(t, LAYER, RMS, True, True, 0, 1.0)
    good = [r for r in range(9) if r not in (2, 4, 7)]
    assert (np.abs(c.get(c.out)[good] - x[good]) <= dx[good]).all() and (np.abs(c.get(c.y)[good] - y[good]) <= dy[good]).all()
    assert np.isnan(c.get(c.y)[[2, 4, 7]]).all() and np.isnan(c.get(c.out)[2, 5])
    c.free()
    t["branch"][:] = 0  # a norm of zeros is zero
    t["x"][:] = 0
    c = Call(sess, t)
    _lib.check(c.run(RMS, RMS, True, True), "residual_norm_quantize")
    assert (c.get(c.out) == 0).all() and (c.get(c.y) == 0).all()
    c.free()


def test_captured(sess):
    from gpu_helpers import new_session
    s = new_session()
    lib, stream, graph, ready = s.lib, ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    try:
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, stream), "set_stream")
        t = inputs(40, 520, 1)
        c = Call(s, t)
        _lib.check(c.run(RMS, LAYER, True, True, 13), "eager")
        x, y = c.get(c.out), c.get(c.y)
        assert lib.hipStreamBeginCapture(stream, 1) == 0
        code = c.run(RMS, LAYER, True, True, 13)
        assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0 and code == _lib.OK
        assert lib.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)) == 0
        n = x.size
        for i in range(3):
            next(b for b in c.bufs if b.ptr == c.out).upload(np.full(n, float(i), np.float32))
            _lib.check(c.run(NONE, RMS), "other work")
            assert lib.hipGraphLaunch(ready, stream) == 0
            assert np.array_equal(bits(c.get(c.out)), bits(x)) and np.array_equal(bits(c.get(c.y)), bits(y))
        s.synchronize()
        assert lib.hipGraphExecDestroy(ready) == 0 and lib.hipGraphDestroy(graph) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, None), "set_stream")
        assert lib.hipStreamDestroy(stream) == 0
    finally:
        s.close()


def test_refusals(sess):
    c = Call(sess, inputs(4, 64))
    arg = _lib.ERR_ARGUMENT
    call = sess.residual_norm_quantize
    x, b, o, y = c.p["x"], c.p["branch"], c.out, c.y
    assert call(0, None, b, 4, 64, o, y) == arg and call(0, x, None, 4, 64, o, y) == arg and call(0, x, b, 4, 64, None, y) == arg
    assert call(0, x, b, 0, 64, o, y) == arg and call(0, x, b, 4, 0, o, y) == arg
    assert call(0, x, b, 4, 64, o, o) == arg and call(0, x, b, 4, 64, o, None) == arg
    assert call(0, x, b, 4, 64, o, y, pre=3) == arg and call(0, x, b, 4, 64, o, y, post=-1) == arg
    assert call(0, x, b, 4, 64, o, y, pre=NONE) == arg and call(Q8_0, x, b, 4, 64, o, None, pre=NONE) == arg
    assert call(0, x, b, 4, 64, o, None, pre=NONE, modulation_ptr=c.p["modulation"]) == arg
    assert call(0, x, b, 4, 64, o, y, y) == arg                      # blocks without a type
    assert call(2, x, b, 4, 64, o, y) == _lib.ERR_UNSUPPORTED
    assert call(Q5_K, x, b, 4, 64, o, y) == arg                      # not whole blocks
    assert call(0, x, b, 4, 64, o, y, target_begin=5) == arg
    assert call(0, x, b, 4, 64, o, y, target_begin=2, gate_ptr=c.p["gate"]) == arg
    assert call(0, x + 2, b, 4, 64, o, y) == arg
    assert call(0, x, b, 1 << 20, 64, o, y) == arg                   # past the allocations
    assert sess.lib.pixhip_residual_norm_quantize(sess.handle, 0, x, b, 4, 64, None, o, y, None) == arg
    assert (c.get(o) == 7).all() and (c.get(y) == 7).all()
    c.free()
