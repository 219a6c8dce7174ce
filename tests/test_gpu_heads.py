"""pixhip_split_heads and pixhip_cache_append_rotated through the C ABI, bit for bit
against their definition: a head's statistics in 64 bits, every product and sum after
them rounded to 32 (numpy), and against the calls that they stand for.  (The sums of a
head's squares are formed in another order than numpy's; both are within 2^-47 of the
exact one, which moves 1 / sqrt's rounding to 32 bits once in some 2^23 heads: the
seeds are fixed, and none of these heads is such a one.)
"""
import ctypes

import numpy as np
import pytest

from gpu_helpers import Pinned, new_session
from pixelina_amd import _lib
from test_gpu_cache import append, held, read, same

pytestmark = pytest.mark.gpu

NONE, RMS, LAYER = _lib.NORM_NONE, _lib.NORM_RMS, _lib.NORM_LAYER
EPS = 1e-6


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


def turned(x, dim, norm, weight, cosine, sine, rotary, interleaved):
    """Heads of x [rows][heads * dim] by the definition."""
    x = x.reshape(x.shape[0], -1, dim)
    if norm != NONE:
        wide = x.astype(np.float64)
        if norm == LAYER:
            wide = wide - wide.mean(axis=-1, keepdims=True)
        inverse = (1 / np.sqrt((wide * wide).mean(axis=-1, keepdims=True) + np.float64(np.float32(EPS)))).astype(np.float32)
        x = wide.astype(np.float32) * inverse
        if weight is not None:
            x = x * weight
    out = x.copy()
    if rotary:
        first, second = (np.arange(0, rotary, 2), np.arange(1, rotary, 2)) if interleaved else (np.arange(rotary // 2), np.arange(rotary // 2, rotary))
        a, b, c, s = x[..., first], x[..., second], cosine[:, None], sine[:, None]
        out[..., first] = a * c - b * s
        out[..., second] = a * s + b * c
    return out.reshape(x.shape[0], -1)


def make(rows, heads, kv, dim, rotary, seed=0, pad=0):
    rng = np.random.default_rng(rows * 131 + heads * 7 + dim + seed)
    n = lambda *shape: rng.standard_normal(shape).astype(np.float32)  # noqa: E731
    angle = rng.uniform(0, 50, (rows, rotary // 2))
    return {"qkv": n(rows, (heads + 2 * kv) * dim + pad) * 3, "qw": 1 + n(dim) / 4, "kw": 1 + n(dim) / 4, "cos": np.cos(angle).astype(np.float32),
            "sin": np.sin(angle).astype(np.float32)}


def upload(sess, t, shift=0):
    """Device copies, `shift` bytes off a 16-byte boundary: (addresses, buffers)."""
    bufs = {k: sess.alloc(v.nbytes + 32).upload(v, shift) for k, v in t.items()}
    return {k: b.ptr + shift for k, b in bufs.items()}, bufs


def rotation(sess, p, rotary, interleaved, norm):
    return sess.rotation(p["cos"] if rotary else None, p["sin"] if rotary else None, rotary, interleaved, norm, p["qw"], p["kw"], EPS)


def parts(t, heads, kv, dim):
    q, k = heads * dim, kv * dim
    return t["qkv"][:, :q], t["qkv"][:, q:q + k], t["qkv"][:, q + k:q + 2 * k]


CASES = [  # rows, heads, kv, dim, rotary, interleaved, norm, pad, shift
    (1, 32, 8, 128, 128, False, RMS, 0, 0), (77, 30, 30, 128, 128, True, RMS, 0, 0), (33, 20, 5, 80, 80, False, NONE, 0, 0), (5, 14, 2, 90, 46, True, NONE, 0, 0),
    (9, 3, 1, 128, 64, False, LAYER, 4, 0), (9, 3, 3, 96, 40, False, RMS, 3, 0), (2, 1, 1, 1, 0, False, RMS, 0, 0), (3, 2, 1, 2, 2, True, RMS, 1, 0),
    (4, 5, 2, 33, 32, False, LAYER, 0, 0), (7, 4, 2, 64, 64, True, LAYER, 0, 4), (700, 4, 4, 128, 128, False, RMS, 0, 0), (600, 5, 3, 36, 24, True, RMS, 0, 0),
    (3, 2, 1, 129, 128, False, RMS, 0, 0), (6, 3, 3, 256, 256, True, RMS, 0, 0), (2, 2, 1, 512, 512, False, LAYER, 0, 0), (2, 1, 1, 511, 510, True, RMS, 0, 0),
    (3, 7, 7, 100, 8, False, RMS, 0, 0), (3, 7, 7, 100, 0, False, RMS, 0, 0), (2, 3, 1, 20, 16, False, LAYER, 0, 0), (40000, 1, 1, 8, 8, False, RMS, 0, 0)]


@pytest.mark.parametrize("rows,heads,kv,dim,rotary,interleaved,norm,pad,shift", CASES)
def test_split_heads(sess, rows, heads, kv, dim, rotary, interleaved, norm, pad, shift):
    t = make(rows, heads, kv, dim, rotary, pad=pad)
    p, bufs = upload(sess, t, shift)
    q, k, v = parts(t, heads, kv, dim)
    want = [turned(q, dim, norm, t["qw"], t["cos"], t["sin"], rotary, interleaved), turned(k, dim, norm, t["kw"], t["cos"], t["sin"], rotary, interleaved), v]
    outs = [sess.to_device(np.full(a.size + 16, 7.0, np.float32)) for a in (q, k, v)]
    at = [p["qkv"], p["qkv"] + 4 * heads * dim, p["qkv"] + 4 * (heads + kv) * dim]
    ld = t["qkv"].shape[1]
    for chosen in ((True, True, True), (False, True, False), (True, False, True)):
        ins, to = ([a if c else None for a, c in zip(x, chosen)] for x in (at, [b.ptr for b in outs]))
        for b, w in zip(outs, want):
            b.upload(np.full(w.size + 16, 7.0, np.float32))
        _lib.check(sess.split_heads(*ins, rows, heads, kv, dim, rotation(sess, p, rotary, interleaved, norm), *to, ld=ld), "split_heads")
        for b, w, c in zip(outs, want, chosen):
            got = b.download(np.float32, w.size + 16)
            assert (got[w.size if c else 0:] == 7).all()
            assert not c or same(got[:w.size].reshape(w.shape), w)
    for b in [*outs, *bufs.values()]:
        b.free()


def test_split_heads_in_place_and_without_a_rotation(sess):
    rows, heads, kv, dim = 50, 6, 2, 64
    t = make(rows, heads, kv, dim, dim)
    q, k, v = (np.ascontiguousarray(a) for a in parts(t, heads, kv, dim))
    p, bufs = upload(sess, t)
    b = [sess.to_device(a) for a in (q, k, v)]
    _lib.check(sess.split_heads(*(x.ptr for x in b), rows, heads, kv, dim, rotation(sess, p, dim, False, RMS), *(x.ptr for x in b)), "in place")
    want = [turned(q, dim, RMS, t["qw"], t["cos"], t["sin"], dim, False), turned(k, dim, RMS, t["kw"], t["cos"], t["sin"], dim, False), v]
    for x, w in zip(b, want):
        assert same(x.download(np.float32, w.size).reshape(w.shape), w)
    out = sess.alloc(q.nbytes)
    _lib.check(sess.split_heads(p["qkv"], None, None, rows, heads, kv, dim, None, out.ptr, ld=t["qkv"].shape[1]), "copy")
    assert same(out.download(np.float32, q.size).reshape(q.shape), q)
    # rotary 0 with tables: the whole head; weights absent: 1
    r = sess.rotation(p["cos"], p["sin"], norm=RMS, eps=EPS)
    _lib.check(sess.split_heads(p["qkv"], None, None, rows, heads, kv, dim, r, out.ptr, ld=t["qkv"].shape[1]), "whole head")
    assert same(out.download(np.float32, q.size).reshape(q.shape), turned(q, dim, RMS, None, t["cos"], t["sin"], dim, False))
    for x in [*b, out, *bufs.values()]:
        x.free()


def test_the_calls_it_stands_for(sess):
    rows, heads, dim = 130, 30, 128
    t = make(rows, heads, heads, dim, dim, 3)
    p, bufs = upload(sess, t)
    for interleaved in (False, True):
        for norm in (RMS, LAYER):
            q = np.ascontiguousarray(parts(t, heads, heads, dim)[0])
            x, y, z = sess.to_device(q), sess.alloc(q.nbytes), sess.alloc(q.nbytes)
            _lib.check(sess.norm_quantize(0, x.ptr, rows * heads, dim, p["qw"], EPS, norm == LAYER, None, y.ptr), "norm")
            _lib.check(sess.rope(y.ptr, rows, heads * dim, heads, p["cos"], p["sin"], interleaved), "rope")
            _lib.check(sess.split_heads(p["qkv"], None, None, rows, heads, heads, dim, rotation(sess, p, dim, interleaved, norm), z.ptr,
                                        ld=t["qkv"].shape[1]), "split_heads")
            assert np.array_equal(y.download(np.uint32, q.size), z.download(np.uint32, q.size))
            for b in (x, y, z):
                b.free()
    for b in bufs.values():
        b.free()


@pytest.mark.parametrize("rows,heads,kv,dim,rotary,interleaved,norm,pad,shift", [c for c in CASES if c[3] <= 128])
@pytest.mark.parametrize("start", [0, 1, 31, 32, 77])
def test_append_rotated(sess, start, rows, heads, kv, dim, rotary, interleaved, norm, pad, shift):
    """The cache holds what pixhip_cache_append would make of the turned keys; a second append goes on from it."""
    rows = min(rows, 200)
    t = make(rows, heads, kv, dim, rotary, start, pad)
    q, k, v = parts(t, heads, kv, dim)
    kt = turned(k, dim, norm, t["kw"], t["cos"], t["sin"], rotary, interleaved)
    rng = np.random.default_rng(start)
    k0, v0 = (rng.standard_normal((start, kv * dim)).astype(np.float32) for _ in range(2))
    weights = rng.random((rows, kv)).astype(np.float32)
    p, bufs = upload(sess, t, shift)
    wb, qb = sess.to_device(weights), sess.to_device(np.full(q.size + 16, 7.0, np.float32))
    cache = sess.cache(2, kv, dim, start + rows + 40)
    if start:
        append(sess, cache, k0, v0, 1)
    ld = t["qkv"].shape[1]
    _lib.check(sess.cache_append_rotated(cache, 1, p["qkv"], p["qkv"] + 4 * heads * dim, p["qkv"] + 4 * (heads + kv) * dim, rows, heads,
                                         rotation(sess, p, rotary, interleaved, norm), qb.ptr, ld=ld, weights_ptr=wb.ptr), "append_rotated")
    assert sess.cache_length(cache, 1) == start + rows and sess.cache_length(cache, 0) == 0
    got = qb.download(np.float32, q.size + 16)
    assert (got[q.size:] == 7).all() and same(got[:q.size].reshape(q.shape), turned(q, dim, norm, t["qw"], t["cos"], t["sin"], rotary, interleaved))
    k1, v1 = np.concatenate([k0, kt]), np.concatenate([v0, v])
    got = read(sess, cache, kv, dim, layer=1)
    assert same(got[0], held(k1, kv)) and same(got[1], held(v1, kv))
    assert same(got[2], np.concatenate([np.zeros((start, kv), np.float32), weights]))
    # more rows: the open block is quantized again from the fp32 rows that the call left
    more = [rng.standard_normal((7, kv * dim)).astype(np.float32) for _ in range(2)]
    append(sess, cache, *more, layer=1)
    got = read(sess, cache, kv, dim, layer=1)
    assert same(got[0], held(np.concatenate([k1, more[0]]), kv)) and same(got[1], held(np.concatenate([v1, more[1]]), kv))
    sess.cache_destroy(cache)
    for b in (wb, qb, *bufs.values()):
        b.free()


def test_append_rotated_row_by_row_and_cut_back(sess):
    """One row at a time, with a drafted row taken back in between, holds what one call holds; q may be left out."""
    rows, heads, kv, dim = 70, 4, 2, 128
    t = make(rows, heads, kv, dim, dim, 11)
    p, bufs = upload(sess, t)
    ld = t["qkv"].shape[1]
    one, many = sess.cache(1, kv, dim, rows), sess.cache(1, kv, dim, rows + 1)
    k, v = p["qkv"] + 4 * heads * dim, p["qkv"] + 4 * (heads + kv) * dim
    _lib.check(sess.cache_append_rotated(one, 0, None, k, v, rows, 0, rotation(sess, p, dim, False, RMS), ld=ld), "whole")
    for r in range(rows):
        table = sess.rotation(p["cos"] + 4 * r * dim // 2, p["sin"] + 4 * r * dim // 2, dim, False, RMS, p["qw"], p["kw"], EPS)
        for take in (0, 1):
            if take:
                _lib.check(sess.cache_truncate(many, 0, r), "truncate")
            elif r % 5:
                continue
            _lib.check(sess.cache_append_rotated(many, 0, None, k + 4 * r * ld, v + 4 * r * ld, 1, 0, table, ld=ld), "row")
    for a, b in zip(read(sess, one, kv, dim), read(sess, many, kv, dim)):
        assert same(a, b)
    for c in (one, many):
        sess.cache_destroy(c)
    for b in bufs.values():
        b.free()


def test_values_that_are_not_finite(sess):
    """NaN in a head spoils that head alone; a rotation by tables of 0 and 1 keeps what does not turn."""
    rows, heads, kv, dim = 3, 4, 2, 64
    t = make(rows, heads, kv, dim, 32, 2)
    t["qkv"][1, 70], t["qkv"][2, 50] = np.nan, np.inf
    p, bufs = upload(sess, t)
    q = parts(t, heads, kv, dim)[0]
    out = sess.alloc(q.size * 4)
    with np.errstate(invalid="ignore"):
        for norm in (NONE, RMS):
            _lib.check(sess.split_heads(p["qkv"], None, None, rows, heads, kv, dim, rotation(sess, p, 32, False, norm), out.ptr, ld=t["qkv"].shape[1]), "split")
            want, got = turned(q, dim, norm, t["qw"], t["cos"], t["sin"], 32, False), out.download(np.float32, q.size).reshape(q.shape)
            assert np.array_equal(np.isnan(got), np.isnan(want)) and same(np.nan_to_num(got), np.nan_to_num(want))
    for b in (out, *bufs.values()):
        b.free()


def test_host_operands(sess):
    rows, heads, kv, dim = 19, 4, 2, 64
    t = make(rows, heads, kv, dim, dim, 8)
    q, k, v = parts(t, heads, kv, dim)
    want = [turned(q, dim, RMS, t["qw"], t["cos"], t["sin"], dim, True), turned(k, dim, RMS, t["kw"], t["cos"], t["sin"], dim, True), v]
    pinned = {n: Pinned(sess, np.ascontiguousarray(a)) for n, a in t.items()}
    ld = t["qkv"].shape[1]
    for p in ({n: a.ctypes.data for n, a in t.items()}, {n: a.p.value for n, a in pinned.items()}):
        outs = [sess.alloc(w.nbytes) for w in want]
        at = [p["qkv"], p["qkv"] + 4 * heads * dim, p["qkv"] + 4 * (heads + kv) * dim]
        _lib.check(sess.split_heads(*at, rows, heads, kv, dim, rotation(sess, p, dim, True, RMS), *(b.ptr for b in outs), ld=ld), "split_heads")
        for b, w in zip(outs, want):
            assert same(b.download(np.float32, w.size).reshape(w.shape), w)
            b.free()
    for a in pinned.values():
        a.free()


def test_captured(sess):
    rows, heads, kv, dim = 5, 8, 2, 128
    t = make(rows, heads, kv, dim, dim, 21)
    q, k, v = parts(t, heads, kv, dim)
    want = turned(q, dim, RMS, t["qw"], t["cos"], t["sin"], dim, False)
    kt = turned(k, dim, RMS, t["kw"], t["cos"], t["sin"], dim, False)
    s = new_session()
    lib, stream, graph, ready = s.lib, ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    try:
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, stream), "set_stream")
        p, bufs = upload(s, t)
        out, cache = s.to_device(np.zeros(q.size, np.float32)), s.cache(1, kv, dim, 64)
        s.synchronize()
        assert lib.hipStreamBeginCapture(stream, 1) == 0
        code = s.cache_append_rotated(cache, 0, p["qkv"], p["qkv"] + 4 * heads * dim, p["qkv"] + 4 * (heads + kv) * dim, rows, heads,
                                      rotation(s, p, dim, False, RMS), out.ptr, ld=t["qkv"].shape[1])
        assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0 and code == _lib.OK
        assert lib.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)) == 0
        for _ in range(3):
            out.upload(np.zeros(q.size, np.float32))
            assert lib.hipGraphLaunch(ready, stream) == 0
            got = read(s, cache, kv, dim)
            assert same(out.download(np.float32, q.size).reshape(q.shape), want) and same(got[0], held(kt, kv)) and same(got[1], held(v, kv))
        s.synchronize()
        assert lib.hipGraphExecDestroy(ready) == 0 and lib.hipGraphDestroy(graph) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, None), "set_stream")
        assert lib.hipStreamDestroy(stream) == 0
    finally:
        s.close()


def test_refusals(sess):
    rows, heads, kv, dim = 4, 4, 2, 64
    t = make(rows, heads, kv, dim, dim)
    p, bufs = upload(sess, t)
    x, out, ld, arg = p["qkv"], sess.to_device(np.full(rows * heads * dim, 7.0, np.float32)), t["qkv"].shape[1], _lib.ERR_ARGUMENT
    good = rotation(sess, p, dim, False, RMS)
    call = sess.split_heads
    assert call(x, None, None, 0, heads, kv, dim, good, out.ptr, ld=ld) == arg
    assert call(x, None, None, rows, 0, kv, dim, good, out.ptr, ld=ld) == arg
    assert call(None, None, None, rows, heads, kv, dim, good) == arg
    assert call(x, None, None, rows, heads, kv, dim, good, None, ld=ld) == arg
    assert call(None, x, None, rows, heads, 0, dim, good, None, out.ptr, ld=ld) == arg
    assert call(x, None, None, rows, heads, kv, 0, good, out.ptr, ld=ld) == arg
    assert call(x, None, None, rows, heads, kv, 513, None, out.ptr) == _lib.ERR_UNSUPPORTED
    assert call(x, None, None, rows, heads, kv, dim, good, out.ptr, ld=heads * dim - 1) == arg
    assert call(x, None, None, rows, heads, kv, dim, good, out.ptr, ld=1 << 60) == arg
    assert call(x, None, None, rows, heads, kv, dim, rotation(sess, p, 66, False, RMS), out.ptr, ld=ld) == arg
    assert call(x, None, None, rows, heads, kv, dim, rotation(sess, p, 5, False, RMS), out.ptr, ld=ld) == arg
    assert call(x, None, None, rows, heads, kv, 63, sess.rotation(p["cos"], p["sin"]), out.ptr, ld=ld) == arg  # an odd head turned whole
    assert call(x, None, None, rows, heads, kv, dim, sess.rotation(p["cos"], None, dim), out.ptr, ld=ld) == arg
    assert call(x, None, None, rows, heads, kv, dim, rotation(sess, p, dim, False, 3), out.ptr, ld=ld) == arg
    assert call(x + 2, None, None, rows, heads, kv, dim, good, out.ptr, ld=ld) == arg
    assert call(x, None, None, 1 << 20, heads, kv, dim, good, out.ptr, ld=ld) == arg  # past the allocations
    host = np.zeros(rows * heads * dim, np.float32)
    assert call(x, None, None, rows, heads, kv, dim, good, host.ctypes.data, ld=ld) == arg
    cache = sess.cache(1, kv, dim, 32)
    k, v = x + 4 * heads * dim, x + 4 * (heads + kv) * dim
    call = sess.cache_append_rotated
    assert call(cache, 1, x, k, v, rows, heads, good, out.ptr, ld=ld) == arg
    assert call(cache, 0, x, None, v, rows, heads, good, out.ptr, ld=ld) == arg
    assert call(cache, 0, x, k, v, rows, heads, good, None, ld=ld) == arg
    assert call(cache, 0, x, k, v, rows, 0, good, out.ptr, ld=ld) == arg
    assert call(cache, 0, x, k, v, 33, heads, good, out.ptr, ld=ld) == _lib.ERR_MEMORY
    assert call(cache, 0, x, k, v, rows, heads, rotation(sess, p, 66, False, RMS), out.ptr, ld=ld) == arg
    assert sess.cache_length(cache, 0) == 0 and (out.download(np.float32, rows * heads * dim) == 7).all()
    sess.cache_destroy(cache)
    for b in (out, *bufs.values()):
        b.free()
