"""pixhip_split_heads and pixhip_cache_append_rotated refuse outputs that lie over what
other workgroups still read, and take those that lie apart from it, however close."""
import numpy as np
import pytest

from gpu_helpers import Pinned, new_session
from pixelina_amd import _lib
from test_gpu_cache import held, read, same
from test_gpu_heads import RMS, make, parts, rotation, turned, upload

pytestmark = pytest.mark.gpu

ROWS, HEADS, KV, DIM = 6, 4, 2, 64
Q, K = HEADS * DIM, KV * DIM


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


@pytest.fixture
def call(sess):
    """The rows of a projection, with room behind them, and their rotation."""
    t = make(ROWS, HEADS, KV, DIM, DIM)
    p, bufs = upload(sess, t)
    room = sess.to_device(np.concatenate([t["qkv"].reshape(-1), np.full(3 * ROWS * Q, 7.0, np.float32)]))
    yield t, p, room, rotation(sess, p, DIM, False, RMS)
    for b in (room, *bufs.values()):
        b.free()


def test_split_heads_refuses_outputs_over_inputs(sess, call):
    t, p, room, turn = call
    x, ld = room.ptr, Q + 2 * K
    k, v, end = x + 4 * Q, x + 4 * (Q + K), x + 4 * ROWS * ld
    before = room.download(np.float32, room.nbytes // 4)
    apart = end + 4 * ROWS * Q
    # in order: q, k, v and their outputs
    for args in ((x, None, None, x, None, None), (None, k, None, None, k, None), (None, None, v, None, None, v),       # strided rows in place
                 (x, None, None, x + 16, None, None), (x, None, None, end - 8 * K - 4, None, None),  # shifted, on a row's last value
                 (x, k, v, end, k, apart), (x, k, v, end, apart, x), (x, k, None, v - 4, end, None),        # over another's rows
                 (x, k, None, end, end + 4 * ROWS * Q - 4, None), (x, k, v, end, apart, apart + 4)):              # outputs over outputs
        assert sess.split_heads(*args[:3], ROWS, HEADS, KV, DIM, turn, *args[3:], ld=ld) == _lib.ERR_ARGUMENT, args
    # contiguous rows over the other tensors' rows, and over each other
    for args in ((x, x, None, x, end, None), (end, x, x, x, apart, apart + 4 * ROWS * K), (x, end, None, end + 16, apart, None), (x, end, None, x, x, None)):
        assert sess.split_heads(*args[:3], ROWS, HEADS, KV, DIM, turn, *args[3:]) == _lib.ERR_ARGUMENT, args
    # over tables and weights
    tables = sess.to_device(np.zeros(4 * ROWS * Q, np.float32))
    at = tables.ptr
    for r in (sess.rotation(at, p["sin"], DIM, False, RMS, p["qw"], p["kw"]), sess.rotation(p["cos"], at + 4 * ROWS * Q - 4, DIM, False, RMS, p["qw"], p["kw"]),
              sess.rotation(p["cos"], p["sin"], DIM, False, RMS, at + 400, p["kw"])):
        assert sess.split_heads(x, None, None, ROWS, HEADS, KV, DIM, r, at, ld=ld) == _lib.ERR_ARGUMENT
    pinned = Pinned(sess, t["qkv"])
    assert sess.split_heads(pinned.p.value, None, None, ROWS, HEADS, KV, DIM, turn, pinned.p.value, ld=ld) == _lib.ERR_ARGUMENT
    sess.synchronize()
    assert np.array_equal(before, room.download(np.float32, before.size)) and (tables.download(np.float32, 4 * ROWS * Q) == 0).all()
    assert np.array_equal(pinned.read(np.float32, t["qkv"].shape), t["qkv"])
    tables.free()
    pinned.free()


def test_split_heads_takes_outputs_beside_inputs(sess, call):
    t, p, room, turn = call
    q, k, v = parts(t, HEADS, KV, DIM)
    ld, x = Q + 2 * K, room.ptr
    want = turned(q, DIM, RMS, t["qw"], t["cos"], t["sin"], DIM, False)
    # right behind the last row's last value of q, and a row's own slice where there is but one row
    end = x + 4 * ((ROWS - 1) * ld + Q)
    _lib.check(sess.split_heads(x, None, None, ROWS, HEADS, KV, DIM, turn, end, ld=ld), "behind the rows")
    got = room.download(np.float32, room.nbytes // 4)[(ROWS - 1) * ld + Q:][:want.size]
    assert same(got.reshape(want.shape), want)
    room.upload(t["qkv"].reshape(-1))
    _lib.check(sess.split_heads(x, x + 4 * Q, None, 1, HEADS, KV, DIM, turn, x, x + 4 * Q, ld=ld), "one row in place")
    got = room.download(np.float32, ld)
    assert same(got[:Q], want[0]) and same(got[Q:Q + K], turned(k, DIM, RMS, t["kw"], t["cos"], t["sin"], DIM, False)[0]) and same(got[Q + K:], v[0])
    # in what lies between two rows
    room.upload(t["qkv"].reshape(-1))
    _lib.check(sess.split_heads(x, None, None, 2, 1, KV, DIM, turn, x + 4 * (ld - 2 * DIM), ld=ld), "between two rows")
    got = room.download(np.float32, ld)
    assert same(got[ld - 2 * DIM:].reshape(2, DIM), turned(t["qkv"][:2, :DIM], DIM, RMS, t["qw"], t["cos"][:2], t["sin"][:2], DIM, False))


def test_append_rotated_refuses_outputs_over_inputs(sess, call):
    t, p, room, turn = call
    x, ld = room.ptr, Q + 2 * K
    k, v, end = x + 4 * Q, x + 4 * (Q + K), x + 4 * ROWS * ld
    before = room.download(np.float32, room.nbytes // 4)
    cache = sess.cache(1, KV, DIM, 64)
    weights = end + 4 * ROWS * Q
    for out in (x, k, v, end - 4, x + 4, weights - 4 * ROWS * Q + 4, weights):
        assert sess.cache_append_rotated(cache, 0, x, k, v, ROWS, HEADS, turn, out, ld=ld, weights_ptr=weights) == _lib.ERR_ARGUMENT, out - x
    assert sess.cache_length(cache, 0) == 0 and np.array_equal(before, room.download(np.float32, before.size))
    _lib.check(sess.cache_append_rotated(cache, 0, x, k, v, ROWS, HEADS, turn, end, ld=ld, weights_ptr=weights), "beside")
    q, kk, vv = parts(t, HEADS, KV, DIM)
    got = read(sess, cache, KV, DIM)
    assert same(got[0], held(turned(kk, DIM, RMS, t["kw"], t["cos"], t["sin"], DIM, False), KV)) and same(got[1], held(vv, KV))
    got = room.download(np.float32, room.nbytes // 4)[ROWS * ld:][:ROWS * Q].reshape(ROWS, Q)
    assert same(got, turned(q, DIM, RMS, t["qw"], t["cos"], t["sin"], DIM, False))
    sess.cache_destroy(cache)
