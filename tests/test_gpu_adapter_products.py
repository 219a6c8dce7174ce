"""Single products of an adapter's values against 64 bits: what the splits in bf16
planes leave out, on its own.

The bound, relative to a product x w of leading bits' values of 1.  BF16 weights leave
out nothing, F16 weights the third plane of x times the second of w.  A second plane is
below 2^-7 where the first is cut off and at most 2^-8 where it is rounded, the third then at
most 2^-16 where the second alone is rounded and 2^-17 where both are; of the first matrix
w's first plane and x's second are rounded, of the second one x's first two: 2^-24.  F32
weights, with all planes rounded, leave out 2 * 2^-25 + 2^-34.  The sums that join the
products: up to five before the last, of at most 2^-6 of the product (2^-7 and 2^-8 for the
second planes) and off by a step, 2^-23, each (whichever way a matrix instruction rounds),
the last by a step of the whole; the other of the two matrices is ones, whose products and
sums are exact.
"""
import numpy as np
import pytest

from gpu_helpers import new_session
from pixelina_amd import _lib
from test_gpu_adapters import BF16, F16, F32, Adapter, run, stored

pytestmark = pytest.mark.gpu

SUMS = 2.0 ** -23 * (1 + 5 * 2.0 ** -6)
LEFT_OUT = {F32: 2.0 ** -24 + 2.0 ** -34, F16: 2.0 ** -24, BF16: 0.0}
# the most that planes cut off instead of rounded leave out, and what lies about the ends of a plane
MANTISSAS = np.array([0x3f80ffff, 0x3f80e000, 0x3f80e001, 0x3f808000, 0x3f807fff, 0x3f818000, 0x3f818001, 0x3fffffff, 0x3f800001, 0x3f80ff80, 0x3f80ff81,
                      0x3f80007f, 0x3f800080, 0x3f7fffff], np.uint32).view(np.float32)


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


def mantissas(rng, n):
    v = (rng.integers(0, 1 << 23, n).astype(np.uint32) | np.uint32(0x3f800000)).view(np.float32)
    v[:len(MANTISSAS)] = MANTISSAS
    return v * rng.choice(np.array([1, -1], np.float32), n)


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("inner", [1, 4096])
def test_products_of_the_first_matrix(sess, wtype, inner):
    """In one launch, and (of a long inner size) in two."""
    rng, cols, rank, at = np.random.default_rng(5), 300, 256, inner // 3
    x, down = np.zeros((cols, inner), np.float32), np.zeros((rank, inner), np.float32)
    x[:, at], down[:, at] = mantissas(rng, cols), mantissas(rng, rank)
    down[len(MANTISSAS), at] = 1 + 7 * 2.0 ** -10
    a = Adapter(sess, rng, wtype, rank, inner, rank, down, np.eye(rank, dtype=np.float32))
    y = run(sess, x, np.zeros((cols, rank), np.float32), [(0, cols, a, 1.0)], rank, "zero")
    a.free()
    want = np.outer(x[:, at].astype(np.float64), a.down[:, at].astype(np.float64))
    assert (np.abs(y - want) <= (LEFT_OUT[wtype] + SUMS) * np.abs(want)).all()


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("inner,cols", [(1, 300), (2048, 300), (40, 2300)])
def test_products_of_the_second_matrix(sess, wtype, inner, cols):
    rng, rows = np.random.default_rng(6), 600
    x, up = np.zeros((cols, inner), np.float32), mantissas(rng, rows)[:, None]
    x[:, inner // 2] = mantissas(rng, cols)
    up[len(MANTISSAS)] = 1 + 7 * 2.0 ** -10
    a = Adapter(sess, rng, wtype, 1, inner, rows, np.ones((1, inner), np.float32), up)
    y = run(sess, x, np.zeros((cols, rows), np.float32), [(0, cols, a, 1.0)], rows, "zero")
    a.free()
    want = np.outer(x[:, inner // 2].astype(np.float64), a.up[:, 0].astype(np.float64))
    assert (np.abs(y - want) <= (LEFT_OUT[wtype] + SUMS) * np.abs(want)).all()


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("inner", [3, 2048])
def test_values_next_to_the_largest(sess, wtype, inner):
    """Values that rounded to bf16 would be infinite, as rows, as sums and as weights; selections give them whole."""
    rng, rows, cols = np.random.default_rng(7), 40, 20
    big = np.array([0x7f7fffff, 0x7f7f8000, 0x7f7f7fff, 0x7f7f8001, 0x7f7fff80], np.uint32).view(np.float32)
    x, ones = np.zeros((cols, inner), np.float32), np.ones((1, inner), np.float32)
    x[:, inner - 1] = np.resize(np.concatenate([big, -big]), cols)
    zeros = np.zeros((cols, rows), np.float32)
    scale = np.linspace(-1, 1, rows, dtype=np.float32)[:, None]
    scale[:4, 0] = 1, -1, 0.5, 0
    a = Adapter(sess, rng, wtype, 1, inner, rows, ones, scale)
    y = run(sess, x, zeros, [(0, cols, a, 1.0)], rows, "zero")
    a.free()
    want = np.outer(x[:, inner - 1].astype(np.float64), a.up[:, 0].astype(np.float64))
    assert np.array_equal(y[:, :4], want[:, :4].astype(np.float32))
    # (x is within 2^-8 of 2^128: where its first plane is the largest bf16, the second is at most 2^-8 of x too,
    # and the third 2^-17)
    assert (np.abs(y - want) <= (LEFT_OUT[wtype] + SUMS) * np.abs(want)).all()
    if wtype == F16:
        return
    # the matrices' own; a bf16 value is its first plane, with the largest of bf16 the end
    ends = big if wtype == F32 else np.array([0x7f7f0000], np.uint32).view(np.float32)
    for matrix in ("down", "up"):
        down, up = np.zeros((4, inner), np.float32), np.zeros((rows, 4), np.float32)
        down[:, inner - 1], up[np.arange(rows), np.arange(rows) % 4] = 1, 1
        if matrix == "down":
            down[:, inner - 1] = np.resize(ends, 4)
        else:
            up[np.arange(rows), np.arange(rows) % 4] = np.resize(ends, rows)
        a = Adapter(sess, rng, wtype, 4, inner, rows, down, up)
        x[:, inner - 1] = np.resize([1, -1, 0.5], cols)
        y = run(sess, x, zeros, [(0, cols, a, 1.0)], rows, "zero")
        a.free()
        assert np.array_equal(y, ((x.astype(np.float64) @ a.down.astype(np.float64).T) @ a.up.astype(np.float64).T).astype(np.float32))


def test_weights_that_are_infinite_or_nan(sess):
    """An output whose weights hold one is not finite; the other outputs are as they were."""
    rng, inner, rows, cols = np.random.default_rng(8), 50, 70, 18
    x = rng.standard_normal((cols, inner)).astype(np.float32)
    for wtype in (F32, F16, BF16):
        down, up = rng.standard_normal((5, inner)).astype(np.float32), rng.standard_normal((rows, 5)).astype(np.float32)
        up[7, 2], up[33, 4], up[69, 0] = np.inf, np.nan, -np.inf
        a = Adapter(sess, rng, wtype, 5, inner, rows, down, up)
        y = run(sess, x, np.zeros((cols, rows), np.float32), [(0, cols, a, 1.0)], rows, "zero")
        a.free()
        bad = np.isin(np.arange(rows), (7, 33, 69))
        assert not np.isfinite(y[:, bad]).any() and np.isfinite(y[:, ~bad]).all()
        up = stored(rng.standard_normal((rows, 5)), wtype)[1]
        down[3, 20] = -np.inf
        a = Adapter(sess, rng, wtype, 5, inner, rows, down, up)
        assert not np.isfinite(run(sess, x, np.zeros((cols, rows), np.float32), [(0, cols, a, 1.0)], rows, "zero")).any()
        a.free()
