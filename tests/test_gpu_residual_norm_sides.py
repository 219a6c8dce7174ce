"""pixhip_residual_norm_quantize with rows of two sides into quantized activations: each
row's sum, norm, blocks and products of the next layer, bit for bit, are those of the
calls that it stands for with that side's gate and modulation, in the form of every
row length (rows of one to eight waves, vectors in LDS or not, a launch a side, the
longest)."""
import numpy as np
import pytest

from gpu_helpers import new_session
from pixelina_amd import Q5_K, Q8_0, _lib, synth
from test_gpu_residual_norm import LAYER, NONE, RMS, Call, bits, composed, inputs

pytestmark = pytest.mark.gpu

OUTPUTS = 64


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


def linear(sess, wtype, inner):
    w = (np.random.default_rng(inner).standard_normal((OUTPUTS, inner)) * 0.05).astype(np.float32)
    if wtype == Q5_K:
        return sess.weight(f"sides:k{inner}", synth.pack_q5_K(w), Q5_K, inner, OUTPUTS)
    from oracle_lib import oracle, quantize
    return sess.weight(f"sides:q{inner}", quantize(oracle(), "orc", w, "q8_0"), Q8_0, inner, OUTPUTS)


def multiplied(sess, h, rows):
    y = sess.alloc(4 * rows * OUTPUTS)
    _lib.check(sess.matmul_stage(h, None, rows, y.ptr, _lib.STAGE_MULTIPLY), "multiply")
    out = y.download(np.float32, rows * OUTPUTS).reshape(rows, OUTPUTS)
    y.free()
    return out


@pytest.mark.parametrize("wtype,rows,inner", [
    (Q8_0, 41, 544), (Q8_0, 19, 1536), (Q8_0, 300, 3840), (Q8_0, 21, 4096), (Q8_0, 17, 6144), (Q8_0, 9, 8192), (Q8_0, 9, 8224), (Q8_0, 300, 8224), (Q8_0, 5, 10272),
    (Q8_0, 3, 20480), (Q8_0, 3, 20512), (Q5_K, 41, 512), (Q5_K, 19, 1536), (Q5_K, 300, 3840), (Q5_K, 21, 4096), (Q5_K, 17, 6144), (Q5_K, 9, 8192), (Q5_K, 9, 8448),
    (Q5_K, 300, 8448), (Q5_K, 5, 10240), (Q5_K, 3, 20480), (Q5_K, 3, 20736)])
@pytest.mark.parametrize("post,pre", [(RMS, RMS), (LAYER, LAYER), (NONE, LAYER)])
def test_quantized_rows_of_two_sides(sess, wtype, rows, inner, post, pre):
    t = inputs(rows, inner, 23)
    h = linear(sess, wtype, inner)
    row = inner // 32 * 34 if wtype == Q8_0 else inner // 256 * 292
    want = []
    for side in (0, 1):
        c = Call(sess, t)
        for k in ("gate", "modulation"):
            c.p[k] += 4 * inner * side
        blocks = sess.alloc(rows * row)
        x, y = composed(c, post, pre, True, True, wtype, blocks.ptr)
        want.append((bits(x), bits(y), blocks.download(np.uint8, rows * row).reshape(rows, row), bits(multiplied(sess, h, rows))))
        blocks.free()
        c.free()
    for split, shift in ((1, 0), (rows // 2, 4), (rows - 1, 0), (rows, 0)):
        c = Call(sess, t, shift)
        blocks = sess.to_device(np.full(rows * row + 64, 9, np.uint8))
        _lib.check(c.run(post, pre, True, True, split, wtype=wtype, blocks=blocks.ptr), "residual_norm_quantize")
        held = blocks.download(np.uint8, rows * row + 64)
        assert (held[rows * row:] == 9).all()
        got = bits(c.get(c.out)), bits(c.get(c.y)), held[:rows * row].reshape(rows, row), bits(multiplied(sess, h, rows))
        for mine, after, before in zip(got, *want):
            assert np.array_equal(mine[:split], before[:split]) and np.array_equal(mine[split:], after[split:])
        # quantized alone
        _lib.check(c.run(post, pre, True, True, split, wtype=wtype, want_y=False), "residual_norm_quantize")
        assert np.array_equal(bits(multiplied(sess, h, rows)), got[3])
        blocks.free()
        c.free()
