"""pixhip_residual_norm_quantize refuses outputs that lie over a part of what it reads, and
takes those that lie beside it."""
import numpy as np
import pytest

from gpu_helpers import new_session
from pixelina_amd import _lib
from test_gpu_residual_norm import RMS, bits, definition, inputs

pytestmark = pytest.mark.gpu

ROWS, INNER = 5, 64
N = ROWS * INNER


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


def test_outputs_over_inputs(sess):
    t = inputs(ROWS, INNER)
    room = sess.alloc(4 * 8 * N)
    # stream, branch, a free block, the vectors, and room behind them
    held = np.concatenate([t["x"].reshape(-1), t["branch"].reshape(-1), np.full(N, 7, np.float32), t["post_weight"], t["pre_weight"], t["gate"].reshape(-1),
                           t["modulation"].reshape(-1), np.full(8 * N - 3 * N - 6 * INNER, 7, np.float32)])
    x, b, free, vectors = (room.ptr + 4 * N * i for i in range(4))
    behind = vectors + 4 * 6 * INNER
    names = dict(zip(("post_weight_ptr", "pre_weight_ptr", "gate_ptr", "gate_before_ptr", "modulation_ptr", "modulation_before_ptr"), range(vectors, behind, 4 * INNER)))

    def call(out, y):
        return sess.residual_norm_quantize(0, x, b, ROWS, INNER, out, y, post=RMS, pre=RMS, target_begin=2, **names)
    room.upload(held)
    for out, y in ((x + 4, behind), (x + 4 * INNER, behind), (b - 4, behind), (b + 4 * (N - 1), behind), (behind, x + 4), (behind, b + 16), (free, free + 4),
                   (behind, behind + 4 * (N - 1)), (free + 4, behind), (vectors - 4 * (N - 1), behind), (behind - 4, behind + 4 * N), (behind + 4 * N, free + 4),
                   (x, x + 4), *((p, behind) for p in names.values())):
        assert call(out, y) == _lib.ERR_ARGUMENT, (out - x, y - x)
    assert np.array_equal(bits(room.download(np.float32, held.size)), bits(held))
    want = definition(t, RMS, RMS, True, True, 2, 1.0)
    for out, y in ((free, behind), (x, behind), (b, free), (behind, x), (free, b), (x, b), (b, x)):
        room.upload(held)
        _lib.check(call(out, y), "residual_norm_quantize")
        got = room.download(np.float32, held.size)
        for p, value, bound in ((out, *want[:2]), (y, *want[2:])):
            assert (np.abs(got[(p - x) // 4:][:N].reshape(ROWS, INNER) - value) <= bound).all()
    room.free()
