"""Adapters of many rows in every form that takes them: tiles of rows in twos in the first
launch (4096 rows of 256 CUs and more) with up to 16, 32, 64, 128 and 256 ranks; in the
second groups of four tiles, where rows / 64 times outputs / 32 is 64 per CU and more and
no rank is above 128, or of two; results stored around the caches, whose rows are whole
lines of 128 bytes and 4 MB and more in all, or through them."""
import numpy as np
import pytest

from gpu_helpers import new_session
from test_gpu_adapters import BF16, F16, F32, Adapter, check, data, definition, run

pytestmark = pytest.mark.gpu

CUS = 256
ROWS = 16 * CUS + 512


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


def ranges(rng, sess, wtype, rank, inner, rows):
    """Two adapters over requests of unequal length, rows of none between them."""
    a, b = Adapter(sess, rng, wtype, rank, inner, rows), Adapter(sess, rng, wtype, max(1, rank // 3), inner, rows)
    return a, b, [(0, 37, b, 1.0), (37, 2100, a, 0.5), (2111, ROWS - 3, a, -1.0), (ROWS - 3, ROWS, b, 2.0)]


@pytest.mark.parametrize("wtype", [F32, F16, BF16])
@pytest.mark.parametrize("rank,inner,rows,fours,lines", [
    (7, 96, 7680, True, True), (20, 130, 7680, True, True), (64, 96, 7680, True, True), (128, 70, 7680, True, True), (64, 97, 7679, True, False),
    (16, 200, 512, False, True), (40, 96, 1024, False, True), (100, 64, 544, False, True), (256, 96, 512, False, True), (33, 61, 515, False, False)])
def test_forms(sess, wtype, rank, inner, rows, fours, lines):
    assert (rank <= 128 and ROWS // 64 * -(-rows // 32) >= 64 * CUS) == fours and (rows % 32 == 0 and 4 * ROWS * rows >= 4 << 20) == lines
    rng, x, base = data(rank, ROWS, inner, rows)
    a, b, all_ranges = ranges(rng, sess, wtype, rank, inner, rows)
    want = definition(x, base, all_ranges)
    first = run(sess, x, base, all_ranges, rows)
    check(first, want)
    none = np.r_[2100:2111]
    assert np.array_equal(first[none].view(np.uint32), base[none].view(np.uint32))
    assert np.array_equal(run(sess, x, base, all_ranges, rows, "in place").view(np.uint32), first.view(np.uint32))
    a.free()
    b.free()
