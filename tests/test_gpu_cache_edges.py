"""The 8-bit key/value cache at the edges of its range: against the definition in
64 bits (test_gpu_cache.py), inputs on which running maxima, units or the
bookkeeping of a call could leave fp32's range or a row's own tokens.

The bound of `attend_terms`.  As test_gpu_cache.py's for the scores (e, natural
units) and the probabilities (2 e + 2^-17 relative, twice for the sum), but an
output is held to the sum of its own terms p_j |V_j|, and for each token to 2^-27 of
the largest term of its row: half of a probability's smallest digit is at most
that.  A probability below 2^-99 may count as zero, its token's term with it.
"""
import ctypes

import numpy as np
import pytest

from gpu_helpers import Pinned, new_session
from pixelina_amd import _lib
from test_gpu_cache import B, append, attend64, attention, held, read, rows_of, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


def attend_terms(q, k, v, heads, kv, causal=True):
    """(outputs, weights [n][kv], bound per output, bound per weight) of query rows over held keys and values."""
    rows, n = q.shape[0], k.shape[0]
    dim, group = q.shape[1] // heads, heads // kv
    q3, k3, v3 = (a.astype(np.float64).reshape(a.shape[0], -1, dim) for a in (q, k, v))
    out, bound = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim))
    w, wb = np.zeros((n, kv)), np.zeros((n, kv))
    for h in range(heads):
        kh, vh = k3[:, h // group], v3[:, h // group]
        s = q3[:, h] @ kh.T / np.sqrt(dim)
        hidden = np.arange(n)[None] > (n - rows + np.arange(rows) if causal else np.full(rows, n))[:, None]
        mag = np.where(hidden, 0, np.abs(q3[:, h]) @ np.abs(kh).T / np.sqrt(dim))
        peak = np.where(hidden, 0, np.abs(kh).max(axis=1)[None]).max(axis=1)
        e = ((dim + 8) * 2.0 ** -24 * mag.max(axis=1) + 2.0 ** -24 * dim * np.abs(q3[:, h]).max(axis=1) * peak / np.sqrt(dim))[:, None]
        s = np.where(hidden, -np.inf, s)
        p = np.exp(s - s.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        rel = 2 * (2 * e + 2.0 ** -17)
        out[:, h] = p @ vh
        bound[:, h] = rel * (p @ np.abs(vh)) + n * 2.0 ** -27 * (p * np.abs(vh).max(axis=1)[None]).max(axis=1, keepdims=True)
        bound[:, h] += np.where(p < 2.0 ** -99, p, 0) @ np.abs(vh) + 2.0 ** -125
        w[:, h // group] += p.sum(axis=0)
        wb[:, h // group] += (p * (rel + (rows * heads / kv + 2) * 2.0 ** -24)).sum(axis=0) + rows * 2.0 ** -125
    return out.reshape(rows, -1), w, bound.reshape(rows, -1), wb


def check(sess, k, v, q, heads, kv, causal=True, weigh=True):
    """One call on a cache of its own, outputs and weights within the bound; returns the outputs."""
    dim = k.shape[1] // kv
    cache = sess.cache(1, kv, dim, len(k))
    append(sess, cache, k, v)
    y = attention(sess, cache, q, heads, causal, weigh, 0.0)
    got = read(sess, cache, kv, dim)[2]
    sess.cache_destroy(cache)
    ref, w, bound, wb = attend_terms(q, held(k, kv), held(v, kv), heads, kv, causal)
    assert np.isfinite(y).all()
    print(f"  of the bound {(np.abs(y - ref) / bound).max():.2f}", flush=True)
    assert (np.abs(y - ref) <= bound).all()
    if weigh:
        assert np.isfinite(got).all()
        print(f"  weights: of the bound {(np.abs(got - w) / np.maximum(wb, 1e-300)).max():.2f}", flush=True)
        assert (np.abs(got - w) <= wb).all()
    return y


@pytest.mark.parametrize("gap", [60, 90, 110, 1000])
@pytest.mark.parametrize("rows,n,heads,kv,weigh", [
    (1, 300, 4, 1, False), (1, 300, 4, 1, True),       # few queries
    (300, 300, 1, 1, False), (300, 300, 1, 1, True),   # many, in pieces
    (40, 300, 1, 1, True),
    (1100, 1100, 16, 16, False),                       # many, in one piece
])
def test_zero_values_with_the_largest_scores(sess, rows, n, heads, kv, weigh, gap):
    """A block of values 0 whose scores lead the others' by up to 1000: what is left of the output is theirs, however small."""
    rng = np.random.default_rng(rows + n + gap)
    dim = 64
    k, v = rows_of(rng, n, kv, dim)
    q = rng.standard_normal((rows, heads * dim)).astype(np.float32)
    k[:, ::dim], q[:, ::dim] = 0, 8
    k[2 * B:3 * B, ::dim] = gap
    v[2 * B:3 * B] = 0
    v[B:2 * B] *= np.float32(2.0 ** -70)
    v[3 * B:5 * B] *= np.float32(2.0 ** 60)
    print(f"rows={rows} n={n} heads={heads}/{kv} weigh={weigh} gap={gap}", flush=True)
    check(sess, k, v, q, heads, kv, True, weigh)
