"""The 8-bit key/value cache (pixhip_cache_*) through the C ABI against its
definition in 64 bits (numpy): what a cache holds bit for bit (codes, scales,
eviction, forks), attention over it within a bound taken from its arithmetic.

Attention's bound.  A query is held to 2^-24 of its largest value and a score is
an fp32 sum of `dim` products, so a score (natural units) is off by at most
  e = (dim + 8) * 2^-24 * max_j sum_d |q_d| |K_jd| / sqrt(dim) + 2^-24 * dim * max|q| max|K| / sqrt(dim);
a probability then by 2 e + 2^-17 relative (exp2 and its argument, the sum, the
merges: together under 64 roundings of 2^-23), and an output by that times the
largest |V| of the head, counted twice for the sum over the probabilities.
"""
import ctypes

import numpy as np
import pytest

from gpu_helpers import Pinned, new_session
from pixelina_amd import _lib

pytestmark = pytest.mark.gpu

B = 32


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


# ---- the definition ----

def held(x, kv):
    """What a cache holds of rows x [n][kv * dim] (fp32): values as code * s in fp32."""
    n, ch = x.shape
    dim = ch // kv
    nb = -(-n // B)
    p = np.zeros((nb * B, ch), np.float32)
    p[:n] = x
    p = p.reshape(nb, B, kv, dim)
    fin = np.where(np.isfinite(p), np.abs(p), np.float32(0))
    s = (fin.max(axis=(1, 3)) / np.float32(127)).astype(np.float32)
    s[s < np.float32(2.0 ** -100)] = 0
    s4 = s[:, None, :, None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(s4 > 0, np.rint(np.where(np.isfinite(p), p, 0).astype(np.float64) / np.where(s4 > 0, s4, 1).astype(np.float64)), 0.0)
    q = np.where(np.isposinf(p) & (s4 > 0), 127.0, np.where(np.isneginf(p) & (s4 > 0), -127.0, q))
    return (q.astype(np.int8).astype(np.float32) * s4).reshape(nb * B, ch)[:n]


def attend64(q, k, v, heads, kv, causal=True, k_dim=None):
    """(outputs, weights [n][kv], bound per row) of query rows over held keys and values."""
    rows, n = q.shape[0], k.shape[0]
    dim, group = q.shape[1] // heads, heads // kv
    q3, k3, v3 = (a.astype(np.float64).reshape(a.shape[0], -1, dim) for a in (q, k, v))
    out, bound = np.zeros((rows, heads, dim)), np.zeros((rows, heads, 1))
    w, wb = np.zeros((n, kv)), np.zeros((n, kv))
    for h in range(heads):
        kh, vh = k3[:, h // group], v3[:, h // group]
        s = q3[:, h] @ kh.T / np.sqrt(dim)
        mag = np.abs(q3[:, h]) @ np.abs(kh).T / np.sqrt(dim)
        e = ((dim + 8) * 2.0 ** -24 * mag.max(axis=1) +
             2.0 ** -24 * dim * np.abs(q3[:, h]).max(axis=1) * np.abs(kh).max() / np.sqrt(dim))[:, None]
        if causal:
            s = np.where(np.arange(n)[None] > (n - rows + np.arange(rows))[:, None], -np.inf, s)
        p = np.exp(s - s.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        out[:, h] = p @ vh
        bound[:, h] = 2 * (2 * e + 2.0 ** -17) * np.abs(vh).max()
        w[:, h // group] += p.sum(axis=0)
        wb[:, h // group] += (p * 2 * (2 * e + 2.0 ** -17)).sum(axis=0)
    return out.reshape(rows, -1), w, np.broadcast_to(bound, out.shape).reshape(rows, -1), wb


# ---- calls ----

def append(sess, cache, k, v, layer=0, weights=None):
    kb, vb = sess.to_device(np.ascontiguousarray(k, np.float32)), sess.to_device(np.ascontiguousarray(v, np.float32))
    wb = sess.to_device(np.ascontiguousarray(weights, np.float32)) if weights is not None else None
    _lib.check(sess.cache_append(cache, layer, kb.ptr, vb.ptr, k.shape[0], 0, wb.ptr if wb else None), "append")
    for b in (kb, vb, wb):
        if b:
            b.free()


def read(sess, cache, kv, dim, first=0, rows=None, layer=0):
    rows = sess.cache_length(cache, layer) - first if rows is None else rows
    kb, vb, wb = sess.alloc(rows * kv * dim * 4), sess.alloc(rows * kv * dim * 4), sess.alloc(rows * kv * 4)
    _lib.check(sess.cache_read(cache, layer, first, rows, kb.ptr, vb.ptr, wb.ptr), "read")
    out = [b.download(np.float32, rows * c).reshape(rows, c) for b, c in ((kb, kv * dim), (vb, kv * dim), (wb, kv))]
    for b in (kb, vb, wb):
        b.free()
    return out


def attention(sess, cache, q, heads, causal=True, weigh=False, decay=1.0, layer=0):
    qb, ob = sess.to_device(np.ascontiguousarray(q, np.float32)), sess.to_device(np.full(q.shape, 7.0, np.float32))
    _lib.check(sess.cache_attention(cache, layer, qb.ptr, q.shape[0], heads, ob.ptr, 0, causal, weigh, decay), "attention")
    y = ob.download(np.float32, q.size).reshape(q.shape)
    qb.free()
    ob.free()
    return y


def evict(sess, cache, kv, keep, recent, layer=0):
    nb = -(-sess.cache_length(cache, layer) // B)
    n = min(keep, nb)
    kb = sess.to_device(np.full(kv * n + 8, -7, np.int32))
    _lib.check(sess.cache_evict(cache, layer, keep, recent, kb.ptr), "evict")
    out = kb.download(np.int32, kv * n + 8)
    kb.free()
    assert (out[kv * n:] == -7).all()
    return out[:kv * n].reshape(kv, n)


def same(a, b):
    return np.array_equal(np.ascontiguousarray(a).view(np.uint32), np.ascontiguousarray(b).view(np.uint32))


def rows_of(rng, n, kv, dim):
    k = rng.standard_normal((n, kv * dim)) * np.exp(0.5 * rng.standard_normal(kv * dim))
    return k.astype(np.float32), rng.standard_normal((n, kv * dim)).astype(np.float32)


# ---- what a cache holds ----

@pytest.mark.parametrize("n,kv,dim", [(1, 1, 1), (31, 3, 30), (32, 2, 64), (33, 8, 128), (100, 1, 80), (257, 5, 65), (64, 4, 4), (70, 7, 127)])
def test_append_and_read(sess, n, kv, dim):
    rng = np.random.default_rng(n * 131 + dim)
    k, v = rows_of(rng, n, kv, dim)
    print(f"n={n} kv={kv} dim={dim}", flush=True)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v)
    gk, gv, gw = read(sess, cache, kv, dim)
    assert same(gk, held(k, kv)) and same(gv, held(v, kv)) and not gw.any()
    if n > 2:
        pk, pv, _ = read(sess, cache, kv, dim, 1, n - 2)
        assert same(pk, gk[1:-1]) and same(pv, gv[1:-1])
    sess.cache_destroy(cache)


@pytest.mark.parametrize("cuts", [[1] * 70, [31, 2, 37], [32, 32, 6], [5, 60, 5], [33, 37], [64, 1, 5]])
def test_the_cuts_of_the_rows_do_not_matter(sess, cuts):
    rng = np.random.default_rng(7)
    kv, dim, n = 2, 80, sum(cuts)
    k, v = rows_of(rng, n, kv, dim)
    k *= np.exp(rng.standard_normal((n, 1))).astype(np.float32)  # the open block's scale grows again and again
    cache = sess.cache(1, kv, dim, n)
    at = 0
    for c in cuts:
        append(sess, cache, k[at:at + c], v[at:at + c])
        at += c
    gk, gv, _ = read(sess, cache, kv, dim)
    assert same(gk, held(k, kv)) and same(gv, held(v, kv))
    sess.cache_destroy(cache)


def test_values_at_the_edges(sess):
    """Ties between codes, zeros, subnormals, the smallest kept scale, the largest finite value, infinities and NaN."""
    kv, dim = 1, 64
    x = np.zeros((5 * B, dim), np.float32)
    x[0] = (np.arange(dim) - 31.5).astype(np.float32)       # scale 1: every value is a tie
    x[1, 0] = 127.0
    x[B:2 * B] = np.float32(1e-42)                           # a block of subnormals
    x[2 * B, :4] = [2.0 ** -93, -2.0 ** -94, 2.0 ** -100, 0]  # just above the smallest scale
    x[3 * B, :6] = [np.inf, -np.inf, np.nan, 2.0, -1.0, 3.4028235e38 / 4]
    x[4 * B, :3] = [np.inf, np.nan, -np.inf]                 # no finite value but zeros
    cache = sess.cache(1, kv, dim, len(x))
    append(sess, cache, x, -x)
    gk, gv, _ = read(sess, cache, kv, dim)
    assert same(gk, held(x, kv)) and same(gv, held(-x, kv))
    assert np.isfinite(gk).all() and not gk[4 * B:].any() and not gk[B:2 * B].any()
    sess.cache_destroy(cache)


def test_strided_rows_and_host_rows(sess):
    """Keys and values as slices of one projection's output; the same from pinned and from pageable memory; a misaligned tensor."""
    rng = np.random.default_rng(3)
    n, kv, dim = 45, 2, 40
    ch = kv * dim
    fused = rng.standard_normal((n, 3 * ch + 5)).astype(np.float32)
    k, v = np.ascontiguousarray(fused[:, ch:2 * ch]), np.ascontiguousarray(fused[:, 2 * ch:3 * ch])
    fb = sess.to_device(fused)
    cache = sess.cache(4, kv, dim, n)
    _lib.check(sess.cache_append(cache, 0, fb.ptr + 4 * ch, fb.ptr + 8 * ch, n, 3 * ch + 5), "append")
    _lib.check(sess.cache_append(cache, 1, k.ctypes.data, v.ctypes.data, n), "append")
    hk, hv = Pinned(sess, k), Pinned(sess, v)
    _lib.check(sess.cache_append(cache, 2, hk.p.value, hv.p.value, n), "append")
    odd = sess.alloc(4 + k.nbytes)
    odd.upload(k, 4)
    _lib.check(sess.cache_append(cache, 3, odd.ptr + 4, odd.ptr + 4, n), "append")
    for layer in range(3):
        gk, gv, _ = read(sess, cache, kv, dim, layer=layer)
        assert same(gk, held(k, kv)) and same(gv, held(v, kv)), layer
    gk, gv, _ = read(sess, cache, kv, dim, layer=3)
    assert same(gk, held(k, kv)) and same(gv, held(k, kv))
    # a misaligned and a pinned destination
    _lib.check(sess.cache_read(cache, 0, 0, n, odd.ptr + 4, hv.p.value), "read")
    assert same(odd.download(np.float32, n * ch, 4).reshape(n, ch), held(k, kv))
    assert same(hv.read(np.float32, (n, ch)), held(v, kv))
    for b in (fb, odd):
        b.free()
    hk.free()
    hv.free()
    sess.cache_destroy(cache)


def test_rows_behind_the_last_are_left(sess):
    """A layer's calls touch neither the other layers nor, on reading, what lies behind the destination."""
    rng = np.random.default_rng(4)
    kv, dim = 3, 64
    k, v = rows_of(rng, 40, kv, dim)
    cache = sess.cache(3, kv, dim, 64)
    for layer in range(3):
        append(sess, cache, k + layer, v - layer, layer)
    append(sess, cache, k[:9], v[:9], 1)
    for layer in (0, 2):
        gk, gv, _ = read(sess, cache, kv, dim, layer=layer)
        assert same(gk, held(k + layer, kv)) and same(gv, held(v - layer, kv))
    buf = sess.to_device(np.full(10 * kv * dim + 16, 5.0, np.float32))
    _lib.check(sess.cache_read(cache, 0, 7, 10, buf.ptr), "read")
    got = buf.download(np.float32, 10 * kv * dim + 16)
    assert (got[10 * kv * dim:] == 5.0).all() and same(got[:10 * kv * dim].reshape(10, -1), held(k, kv)[7:17])
    buf.free()
    sess.cache_destroy(cache)


def test_truncate(sess):
    """Back to where the last append began, and within the open block: as if the rows had never come.  Further back: the
    rows left in the block count as the values they were held as."""
    rng = np.random.default_rng(5)
    kv, dim = 2, 128
    k, v = rows_of(rng, 150, kv, dim)
    cache = sess.cache(1, kv, dim, 200)
    append(sess, cache, k[:77], v[:77])
    for again in range(2):
        append(sess, cache, k[77:], v[77:])
        _lib.check(sess.cache_truncate(cache, 0, 77), "truncate")
        assert sess.cache_length(cache, 0) == 77
        append(sess, cache, v[:50], k[:50])
        gk, _, _ = read(sess, cache, kv, dim)
        assert same(gk, held(np.concatenate([k[:77], v[:50]]), kv))
        _lib.check(sess.cache_truncate(cache, 0, 77), "truncate")
    append(sess, cache, k[77:90], v[77:90])
    _lib.check(sess.cache_truncate(cache, 0, 80), "truncate")  # inside the open block
    append(sess, cache, k[80:], v[80:])
    gk, gv, _ = read(sess, cache, kv, dim)
    assert same(gk, held(k, kv)) and same(gv, held(v, kv))
    _lib.check(sess.cache_truncate(cache, 0, 40), "truncate")  # a block that was full long ago
    append(sess, cache, v[:3], k[:3])
    gk, gv, _ = read(sess, cache, kv, dim)
    assert same(gk, held(np.concatenate([k[:32], held(k, kv)[32:40], v[:3]]), kv))
    assert same(gv, held(np.concatenate([v[:32], held(v, kv)[32:40], k[:3]]), kv))
    _lib.check(sess.cache_truncate(cache, 0, 0), "truncate")
    append(sess, cache, k[:5], v[:5])
    assert same(read(sess, cache, kv, dim)[0], held(k[:5], kv))
    sess.cache_destroy(cache)


# ---- attention ----

@pytest.mark.parametrize("rows,n,heads,kv,dim,causal", [
    (1, 1, 1, 1, 1, True),           # one key, one dim
    (1, 1, 8, 2, 128, True),
    (1, 31, 4, 4, 64, True),         # less than a block
    (1, 33, 28, 4, 128, True),       # one row past it, seven heads per kv head
    (1, 64, 5, 1, 80, True),         # five heads per kv head
    (1, 65, 3, 3, 30, True),
    (1, 2501, 32, 8, 128, True),     # a decode step
    (1, 9000, 16, 2, 64, True),      # many key pieces, eight heads per kv head
    (2, 130, 6, 2, 96, True),
    (3, 3, 4, 2, 128, True),         # the first rows of a sequence: the first sees itself alone
    (5, 700, 40, 4, 72, True),       # 50 queries per kv head
    (7, 95, 2, 1, 4, False),
    (9, 5, 4, 2, 128, False),        # more rows than keys
    (16, 300, 8, 8, 128, True),
    (17, 320, 8, 8, 65, True),
    (33, 33, 2, 1, 127, True),
    (128, 1281, 32, 8, 128, True),   # a chunk of a prefill
    (128, 128, 4, 1, 64, True),
    (130, 515, 7, 7, 128, False),
    (200, 777, 10, 2, 80, True),
    (300, 2000, 1, 1, 128, True),
])
@pytest.mark.parametrize("weigh", [False, True])
def test_attention(sess, rows, n, heads, kv, dim, causal, weigh):
    rng = np.random.default_rng(rows * 31 + n + dim)
    k, v = rows_of(rng, n, kv, dim)
    q = (1.3 * rng.standard_normal((rows, heads * dim))).astype(np.float32)
    print(f"rows={rows} n={n} heads={heads}/{kv} dim={dim} causal={causal} weigh={weigh}", flush=True)
    cache = sess.cache(1, kv, dim, n)
    old = rng.random((n, kv)).astype(np.float32)
    append(sess, cache, k, v, weights=old)
    y = attention(sess, cache, q, heads, causal, weigh, 0.5)
    ref, w, bound, wb = attend64(q, held(k, kv), held(v, kv), heads, kv, causal)
    err = np.abs(y - ref)
    print(f"  rel={np.linalg.norm(y - ref) / np.linalg.norm(ref):.2e} of the bound {(err / bound).max():.2f}", flush=True)
    assert (err <= bound).all()
    gk, gv, gw = read(sess, cache, kv, dim)
    assert same(gk, held(k, kv)) and same(gv, held(v, kv))
    if weigh:
        off = np.abs(gw - (w + 0.5 * old))
        print(f"  weights: of the bound {(off / (wb + 2.0 ** -22 * (w + old))).max():.2f}", flush=True)
        assert (off <= wb + 2.0 ** -22 * (w + old) + 2.0 ** -100).all()
    else:
        assert same(gw, old)
    # the same bits again (decay 0: what the weights were does not matter)
    assert same(attention(sess, cache, q, heads, causal, weigh, 0.0), y)
    first = read(sess, cache, kv, dim)[2]
    assert same(attention(sess, cache, q, heads, causal, weigh, 0.0), y)
    assert same(read(sess, cache, kv, dim)[2], first)
    sess.cache_destroy(cache)


@pytest.mark.parametrize("rows,n", [(1, 300), (4, 300), (70, 300)])
def test_blocks_of_very_different_scales(sess, rows, n):
    """Value blocks from 2^-80 to 2^80, one of zeros, keys of one block of zeros: a row's output is held to its own
    largest terms, and the first rows see the small blocks alone."""
    rng = np.random.default_rng(n + rows)
    kv, dim, heads = 1, 64, 4
    k, v = rows_of(rng, n, kv, dim)
    for b, e in enumerate((-80, -60, 0, 20, -5, 60, 80, 3, 0, 0)):
        v[b * B:(b + 1) * B] *= np.float32(2.0 ** e)
    v[2 * B:3 * B] = 0
    k[4 * B:5 * B] = 0
    q = rng.standard_normal((rows, heads * dim)).astype(np.float32)
    cache = sess.cache(1, kv, dim, n)
    for seen in (32, 64, 100, 200, 300):
        if seen < rows:
            continue
        _lib.check(sess.cache_truncate(cache, 0, 0), "truncate")
        append(sess, cache, k[:seen], v[:seen])
        y = attention(sess, cache, q, heads)
        hk, hv = held(k[:seen], kv), held(v[:seen], kv)
        ref, _, bound, _ = attend64(q, hk, hv, heads, kv)
        print(f"rows={rows} seen={seen}: of the bound {(np.abs(y - ref) / bound).max():.2f}", flush=True)
        assert (np.abs(y - ref) <= bound).all()
    sess.cache_destroy(cache)


@pytest.mark.parametrize("rows", [1, 3, 70])
def test_large_scores_and_zero_queries(sess, rows):
    """Scores in the thousands (one key takes all), a query of zeros (equal probabilities), tiny queries."""
    rng = np.random.default_rng(rows)
    n, kv, dim, heads = 200, 2, 128, 6
    k, v = rows_of(rng, n, kv, dim)
    q = rng.standard_normal((rows, heads * dim)).astype(np.float32)
    q[:, :dim] *= 300
    q[:, dim:2 * dim] = 0
    q[:, 2 * dim:3 * dim] *= np.float32(1e-30)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v)
    y = attention(sess, cache, q, heads)
    ref, _, bound, _ = attend64(q, held(k, kv), held(v, kv), heads, kv)
    print(f"of the bound {(np.abs(y - ref) / bound).max():.2f}", flush=True)
    assert (np.abs(y - ref) <= bound).all()
    sess.cache_destroy(cache)


@pytest.mark.parametrize("rows,n", [(1, 70), (4, 70), (70, 140)])
def test_not_a_number_in_a_query(sess, rows, n):
    """A query row with NaN or an infinity gives NaN for its head and touches no other output; NaN in the rows behind
    those a query sees, or in the workspace of an earlier call, does not reach it."""
    rng = np.random.default_rng(n)
    kv, dim, heads = 2, 64, 4
    k, v = rows_of(rng, n, kv, dim)
    q = rng.standard_normal((rows, heads * dim)).astype(np.float32)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v)
    clean = attention(sess, cache, q, heads)
    bad = q.copy()
    bad[0, 3] = np.nan
    bad[rows - 1, 2 * dim + 5] = np.inf
    y = attention(sess, cache, bad, heads)
    spoiled = np.zeros_like(y, bool)
    spoiled[0, :dim] = True
    spoiled[rows - 1, 2 * dim:3 * dim] = True
    assert np.isnan(y[spoiled]).all() and same(y[~spoiled], clean[~spoiled])
    assert same(attention(sess, cache, q, heads), clean)
    sess.cache_destroy(cache)


@pytest.mark.parametrize("rows,n,heads", [(1, 128, 64), (2, 100, 64), (256, 128, 8), (600, 97, 4)])
def test_each_probability(sess, rows, n, heads):
    """Values that are 1 at the token's own dim and 0 elsewhere give back the probabilities: each within the bound of its
    own size, down to 2^-24 of the largest (what lies below a row's smallest digit or half counts as 2^-24 of it)."""
    rng = np.random.default_rng(rows + n)
    kv, dim = 1, 128
    k, _ = rows_of(rng, n, kv, dim)
    v = np.zeros((n, dim), np.float32)
    v[np.arange(n), np.arange(n)] = 1
    q = (1.2 * rng.standard_normal((rows, heads * dim))).astype(np.float32)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v)
    y = attention(sess, cache, q, heads, False).reshape(rows * heads, dim)[:, :n]
    ref, _, bound, _ = attend64(q, held(k, kv), held(v, kv), heads, kv, False)
    ref, bound = ref.reshape(rows * heads, dim)[:, :n], bound.reshape(rows * heads, dim)[:, :n]  # (largest |V| is 1)
    limit = bound * ref + 2.0 ** -24 * ref.max(axis=1, keepdims=True)
    print(f"of the bound {(np.abs(y - ref) / limit).max():.2f}", flush=True)
    assert (np.abs(y - ref) <= limit).all()
    sess.cache_destroy(cache)


def test_strided_queries_and_host_queries(sess):
    rng = np.random.default_rng(12)
    n, kv, dim, heads, rows = 90, 2, 36, 4, 3
    ch = heads * dim
    k, v = rows_of(rng, n, kv, dim)
    fused = rng.standard_normal((rows, ch + 11)).astype(np.float32)
    q = np.ascontiguousarray(fused[:, 3:3 + ch])
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v)
    want = attention(sess, cache, q, heads)
    fb, ob = sess.to_device(fused), sess.alloc(q.nbytes + 4)
    _lib.check(sess.cache_attention(cache, 0, fb.ptr + 12, rows, heads, ob.ptr + 4, ch + 11), "attention")
    assert same(ob.download(np.float32, rows * ch, 4).reshape(rows, ch), want)
    _lib.check(sess.cache_attention(cache, 0, q.ctypes.data, rows, heads, ob.ptr), "attention")
    assert same(ob.download(np.float32, rows * ch).reshape(rows, ch), want)
    hq, ho = Pinned(sess, q), Pinned(sess, np.zeros_like(q))
    _lib.check(sess.cache_attention(cache, 0, hq.p.value, rows, heads, ho.p.value), "attention")
    sess.synchronize()
    assert same(ho.read(np.float32, q.shape), want)
    hq.free()
    ho.free()
    for b in (fb, ob):
        b.free()
    sess.cache_destroy(cache)


# ---- eviction and forks ----

def evict_rule(w, keep, recent):
    """The rule in plain form: kept blocks per head of weights w [n][kv] (sums in 64 bits)."""
    n, kv = w.shape
    nb = -(-n // B)
    keep = min(keep, nb)
    recent = min(recent, keep)
    out = []
    for h in range(kv):
        sums = [w[b * B:(b + 1) * B, h].astype(np.float64).sum() for b in range(nb)]
        order = sorted(range(nb - recent), key=lambda b: (not np.isnan(sums[b]), sums[b], -b), reverse=True)
        out.append(sorted(order[:keep - recent]) + list(range(nb - recent, nb)))
    return np.array(out, np.int32)


def chosen(x, kept, n, kv):
    """Rows of x [n][kv * c] that stay."""
    c = x.shape[1] // kv
    left = [b * B + t for b in kept[0] for t in range(B) if b * B + t < n]
    out = np.empty((len(left), kv * c), x.dtype)
    for h in range(kv):
        at = [b * B + t for b in kept[h] for t in range(B) if b * B + t < n]
        out[:, h * c:(h + 1) * c] = x[at, h * c:(h + 1) * c]
    return out


@pytest.mark.parametrize("n,kv,dim,keep,recent", [
    (1, 1, 64, 1, 1), (33, 2, 64, 1, 1), (64, 1, 4, 2, 2), (65, 3, 30, 2, 1), (300, 2, 128, 10, 3), (300, 2, 128, 4, 4),
    (1000, 8, 128, 20, 1), (4099, 4, 64, 60, 9), (40000, 1, 8, 1000, 50), (70000, 2, 4, 2100, 100), (140000, 1, 4, 1500, 7), (320, 2, 64, 50, 3),
])
def test_evict(sess, n, kv, dim, keep, recent):
    rng = np.random.default_rng(n + keep)
    k, v = rows_of(rng, n, kv, dim)
    w = np.exp(2 * rng.standard_normal((n, kv))).astype(np.float32)
    cache = sess.cache(1, kv, dim, n + 100)
    append(sess, cache, k, v, weights=w)
    print(f"n={n} kv={kv} dim={dim} keep={keep} recent={recent}", flush=True)
    kept = evict(sess, cache, kv, keep, recent)
    want = evict_rule(w, keep, recent)
    assert np.array_equal(kept, want)
    left = n - (-(-n // B) - len(want[0])) * B
    assert sess.cache_length(cache, 0) == left
    hk, hv, hw = (chosen(x, want, n, kv) for x in (held(k, kv), held(v, kv), w))
    gk, gv, gw = read(sess, cache, kv, dim)
    assert same(gk, hk) and same(gv, hv) and same(gw, hw)
    # the freed blocks take new rows, and the open block goes on from its fp32 rows
    nk, nv = rows_of(rng, 100, kv, dim)
    append(sess, cache, nk, nv)
    gk, gv, gw = read(sess, cache, kv, dim)
    open_row = left // B * B
    tail = n - (left - open_row)
    for got, raw, new, old in ((gk, k, nk, hk), (gv, v, nv, hv)):
        full = held(np.concatenate([raw[tail:], new]), kv)
        assert same(got, np.concatenate([old[:open_row], full]))
    assert same(gw, np.concatenate([hw, np.zeros((100, kv), np.float32)]))
    sess.cache_destroy(cache)


def test_evict_ties_and_odd_weights(sess):
    """Equal blocks stay by their place; -0 is 0, NaN less than anything, infinities in order; the weights of a block's rows
    behind the last row do not count."""
    kv, dim, nb = 3, 4, 12
    n = nb * B - 20
    w = np.zeros((n, kv), np.float32)
    w[:, 1] = 1
    w[2 * B, 1] = np.nan
    w[0:B, 2] = -0.0
    w[3 * B, 2] = np.inf
    w[5 * B, 2] = -np.inf
    w[7 * B, 2] = np.nan
    x = np.ones((n, kv * dim), np.float32)
    cache = sess.cache(1, kv, dim, nb * B)
    append(sess, cache, np.ones((nb * B, kv * dim), np.float32), np.ones((nb * B, kv * dim), np.float32), weights=np.full((nb * B, kv), 1e9, np.float32))
    _lib.check(sess.cache_truncate(cache, 0, 0), "truncate")
    append(sess, cache, x, x, weights=w)
    for keep in (11, 10, 9, 4, 1):
        kept = evict(sess, cache, kv, keep, 1)
        want = evict_rule(w, keep, 1)
        assert np.array_equal(kept, want), keep
        w = chosen(w, want, len(w), kv)
    sess.cache_destroy(cache)


def test_attention_after_eviction(sess):
    """Heads hold different rows in mixed blocks of the memory: a step and a chunk over them, then weights counted where
    the rows lie now."""
    rng = np.random.default_rng(99)
    n, kv, dim, heads = 1000, 3, 128, 12
    k, v = rows_of(rng, n, kv, dim)
    cache = sess.cache(1, kv, dim, n + 64)
    append(sess, cache, k, v, weights=rng.random((n, kv)).astype(np.float32))
    evict(sess, cache, kv, 14, 2)
    nk, nv = rows_of(rng, 70, kv, dim)
    append(sess, cache, nk, nv)
    evict(sess, cache, kv, 13, 3)
    for rows in (1, 2, 70):
        hk, hv, old = read(sess, cache, kv, dim)
        q = rng.standard_normal((rows, heads * dim)).astype(np.float32)
        y = attention(sess, cache, q, heads, True, True, 1.0)
        ref, w, bound, wb = attend64(q, hk, hv, heads, kv)
        assert (np.abs(y - ref) <= bound).all()
        gw = read(sess, cache, kv, dim)[2]
        assert (np.abs(gw - (w + old)) <= wb + 2.0 ** -22 * (w + old)).all()
    sess.cache_destroy(cache)


def test_copy(sess):
    """A fork holds the same bits, goes on from the same open rows, and neither side sees the other's rows."""
    rng = np.random.default_rng(8)
    n, kv, dim, layers = 300, 2, 80, 3
    k, v = rows_of(rng, n, kv, dim)
    w = rng.random((n, kv)).astype(np.float32)
    a, b = sess.cache(layers, kv, dim, n + 50), sess.cache(layers, kv, dim, n)
    for layer in range(2):  # the third stays empty
        append(sess, a, k, v, layer, w)
        evict(sess, a, kv, 6 + layer, 1, layer)
    append(sess, b, v, k, 2)
    evict(sess, b, kv, 5, 1, 2)
    _lib.check(sess.cache_copy(b, a), "copy")
    before = [read(sess, a, kv, dim, layer=i) for i in range(2)]
    assert [sess.cache_length(b, i) for i in range(layers)] == [sess.cache_length(a, i) for i in range(layers)] and sess.cache_length(b, 2) == 0
    for i in range(2):
        assert all(same(x, y) for x, y in zip(read(sess, b, kv, dim, layer=i), before[i]))
    append(sess, b, v[:40], k[:40], 1)
    append(sess, b, v[:40], k[:40], 2)
    assert all(same(x, y) for x, y in zip(read(sess, a, kv, dim, layer=1), before[1]))
    append(sess, a, v[:40], k[:40], 1)
    assert all(same(x, y) for x, y in zip(read(sess, a, kv, dim, layer=1), read(sess, b, kv, dim, layer=1)))
    assert same(read(sess, b, kv, dim, layer=2)[0], held(v[:40], kv))
    small = sess.cache(layers, kv, dim, 64)
    assert sess.cache_copy(small, a) == _lib.ERR_MEMORY and sess.cache_copy(a, a) == _lib.ERR_ARGUMENT
    for c in (a, b, small):
        sess.cache_destroy(c)


def test_refusals(sess):
    arg, state, memory = _lib.ERR_ARGUMENT, _lib.ERR_STATE, _lib.ERR_MEMORY
    lib, h = sess.lib, ctypes.c_void_p()
    for bad, code in (((0, 1, 64, 10), arg), ((1, 0, 64, 10), arg), ((1, 1, 0, 10), arg), ((1, 1, 64, 0), arg), ((1, 1, 129, 10), _lib.ERR_UNSUPPORTED),
                      ((1, 1, 64, 1 << 40), arg), ((1 << 62, 8, 128, 4096), memory), ((1 << 20, 8, 128, 1 << 20), memory), ((1, 1 << 20, 64, 32), arg)):
        assert lib.pixhip_cache_create(sess.handle, *bad, ctypes.byref(h)) == code and not h.value, bad
    assert lib.pixhip_cache_create(sess.handle, 1, 1, 64, 10, None) == arg
    cache = sess.cache(2, 2, 64, 60)  # (64 rows)
    x = sess.to_device(np.ones((64, 4 * 64), np.float32))
    out = sess.alloc(64 * 4 * 64 * 4)
    assert sess.cache_attention(cache, 0, x.ptr, 1, 4, out.ptr) == state and sess.cache_evict(cache, 0, 1, 1) == state
    assert sess.cache_read(cache, 0, 0, 1, out.ptr) == arg and sess.cache_truncate(cache, 0, 1) == arg
    assert sess.cache_append(cache, 0, x.ptr, x.ptr, 65) == memory and sess.cache_append(cache, 0, x.ptr, x.ptr, 0) == arg
    assert sess.cache_append(cache, 2, x.ptr, x.ptr, 1) == arg and sess.cache_append(cache, 0, None, x.ptr, 1) == arg
    assert sess.cache_append(cache, 0, x.ptr, x.ptr, 2, 127) == arg and sess.cache_append(cache, 0, x.ptr + 2, x.ptr, 1) == arg
    assert sess.cache_append(cache, 0, x.ptr, x.ptr, 64, 1 << 20) == arg  # runs past the allocation (which the pool may have given twice as long)
    assert sess.cache_length(cache, 0) == 0
    _lib.check(sess.cache_append(cache, 0, x.ptr, x.ptr, 40), "append")
    assert sess.cache_append(cache, 0, x.ptr, x.ptr, 25) == memory and sess.cache_length(cache, 0) == 40
    att = sess.cache_attention
    assert att(cache, 0, x.ptr, 41, 2, out.ptr) == arg                    # causal, more rows than keys
    assert att(cache, 0, x.ptr, 1, 3, out.ptr) == arg and att(cache, 0, x.ptr, 1, 0, out.ptr) == arg
    assert att(cache, 0, x.ptr, 0, 2, out.ptr) == arg and att(cache, 0, None, 1, 2, out.ptr) == arg and att(cache, 0, x.ptr, 1, 2, None) == arg
    assert att(cache, 0, x.ptr, 2, 2, out.ptr, 127) == arg and att(cache, 0, x.ptr, 650, 4, out.ptr, 0, False) == arg
    assert att(cache, 0, x.ptr, 1, 2, out.ptr, 0, True, True, -0.5) == arg and att(cache, 0, x.ptr, 1, 2, out.ptr, 0, True, True, float("nan")) == arg
    host = np.zeros(256, np.float32)
    assert att(cache, 0, x.ptr, 1, 2, host.ctypes.data) == arg            # a pageable output
    assert sess.cache_evict(cache, 0, 1, 0) == arg and sess.cache_evict(cache, 0, 1, 2) == arg
    assert sess.cache_evict(cache, 0, 1, 1, host.ctypes.data) == arg and sess.cache_length(cache, 0) == 40
    assert sess.cache_read(cache, 0, 30, 11, out.ptr) == arg and sess.cache_read(cache, 0, 0, 4) == arg
    assert lib.pixhip_cache_length(cache, 5, ctypes.byref(ctypes.c_size_t())) == arg
    other = new_session()
    try:
        assert other.cache_append(cache, 0, x.ptr, x.ptr, 1) == arg and other.cache_truncate(cache, 0, 0) == arg
        lib.pixhip_cache_destroy(other.handle, cache)  # not its cache: nothing happens
        assert sess.cache_length(cache, 0) == 40
    finally:
        other.close()
    for b in (x, out):
        b.free()
    sess.cache_destroy(cache)
    sess.cache_destroy(cache)  # gone already: nothing happens


# ---- streams, graphs, a whole chat ----

def test_captured_calls(sess):
    """Append, attention with weights and eviction of a fork captured into one graph; replayed with eager work between the
    replays it gives the eager bits each time."""
    rng = np.random.default_rng(21)
    n, kv, dim, heads, rows = 700, 2, 128, 8, 2
    k, v = rows_of(rng, n, kv, dim)
    s = new_session()
    lib, stream, graph, ready = s.lib, ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    try:
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, stream), "set_stream")
        base, work = s.cache(1, kv, dim, n), s.cache(1, kv, dim, n + 64)
        append(s, base, k[:n - rows], v[:n - rows], weights=rng.random((n - rows, kv)).astype(np.float32))
        kb, vb = s.to_device(k[n - rows:]), s.to_device(v[n - rows:])
        qb = s.to_device(rng.standard_normal((rows, heads * dim)).astype(np.float32))
        ob, keptb = s.alloc(rows * heads * dim * 4), s.alloc(kv * 9 * 4)

        def step():
            codes = [s.cache_copy(work, base), s.cache_append(work, 0, kb.ptr, vb.ptr, rows),
                     s.cache_attention(work, 0, qb.ptr, rows, heads, ob.ptr, 0, True, True, 0.9), s.cache_evict(work, 0, 9, 2, keptb.ptr)]
            assert codes == [_lib.OK] * 4

        def results():
            return [ob.download(np.float32, rows * heads * dim), keptb.download(np.int32, kv * 9)] + read(s, work, kv, dim)

        step()
        eager = results()
        s.synchronize()
        assert lib.hipStreamBeginCapture(stream, 1) == 0
        step()
        assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert lib.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)) == 0
        for i in range(4):
            print(f"replay {i}", flush=True)
            ob.upload(np.zeros(rows * heads * dim, np.float32))
            assert lib.hipGraphLaunch(ready, stream) == 0
            assert all(same(x, y) for x, y in zip(results(), eager)), i
            other = s.cache(1, kv, dim, 200 * (i + 1))  # eager work between
            append(s, other, k[:150], v[:150])
            attention(s, other, rng.standard_normal((100, heads * dim)).astype(np.float32), heads, True, True)
            s.cache_destroy(other)
        s.synchronize()
        assert lib.hipGraphExecDestroy(ready) == 0 and lib.hipGraphDestroy(graph) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, None), "set_stream")
        assert lib.hipStreamDestroy(stream) == 0
    finally:
        s.close()


def test_a_chat(sess):
    """What a chat does, in order, on one cache of two layers kept small: a prompt in chunks, steps with weights, eviction
    where the cache is full, the logits' log probabilities last; each step against the definition, on the rows that the
    definition says are left."""
    rng = np.random.default_rng(33)
    kv, dim, heads, layers, vocab, keep = 2, 64, 8, 2, 1111, 5
    cache = sess.cache(layers, kv, dim, 8 * B)
    raw = [{"k": np.zeros((0, kv * dim), np.float32), "v": np.zeros((0, kv * dim), np.float32), "w": np.zeros((0, kv))} for _ in range(layers)]
    base = [np.zeros((0, kv * dim), np.float32) for _ in range(2 * layers)]
    for step, rows in enumerate([50, 50, 1, 1, 30, 1, 1, 64, 1, 33, 1, 1, 1]):
        for layer in range(layers):
            st = raw[layer]
            k, v = rows_of(rng, rows, kv, dim)
            q = rng.standard_normal((rows, heads * dim)).astype(np.float32)
            append(sess, cache, k, v, layer)
            st["k"], st["v"] = np.concatenate([st["k"], k]), np.concatenate([st["v"], v])
            n = len(st["k"])
            fixed = len(base[2 * layer]) // B * B  # rows of blocks that eviction left behind keep their codes
            hk, hv = (np.concatenate([b[:fixed], held(x[fixed:], kv)]) for b, x in ((base[2 * layer], st["k"]), (base[2 * layer + 1], st["v"])))
            y = attention(sess, cache, q, heads, True, True, 1.0, layer)
            ref, w, bound, wb = attend64(q, hk, hv, heads, kv)
            assert (np.abs(y - ref) <= bound).all(), (step, layer)
            gk, gv, gw = read(sess, cache, kv, dim, layer=layer)
            assert same(gk, hk) and same(gv, hv), (step, layer)
            st["w"] = np.concatenate([st["w"], np.zeros((rows, kv))]) + w
            assert (np.abs(gw - st["w"]) <= 1e-3 * st["w"] + 1e-6).all()
            st["w"] = gw.astype(np.float64)
            if -(-n // B) > keep:
                kept = evict(sess, cache, kv, keep, 2, layer)
                assert np.array_equal(kept, evict_rule(gw, keep, 2))
                base[2 * layer], base[2 * layer + 1] = chosen(hk, kept, n, kv), chosen(hv, kept, n, kv)
                st["k"], st["v"] = chosen(st["k"], kept, n, kv), chosen(st["v"], kept, n, kv)
                st["w"] = chosen(gw, kept, n, kv).astype(np.float64)
        logits = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
        ids = rng.integers(0, vocab, rows).astype(np.int32)
        lb, pb, eb, tb, tp = sess.to_device(logits), sess.alloc(rows * 4), sess.alloc(rows * 4), sess.alloc(rows * 12), sess.alloc(rows * 12)
        _lib.check(sess.log_probs(lb.ptr, rows, vocab, ids.ctypes.data, pb.ptr, eb.ptr, 3, tb.ptr, tp.ptr), "log_probs")
        x = logits.astype(np.float64)
        logp = x - x.max(axis=1, keepdims=True)
        logp -= np.log(np.exp(logp).sum(axis=1, keepdims=True))
        assert np.abs(pb.download(np.float32, rows) - logp[np.arange(rows), ids]).max() <= 1e-5
        assert np.array_equal(tb.download(np.int32, rows * 3).reshape(rows, 3), np.argsort(-x, axis=1, kind="stable")[:, :3])
        for b in (lb, pb, eb, tb, tp):
            b.free()
    sess.cache_destroy(cache)


# pieces of several steps of 64 rows (the tile kernel's two loops, odd and even
# counts), and the lengths around which few queries are cut into pieces
@pytest.mark.parametrize("rows,n,heads,kv,dim", [
    (128, 2600, 16, 8, 64),
    (128, 4100, 32, 8, 128),
    (128, 4161, 32, 8, 100),
    (70, 3333, 24, 8, 33),
    (2, 767, 8, 2, 128),
    (2, 768, 8, 2, 128),
    (2, 769, 8, 2, 64),
    (1, 832, 4, 4, 96),
])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_pieces(sess, rows, n, heads, kv, dim, causal):
    rng = np.random.default_rng(rows * 17 + n + dim)
    k, v = rows_of(rng, n, kv, dim)
    q = (1.3 * rng.standard_normal((rows, heads * dim))).astype(np.float32)
    print(f"rows={rows} n={n} heads={heads}/{kv} dim={dim} causal={causal}", flush=True)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v)
    y = attention(sess, cache, q, heads, causal, True, 0.0)
    ref, w, bound, wb = attend64(q, held(k, kv), held(v, kv), heads, kv, causal)
    assert (np.abs(y - ref) <= bound).all()
    assert (np.abs(read(sess, cache, kv, dim)[2] - w) <= wb + rows * heads / kv * 2.0 ** -24 * w).all()  # (a sum of that many terms)
    sess.cache_destroy(cache)


def test_codes_next_to_ties(sess):
    """Quotients at, just below and just above a half: codes by the exact quotient."""
    kv, dim = 1, 128
    x = np.zeros((32, dim), np.float32)
    scale = np.float32(np.float32(1.0) / np.float32(127.0))  # the block's largest is 1
    rng = np.random.default_rng(3)
    half = (rng.integers(-127, 127, 32 * dim) + 0.5).astype(np.float64) * scale
    near = half.astype(np.float32)
    steps = rng.integers(-2, 3, 32 * dim)
    for _ in range(2):
        near = np.where(steps > 0, np.nextafter(near, np.float32(2)), np.where(steps < 0, np.nextafter(near, np.float32(-2)), near))
        steps -= np.sign(steps)
    x[:] = near.reshape(32, dim)
    x[0, 0] = 1.0
    codes = np.rint(x.astype(np.float64) / np.float64(scale))
    want = (codes.astype(np.int8).astype(np.float32) * scale).astype(np.float32)
    cache = sess.cache(1, kv, dim, 32)
    append(sess, cache, x, x)
    k, v, _ = read(sess, cache, kv, dim)
    assert np.array_equal(k, want) and np.array_equal(v, want)
    sess.cache_destroy(cache)


# both sides of the rule that takes up to 256 queries of short caches four at a time
@pytest.mark.parametrize("rows,n,heads,kv,dim", [
    (64, 1000, 4, 1, 128),
    (50, 700, 5, 1, 40),
    (256, 300, 2, 2, 64),
    (257, 300, 2, 2, 64),
    (64, 2049, 16, 4, 128),
    (32, 4096, 16, 4, 128),
])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_short_caches(sess, rows, n, heads, kv, dim, causal):
    rng = np.random.default_rng(rows * 13 + n + dim)
    k, v = rows_of(rng, n, kv, dim)
    q = (1.3 * rng.standard_normal((rows, heads * dim))).astype(np.float32)
    print(f"rows={rows} n={n} heads={heads}/{kv} dim={dim} causal={causal}", flush=True)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v)
    y = attention(sess, cache, q, heads, causal, False, 0.0)
    ref, _, bound, _ = attend64(q, held(k, kv), held(v, kv), heads, kv, causal)
    assert (np.abs(y - ref) <= bound).all()
    sess.cache_destroy(cache)


# weights: kept scores of up to 32 queries per kv head, then both forms of the
# kernel that takes the probabilities again (few tokens, many tokens)
@pytest.mark.parametrize("rows,n,heads,kv,dim", [
    (3, 700, 12, 3, 128),
    (8, 2500, 8, 2, 80),
    (5, 3000, 28, 4, 64),
    (33, 175, 14, 2, 128),
    (150, 1000, 14, 2, 64),
    (70, 2100, 16, 8, 128),
    (300, 5000, 4, 4, 40),
])
@pytest.mark.parametrize("causal", [False, True])
def test_weights(sess, rows, n, heads, kv, dim, causal):
    rng = np.random.default_rng(rows * 11 + n + dim)
    k, v = rows_of(rng, n, kv, dim)
    q = (1.3 * rng.standard_normal((rows, heads * dim))).astype(np.float32)
    old = rng.random((n, kv)).astype(np.float32)
    print(f"rows={rows} n={n} heads={heads}/{kv} dim={dim} causal={causal}", flush=True)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v, weights=old)
    y = attention(sess, cache, q, heads, causal, True, 0.25)
    ref, w, bound, wb = attend64(q, held(k, kv), held(v, kv), heads, kv, causal)
    assert (np.abs(y - ref) <= bound).all()
    off = np.abs(read(sess, cache, kv, dim)[2] - (w + 0.25 * old))
    assert (off <= wb + (rows * heads / kv + 2) * 2.0 ** -24 * (w + old)).all()  # (a sum of that many terms)
    sess.cache_destroy(cache)


@pytest.mark.parametrize("n", [200, 5000])
def test_captured_chunk(sess, n):
    """A chunk's attention with weights (both forms of the weights' kernel) and a step's without, captured and replayed
    with the same calls on another cache between the replays; the step's output takes the place of its queries."""
    rng = np.random.default_rng(n)
    kv, dim, heads, rows = 2, 64, 8, 40
    k, v = rows_of(rng, n, kv, dim)
    q = rng.standard_normal((rows, heads * dim)).astype(np.float32)
    s = new_session()
    lib, stream, graph, ready = s.lib, ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    try:
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, stream), "set_stream")
        cache, other = s.cache(1, kv, dim, n), s.cache(1, kv, dim, n)
        append(s, cache, k, v)
        append(s, other, k[::-1], v[::-1])
        qb, ob, xb = s.to_device(q), s.alloc(q.nbytes), s.to_device(q[:2])

        def calls(c, out):
            assert s.cache_attention(c, 0, qb.ptr, rows, heads, out.ptr, 0, True, True, 0.0) == _lib.OK
            assert s.cache_attention(c, 0, xb.ptr, 2, heads, xb.ptr, 0, True, False, 0.0) == _lib.OK

        def results():
            got = [ob.download(np.float32, q.size), xb.download(np.float32, 2 * heads * dim), read(s, cache, kv, dim)[2]]
            xb.upload(np.ascontiguousarray(q[:2]))
            return got

        calls(cache, ob)
        eager = results()
        ref, w, bound, wb = attend64(q[:2], held(k, kv), held(v, kv), heads, kv, True)
        assert (np.abs(eager[1].reshape(2, -1) - ref) <= bound).all()
        s.synchronize()
        assert lib.hipStreamBeginCapture(stream, 1) == 0
        calls(cache, ob)
        assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert lib.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)) == 0
        spare = s.alloc(q.nbytes)
        for i in range(3):
            print(f"replay {i}", flush=True)
            ob.upload(np.zeros(q.size, np.float32))
            assert lib.hipGraphLaunch(ready, stream) == 0
            assert all(same(x, y) for x, y in zip(results(), eager)), i
            calls(other, spare)
            results()
        s.synchronize()
        assert lib.hipGraphExecDestroy(ready) == 0 and lib.hipGraphDestroy(graph) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, None), "set_stream")
        assert lib.hipStreamDestroy(stream) == 0
    finally:
        s.close()


@pytest.mark.parametrize("n", [16320, 16385, 32801])
def test_weights_of_groups_in_twos(sess, n):
    """255 to 513 groups of 64 tokens: one by one, two to a workgroup (the last one alone), and the kernel for more."""
    rng = np.random.default_rng(n)
    rows, heads, kv, dim = 300, 1, 1, 16
    k, v = rows_of(rng, n, kv, dim)
    q = (2.0 * rng.standard_normal((rows, heads * dim))).astype(np.float32)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v)
    attention(sess, cache, q, heads, True, True, 0.0)
    _, w, _, wb = attend64(q, held(k, kv), held(v, kv), heads, kv, True)
    off = np.abs(read(sess, cache, kv, dim)[2] - w)
    assert (off <= wb + (rows + 2) * 2.0 ** -24 * w).all()
    sess.cache_destroy(cache)


@pytest.mark.parametrize("blocks,recent", [(128, 1), (129, 1), (130, 1), (131, 3)])
def test_evict_around_the_ranked_sizes(sess, blocks, recent):
    """127 to 129 candidates, of which many have equal weights: ranked against one another, and by the bins."""
    rng = np.random.default_rng(blocks + recent)
    kv, dim = 2, 16
    n = blocks * B - 5
    k, v = rows_of(rng, n, kv, dim)
    w = np.repeat(rng.integers(0, 9, (blocks, kv)), B, axis=0)[:n].astype(np.float32)
    w[:B] = np.nan
    cache = sess.cache(1, kv, dim, n)
    for keep in (blocks - 1, 70, 20, recent + 1, recent):
        _lib.check(sess.cache_truncate(cache, 0, 0), "truncate")
        append(sess, cache, k, v, weights=w)
        kept = evict(sess, cache, kv, keep, recent)
        assert np.array_equal(kept, evict_rule(w, keep, recent))
        assert same(read(sess, cache, kv, dim)[0], chosen(held(k, kv), kept, n, kv))
    sess.cache_destroy(cache)
