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


def cut_cases():
    for start, rows in ((60, 8), (20, 20), (24, 8), (0, 32), (0, 64), (32, 32), (31, 34), (77, 73), (0, 128), (1, 1)):
        yield start, rows, 1
    yield 60, 8, 3


@pytest.mark.parametrize("start,rows,calls", cut_cases())
def test_cuts_inside_the_last_append(sess, start, rows, calls):
    """Every cut from where the last append began to its end, then new rows: as if the rows behind the cut had never come,
    except in blocks that lie inside the append with neither its begin's open rows nor its end in them."""
    rng = np.random.default_rng(start * 7 + rows)
    kv, dim = 2, 80
    k, v = rows_of(rng, start + rows + 40, kv, dim)
    k *= np.exp(rng.standard_normal((len(k), 1))).astype(np.float32)
    end = start + rows
    cache = sess.cache(1, kv, dim, end + 40)
    for cut in range(start, end + 1):
        _lib.check(sess.cache_truncate(cache, 0, 0), "truncate")
        for part in np.array_split(np.arange(start), calls):
            if len(part):
                append(sess, cache, k[part], v[part])
        append(sess, cache, k[start:end], v[start:end])
        _lib.check(sess.cache_truncate(cache, 0, cut), "truncate")
        assert sess.cache_length(cache, 0) == cut
        append(sess, cache, v[end:], k[end:])
        begin = cut // B * B  # of the block the cut falls into
        exact = begin <= start < begin + B and start % B or begin <= end - 1 < begin + B
        for got, old, new in zip(read(sess, cache, kv, dim), (k, v), (v, k)):
            stays = old[begin:cut] if exact else held(old, kv)[begin:cut]
            assert same(got, np.concatenate([held(old, kv)[:begin], held(np.concatenate([stays, new[end:]]), kv)])), cut
    sess.cache_destroy(cache)


def test_cuts_of_a_rejected_draft(sess):
    """Drafts of eight rows behind a text, each cut back by another number of rows: the cache holds what it would hold if
    only the rows that stayed had come, one by one."""
    rng = np.random.default_rng(17)
    kv, dim = 2, 64
    text = [rows_of(rng, 8, kv, dim) for _ in range(40)]
    cache, fork = sess.cache(1, kv, dim, 400), sess.cache(1, kv, dim, 400)
    stay = [np.zeros((0, kv * dim), np.float32)] * 2
    for i, (k, v) in enumerate(text):
        append(sess, cache, k, v)
        n = len(stay[0]) + 1 + (5 * i) % 8
        _lib.check(sess.cache_truncate(cache, 0, n), "truncate")
        stay = [np.concatenate([a, b])[:n] for a, b in zip(stay, (k, v))]
        if i % 9 == 4:  # goes on in a copy
            _lib.check(sess.cache_copy(fork, cache), "copy")
            cache, fork = fork, cache
    append(sess, cache, text[0][0], text[0][1])
    gk, gv, _ = read(sess, cache, kv, dim)
    assert same(gk, held(np.concatenate([stay[0], text[0][0]]), kv)) and same(gv, held(np.concatenate([stay[1], text[0][1]]), kv))
    for c in (cache, fork):
        sess.cache_destroy(c)


@pytest.mark.parametrize("seed", range(6))
def test_cuts_among_other_calls(sess, seed):
    """Appends, cuts, evictions and copies in any order against the rule for the rows that count as appended."""
    rng = np.random.default_rng(seed)
    kv, dim, room = 1, 12, 700
    cache, fork = sess.cache(1, kv, dim, room), sess.cache(1, kv, dim, room)
    rows = np.zeros((2, 0, dim), np.float32)   # as they count when their block is quantized again
    codes = np.zeros((2, 0, dim), np.float32)  # as they are held
    ends = []                                  # the blocks whose fp32 rows the layer has
    for _ in range(80):
        n, call = rows.shape[1], rng.choice(["append", "append", "cut", "cut", "evict", "copy"])
        if call == "append" and n < room - 100:
            new = (rng.standard_normal((2, int(rng.choice([1, 3, 17, 32, 40, 100])), dim)) * np.exp(rng.standard_normal((2, 1, 1)))).astype(np.float32)
            if rng.random() < 0.4 and n % B:  # to the end of its block
                new = new[:, :B - n % B]
            append(sess, cache, new[0], new[1])
            rows = np.concatenate([rows, new], axis=1)
            first = n // B * B
            codes = np.stack([np.concatenate([codes[i, :first], held(rows[i, first:], kv)]) for i in range(2)])
            end = (rows.shape[1] - 1) // B
            if ends[-1:] != [end]:
                ends = (ends + [end])[-2:]
        elif call == "cut" and n:
            cut = int(max(0, n - rng.choice([0, 1, 5, 31, 32, 33, 60, 130, n])))
            _lib.check(sess.cache_truncate(cache, 0, cut), "truncate")
            rows, codes, block = rows[:, :cut].copy(), codes[:, :cut], cut // B
            ends = [b for b in ends if b < block or (b == block and cut % B)]
            if cut % B and block not in ends:
                rows[:, block * B:] = codes[:, block * B:]
                ends.append(block)
        elif call == "evict" and n > 4 * B:
            nb, keep = -(-n // B), int(rng.integers(2, 5))
            kb = sess.alloc(4 * keep)
            _lib.check(sess.cache_evict(cache, 0, keep, 1, kb.ptr), "evict")
            kept = kb.download(np.int32, keep)
            kb.free()
            at = np.concatenate([np.arange(b * B, min(n, b * B + B)) for b in kept])
            rows, codes = rows[:, at], codes[:, at]
            ends = [keep - 1] if nb - 1 in ends else []
        elif call == "copy":
            _lib.check(sess.cache_copy(fork, cache), "copy")
            cache, fork = fork, cache
        assert sess.cache_length(cache, 0) == rows.shape[1]
        if rows.shape[1]:
            gk, gv, _ = read(sess, cache, kv, dim)
            assert same(gk, codes[0]) and same(gv, codes[1]), call
    for c in (cache, fork):
        sess.cache_destroy(c)


@pytest.mark.parametrize("rows,n,heads,kv", [(6, 200, 2, 2), (8, 70, 8, 2), (40, 200, 2, 2), (32, 3000, 2, 2), (70, 40000, 1, 1)])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_weights_beside_a_row_that_is_not_a_number(sess, rows, n, heads, kv, value):
    """NaN weights for the rows that such a query sees, and for no others; theirs are the other queries'."""
    rng = np.random.default_rng(rows + n)
    dim, bad, head = 64, rows // 3, 1
    k, v = rows_of(rng, n, kv, dim)
    q = rng.standard_normal((rows, heads * dim)).astype(np.float32)
    if heads == 1:
        head = 0
    q[bad, head * dim + 9] = value
    old = rng.random((n, kv)).astype(np.float32)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v, weights=old)
    attention(sess, cache, q, heads, True, True, 0.5)
    got = read(sess, cache, kv, dim)[2]
    sess.cache_destroy(cache)
    clean = q.copy()
    clean[bad, head * dim:(head + 1) * dim] = 0
    seen = n - rows + bad + 1
    _, w, _, wb = attend_terms(clean, held(k, kv), held(v, kv), heads, kv)
    spoiled = np.zeros((n, kv), bool)
    spoiled[:seen, head // (heads // kv)] = True
    assert np.isnan(got[spoiled]).all()
    assert (np.abs(got - (w + 0.5 * old)) <= wb + 2.0 ** -22 * old)[~spoiled].all()  # (behind `seen` the bad row has no part in w)


@pytest.mark.parametrize("e", [96, 108, 118])
@pytest.mark.parametrize("rows,n,weigh", [(40, 300, True), (70, 16500, True), (40, 33000, True), (300, 300, False), (1, 300, False), (3, 300, True)])
def test_large_keys_and_tiny_queries(sess, rows, n, weigh, e):
    """Keys about 2^e and queries about 2^-e: ordinary scores."""
    rng = np.random.default_rng(rows + n)
    kv, dim, heads = 1, 64, 1
    k, v = rows_of(rng, n, kv, dim)
    q = rng.standard_normal((rows, heads * dim)).astype(np.float32)
    print(f"rows={rows} n={n} weigh={weigh} e={e}", flush=True)
    check(sess, k * np.float32(2.0 ** e), v, q * np.float32(2.0 ** -e), heads, kv, True, weigh)


@pytest.mark.parametrize("rows", [1, 300])
def test_largest_values(sess, rows):
    """Values next to the largest that fp32 holds, equal probabilities: their mean."""
    rng = np.random.default_rng(rows)
    n, kv, dim, heads = 700, 1, 64, 2
    v = (3e38 * (1 - 0.01 * rng.random((n, dim)))).astype(np.float32)
    k = np.zeros_like(v)
    q = rng.standard_normal((rows, heads * dim)).astype(np.float32)
    for weigh in (False, True):
        check(sess, k, v, q, heads, kv, False, weigh)


@pytest.mark.parametrize("sign,low,high", [(sign, *r) for sign in (1, -1) for r in ((16, 24), (22, 32), (30, 60), (90, 124))])
@pytest.mark.parametrize("rows,n,heads,kv,weigh", [
    (1, 300, 8, 2, True), (4, 1000, 8, 2, False),           # few queries
    (300, 300, 2, 2, False), (300, 300, 2, 2, True), (260, 1100, 16, 8, True), (70, 33000, 1, 1, True),  # many
])
def test_one_key_far_above_the_others(sess, rows, n, heads, kv, weigh, sign, low, high):
    """Scores of 2^low to 2^high, the nearest two further apart than fp32 rounds them: each row's output is one token's
    value, whatever the scales of the value blocks, and the weights count who was taken."""
    rng = np.random.default_rng(rows + n + low + sign)
    dim = 64
    steps = rng.integers(100, 121, (n, kv))
    best = rng.integers(0, n - rows + 1, kv)  # (seen by every row)
    steps[best, np.arange(kv)] = 127 if sign > 0 else 60
    # every block's largest is 127 or a negative query's worst, so that codes are whole steps
    for h in range(kv):
        for b in range(0, n, B):
            if sign < 0:
                at = b + int(rng.integers(0, min(B, n - b)))
                if at != best[h]:
                    steps[at, h] = 127
    if sign > 0:  # (blocks below 127 have scales of their own: still far from the best)
        steps = np.where(steps < 127, np.minimum(steps, 120), steps)
    k = np.repeat(steps.astype(np.float32), dim, axis=1)
    v = rng.standard_normal((n, kv * dim)).astype(np.float32)
    for b in range(-(-n // B)):
        v[b * B:(b + 1) * B] *= np.float32(2.0 ** rng.integers(-20, 20))
    size = np.exp2(rng.uniform(low, high - 1, (rows, heads))) / 1024  # (a score is 8 x 127 x this)
    q = np.repeat((sign * size).astype(np.float32), dim, axis=1)
    print(f"rows={rows} n={n} heads={heads}/{kv} weigh={weigh} sign={sign} 2^{low}..2^{high}", flush=True)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v)
    y = attention(sess, cache, q, heads, True, weigh, 0.0)
    got = read(sess, cache, kv, dim)[2]
    sess.cache_destroy(cache)
    hk, hv = held(k, kv).reshape(n, kv, dim), held(v, kv).reshape(n, kv, dim)
    for h in range(heads):
        g = h // (heads // kv)
        order = sign * hk[:, g, 0].astype(np.float64)
        assert order.argmax() == best[g] and np.sort(order)[-1] - np.sort(order)[-2] > 2  # (of 127: 2^9 and more at scores of 2^16)
        want = hv[best[g], g]
        # the digits of one term: 2^-27 of it, and three roundings
        assert (np.abs(y.reshape(rows, heads, dim)[:, h] - want) <= 2.0 ** -20 * np.abs(want).max()).all()
    if weigh:
        want = np.zeros((n, kv))
        want[best, np.arange(kv)] = rows * heads // kv
        assert (np.abs(got - want) <= 2.0 ** -20 * want).all()


@pytest.mark.parametrize("rows,n,heads,weigh", [(256, 8102, 1, False), (32, 40001, 1, True), (6, 9000, 1, True), (300, 700, 1, True)])
def test_scores_far_below_zero(sess, rows, n, heads, weigh):
    """Every score about -180: a step that a query sees nothing of leaves what it has."""
    rng = np.random.default_rng(n)
    kv, dim = 1, 64
    k = (rng.standard_normal((n, kv * dim)) - 15).astype(np.float32)
    v = rng.standard_normal((n, kv * dim)).astype(np.float32)
    q = (0.2 * rng.standard_normal((rows, heads * dim)) + 1.5).astype(np.float32)
    print(f"rows={rows} n={n} weigh={weigh}", flush=True)
    check(sess, k, v, q, heads, kv, True, weigh)


def test_captured_creation_is_refused(sess):
    """A cache is made outside a captured graph: its table would be written by replays alone."""
    s = new_session()
    lib, stream, graph, h = s.lib, ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    try:
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, stream), "set_stream")
        first = s.cache(1, 1, 64, 64)
        s.cache_destroy(first)  # (its memory lies in the pool)
        x = s.to_device(np.ones((8, 64), np.float32))
        s.synchronize()
        assert lib.hipStreamBeginCapture(stream, 1) == 0
        code = lib.pixhip_cache_create(s.handle, 1, 1, 64, 64, ctypes.byref(h))
        assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert code == _lib.ERR_STATE and not h.value and b"captur" in lib.pixhip_last_error()
        if graph.value:
            assert lib.hipGraphDestroy(graph) == 0
        second = s.cache(1, 1, 64, 64)
        _lib.check(s.cache_append(second, 0, x.ptr, x.ptr, 8), "append")
        assert (read(s, second, 1, 64)[0] == 1).all()
        s.cache_destroy(second)
        _lib.check(lib.pixhip_session_set_stream(s.handle, None), "set_stream")
        assert lib.hipStreamDestroy(stream) == 0
    finally:
        s.close()


def test_captured_calls_on_pinned_inputs(sess):
    """Queries and logits in pinned memory: replays read them where they are, as they are then, and write nothing but the
    outputs (buffers made after the capture keep what they hold)."""
    rng = np.random.default_rng(5)
    n, kv, dim, heads, rows, vocab = 200, 2, 64, 4, 40, 5000
    k, v = rows_of(rng, n, kv, dim)
    s = new_session()
    lib, stream, graph, ready = s.lib, ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    try:
        assert lib.hipStreamCreate(ctypes.byref(stream)) == 0
        _lib.check(lib.pixhip_session_set_stream(s.handle, stream), "set_stream")
        cache = s.cache(1, kv, dim, n)
        append(s, cache, k, v)
        q, x = (rng.standard_normal(shape).astype(np.float32) for shape in ((rows, heads * dim), (3, vocab)))
        hq, hx, ids = Pinned(s, q), Pinned(s, x), s.to_device(np.array([1, 2, 3], np.int32))
        ob, lb = s.alloc(q.nbytes), s.alloc(12)

        def calls():
            return [s.cache_attention(cache, 0, hq.p.value, rows, heads, ob.ptr), s.log_probs(hx.p.value, 3, vocab, ids.ptr, lb.ptr)]

        def results():
            return [ob.download(np.float32, q.size), lb.download(np.float32, 3)]

        assert calls() == [_lib.OK] * 2
        s.synchronize()
        assert lib.hipStreamBeginCapture(stream, 1) == 0
        codes = calls()
        assert lib.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0 and codes == [_lib.OK] * 2
        assert lib.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)) == 0
        mine = [s.to_device(np.full(a.shape, 9.0, np.float32)) for a in (q, x, q, x)]
        for i in range(3):
            print(f"replay {i}", flush=True)
            q, x = (rng.standard_normal(a.shape).astype(np.float32) for a in (q, x))
            ctypes.memmove(hq.p, q.ctypes.data, q.nbytes)
            ctypes.memmove(hx.p, x.ctypes.data, x.nbytes)
            assert lib.hipGraphLaunch(ready, stream) == 0
            y, lp = results()
            for b, a in zip(mine, (q, x, q, x)):
                assert (b.download(np.float32, a.size) == 9).all(), i
            assert calls() == [_lib.OK] * 2
            eager = results()
            assert same(y, eager[0]) and np.abs(lp - eager[1]).max() <= 2.0 ** -18
        s.synchronize()
        assert lib.hipGraphExecDestroy(ready) == 0 and lib.hipGraphDestroy(graph) == 0
        for b in (hq, hx):
            b.free()
        _lib.check(lib.pixhip_session_set_stream(s.handle, None), "set_stream")
        assert lib.hipStreamDestroy(stream) == 0
    finally:
        s.close()


@pytest.mark.parametrize("rows,n,heads,kv", [
    (1, 16384, 1, 1), (1, 16449, 1, 1), (1, 33001, 4, 1), (1, 40000, 4, 2), (2, 33100, 2, 1), (4, 70000, 2, 2),
])
@pytest.mark.parametrize("weigh", [False, True])
def test_more_than_64_pieces(sess, rows, n, heads, kv, weigh):
    """Few queries over long caches of few kv heads: up to 128 pieces, two to a lane of the wave that merges them."""
    rng = np.random.default_rng(n)
    dim = 128 if kv == 1 else 64
    k, v = rows_of(rng, n, kv, dim)
    q = (1.3 * rng.standard_normal((rows, heads * dim))).astype(np.float32)
    print(f"rows={rows} n={n} heads={heads}/{kv} weigh={weigh}", flush=True)
    check(sess, k, v, q, heads, kv, True, weigh)


@pytest.mark.parametrize("rows,n,heads,kv,dim", [(300, 700, 56, 8, 64), (17, 4500, 1023, 1, 16)])
@pytest.mark.parametrize("decay", [0.0, 0.5])
def test_weights_of_several_launches(sess, rows, n, heads, kv, dim, decay):
    """More queries per kv head than one launch's planes hold, cut inside a row's group of heads."""
    rng = np.random.default_rng(rows + n)
    k, v = rows_of(rng, n, kv, dim)
    q = (1.3 * rng.standard_normal((rows, heads * dim))).astype(np.float32)
    old = rng.random((n, kv)).astype(np.float32)
    print(f"rows={rows} n={n} heads={heads}/{kv} decay={decay}", flush=True)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v, weights=old)
    y = attention(sess, cache, q, heads, True, True, decay)
    got = read(sess, cache, kv, dim)[2]
    sess.cache_destroy(cache)
    ref, w, bound, wb = attend_terms(q, held(k, kv), held(v, kv), heads, kv)
    assert (np.abs(y - ref) <= bound).all()
    assert (np.abs(got - (w + decay * old)) <= wb + 2.0 ** -22 * (w + old)).all()


@pytest.mark.parametrize("rows,n,heads", [(1, 9001, 4), (1, 40000, 1), (3, 2501, 8), (260, 5000, 1), (40, 1300, 8)])
def test_each_probability_of_a_long_cache(sess, rows, n, heads):
    """Values that are 1 at a dim of their own, for 128 tokens spread over the pieces, and 0 elsewhere: every probability is
    its own score's and the sum's error away, and at most 2^-27 of the largest of the 128."""
    rng = np.random.default_rng(rows + n)
    kv, dim = 1, 128
    k, _ = rows_of(rng, n, kv, dim)
    at = np.sort(rng.choice(n, dim, replace=False))
    v = np.zeros((n, dim), np.float32)
    v[at, np.arange(dim)] = 1
    q = (1.2 * rng.standard_normal((rows, heads * dim))).astype(np.float32)
    print(f"rows={rows} n={n} heads={heads}", flush=True)
    cache = sess.cache(1, kv, dim, n)
    append(sess, cache, k, v)
    y = attention(sess, cache, q, heads, False).reshape(rows * heads, dim)
    sess.cache_destroy(cache)
    kh, qh = held(k, kv).astype(np.float64), q.astype(np.float64).reshape(-1, dim)
    s = qh @ kh.T / np.sqrt(dim)
    p = np.exp(s - s.max(axis=1, keepdims=True))
    p /= p.sum(axis=1, keepdims=True)
    # a score's error, from its own terms (the largest one's and the sum's stand for the others)
    mag = np.abs(qh) @ np.abs(kh).T / np.sqrt(dim)
    e = (dim + 8) * 2.0 ** -24 * mag + (2.0 ** -24 * dim * np.abs(qh).max(axis=1) * np.abs(kh).max() / np.sqrt(dim))[:, None]
    mean = (p * e).sum(axis=1, keepdims=True)
    want, limit = p[:, at], p[:, at] * (e[:, at] + mean + 2.0 ** -18) + 2.0 ** -27 * p[:, at].max(axis=1, keepdims=True)
    print(f"  of the bound {(np.abs(y - want) / limit).max():.2f}", flush=True)
    assert (np.abs(y - want) <= limit).all()
