"""The C++ shim's cache and log-probability calls (hip_cache_*, hip_log_probs of
pixelina_amd/host/backend_hip.h), driven as a chat would by `shim_check cache`:
a prompt appended and weighed, a copy that takes one more row, is cut back and
takes it again, eviction from the first, and the log probabilities of its rows.

Against the same definitions in 64 bits as the tests of the C ABI, with their
bounds.
"""
import os
import subprocess

import numpy as np
import pytest

from test_gpu_cache import attend64, held

pytestmark = pytest.mark.gpu

SHIM_CHECK = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pixelina_amd", "shim_check")


def test_shim_chat(tmp_path):
    assert os.path.exists(SHIM_CHECK), "pixelina_amd/shim_check is not built (run __graft_entry__.build())"
    rng = np.random.default_rng(91)
    rows, heads, kv, dim, vocab = 101, 6, 2, 80, 1003
    k, v = (rng.standard_normal((rows, kv * dim)).astype(np.float32) for _ in range(2))
    q = (1.2 * rng.standard_normal((rows, heads * dim))).astype(np.float32)
    logits = (3.0 * rng.standard_normal((rows, vocab))).astype(np.float32)
    ids = rng.integers(0, vocab, rows).astype(np.int32)
    src, dst = tmp_path / "in.bin", tmp_path / "out.bin"
    with open(src, "wb") as fh:
        fh.write(np.array([rows, heads, kv, dim, vocab], np.uint64).tobytes())
        for a in (k, v, q, logits, ids):
            fh.write(a.tobytes())
    print("running shim_check cache", flush=True)
    proc = subprocess.run([SHIM_CHECK, "cache", str(src), str(dst)], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    sizes = [(rows - 1) * heads * dim, heads * dim, 2, rows, rows, 2 * rows, 2 * kv, 2 * rows]
    out = np.fromfile(dst, np.float32)
    assert out.size == sum(sizes)
    first, last, lengths, log_probs, entropy, top_log_probs, kept, top_ids = np.split(out, np.cumsum(sizes)[:-1])

    ref, w, bound, _ = attend64(q[:-1], held(k[:-1], kv), held(v[:-1], kv), heads, kv, True)
    assert (np.abs(first.reshape(rows - 1, -1) - ref) <= bound).all()
    ref, _, bound, _ = attend64(q[-1:], held(k, kv), held(v, kv), heads, kv, True)
    assert (np.abs(last.reshape(1, -1) - ref) <= bound).all()

    # 100 rows are 4 blocks; kept: the last one and the heaviest of the others
    assert list(lengths) == [32 + 4, rows]
    blocks = w[:96].reshape(3, 32, kv).sum(1)
    order = np.sort(blocks, 0)
    assert ((order[-1] - order[-2]) > 1e-3 * order[-1]).all()  # (no tie that rounding could turn)
    assert np.array_equal(kept.view(np.int32).reshape(kv, 2), np.stack([blocks.argmax(0), np.full(kv, 3)], 1))

    x = logits.astype(np.float64)
    lp = x - x.max(1, keepdims=True)
    lp -= np.log(np.exp(lp).sum(1, keepdims=True))
    spread = np.abs(x - x.max(1, keepdims=True)).max() + np.log(vocab)
    tol = 2.0 ** -23 * spread + 2.0 ** -15
    assert np.abs(log_probs - lp[np.arange(rows), ids]).max() <= tol
    ent = -(np.exp(lp) * lp).sum(1)
    assert (np.abs(entropy - ent) <= 2.0 ** -14 * (1 + ent)).all()
    best = np.argsort(-x, 1, kind="stable")[:, :2]
    assert np.array_equal(top_ids.view(np.int32).reshape(rows, 2), best)
    assert np.abs(top_log_probs.reshape(rows, 2) - np.take_along_axis(lp, best, 1)).max() <= tol
