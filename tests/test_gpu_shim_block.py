"""The C++ shim's calls for what lies between a block's linears (hip_residual_norm_
multiply, hip_adapter_of, hip_adapters, hip_split_heads, hip_cache_append_rotated of
pixelina_amd/host/backend_hip.h), driven by `shim_check block` with its vectors in
pageable memory; against the definitions of the tests of the C ABI, with their bounds.
"""
import os
import subprocess

import numpy as np
import pytest

from test_gpu_adapters import U
from test_gpu_cache import attend64, held, same
from test_gpu_heads import RMS, turned
from test_gpu_residual_norm import definition

pytestmark = pytest.mark.gpu

SHIM_CHECK = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pixelina_amd", "shim_check")


@pytest.mark.parametrize("rows,hidden,heads,kv,dim,rank", [(37, 520, 6, 2, 64, 9), (70, 256, 4, 4, 128, 16), (3, 99, 2, 1, 34, 4)])
def test_shim_block(tmp_path, rows, hidden, heads, kv, dim, rank):
    assert os.path.exists(SHIM_CHECK), "pixelina_amd/shim_check is not built (run __graft_entry__.build())"
    rng = np.random.default_rng(rows)
    width = (heads + 2 * kv) * dim
    n = lambda *shape: rng.standard_normal(shape).astype(np.float32)  # noqa: E731
    angle = rng.uniform(0, 9, (rows, dim // 2))
    t = {"x": n(rows, hidden) * 3, "branch": n(rows, hidden), "post_weight": 1 + n(hidden) / 5, "pre_weight": 1 + n(hidden) / 5, "gate": n(hidden),
         "modulation": n(hidden) / 2}
    rest = [n(rows, width), 1 + n(dim) / 4, 1 + n(dim) / 4, np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32),
            n(rank, hidden) / np.float32(np.sqrt(hidden)), n(width, rank) / 3]
    p, qw, kw, cos, sin, down, up = rest
    src, dst = tmp_path / "in.bin", tmp_path / "out.bin"
    with open(src, "wb") as fh:
        fh.write(np.array([rows, hidden, heads, kv, dim, rank], np.uint64).tobytes())
        for a in (*t.values(), *rest):
            fh.write(np.ascontiguousarray(a, np.float32).tobytes())
    print("running shim_check block", flush=True)
    proc = subprocess.run([SHIM_CHECK, "block", str(src), str(dst)], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    shapes = [(rows, hidden)] * 2 + [(rows, width)] + [(rows, heads * dim)] + [(rows, kv * dim)] * 2 + [(rows, heads * dim)] + [(rows, kv * dim)] * 2 + \
        [(rows, heads * dim)]
    out = np.fromfile(dst, np.float32)
    assert out.size == sum(a * b for a, b in shapes)
    x, y, p2, q, k, v, cq, ck, cv, att = (a.reshape(s) for a, s in zip(np.split(out, np.cumsum([a * b for a, b in shapes])[:-1]), shapes))

    two = {k: np.stack([v, v]) if k in ("gate", "modulation") else v for k, v in t.items()}
    want_x, dx, want_y, dy = definition(two, RMS, RMS, True, True, 0, 1.0)
    assert (np.abs(x - want_x) <= dx).all() and (np.abs(y - want_y) <= dy).all()
    # from the y that the call itself left
    half = rows // 2
    wide = y[half:].astype(np.float64)
    part, big = wide @ down.T.astype(np.float64), np.abs(wide) @ np.abs(down).T.astype(np.float64)
    want = p[half:] + 1.5 * part @ up.T.astype(np.float64)
    bound = 1.5 * ((hidden + 9) * U * big + (rank + 8) * U * np.abs(part)) @ np.abs(up).T.astype(np.float64) + 4 * U * np.abs(want)
    assert same(p2[:half], p[:half]) and (np.abs(p2[half:] - want) <= bound).all()
    pq, pk, pv = p2[:, :heads * dim], p2[:, heads * dim:(heads + kv) * dim], p2[:, (heads + kv) * dim:]
    want_q, want_k = (turned(a, dim, RMS, w, cos, sin, dim, False) for a, w in ((pq, qw), (pk, kw)))
    assert same(q, want_q) and same(k, want_k) and same(v, pv) and same(cq, want_q)
    assert same(ck, held(want_k, kv)) and same(cv, held(pv, kv))
    ref, _, bound, _ = attend64(want_q, ck, cv, heads, kv, True)
    assert (np.abs(att - ref) <= bound).all()
