"""The operators between a block's linears as they are used together: decoder layers of
a small chat model over the 8-bit cache (prompt in chunks, then single tokens, with an
adapter for each of two requests), against the same layers made of the calls that they
stand for; and a DiT block's fused list against its list of single steps.
"""
import numpy as np
import pytest

from gpu_helpers import new_session
from oracle_lib import Q8_0, oracle, quantize
from pixelina_amd import _lib, synth, zimage
from test_gpu_adapters import Adapter, BF16, F16

pytestmark = pytest.mark.gpu

RMS, NONE = _lib.NORM_RMS, _lib.NORM_NONE
HIDDEN, HEADS, KV, DIM, FFN, LAYERS, EPS = 256, 4, 2, 64, 512, 2, 1e-6
WIDTH = (HEADS + 2 * KV) * DIM


@pytest.fixture(scope="module")
def sess():
    s = new_session()
    yield s
    s.close()


class Model:
    """Weights of LAYERS decoder layers, Q8_0, in the session's cache."""

    def __init__(self, sess, rng):
        self.linears, self.vectors = [], []
        for layer in range(LAYERS):
            w = {}
            for name, inner, rows in (("qkv", HIDDEN, WIDTH), ("out", HEADS * DIM, HIDDEN), ("gate", HIDDEN, FFN), ("up", HIDDEN, FFN), ("down", FFN, HIDDEN)):
                packed = quantize(oracle(), "orc", (rng.standard_normal((rows, inner)) / np.sqrt(inner)).astype(np.float32), "q8_0")
                w[name] = (sess.weight(f"step:{layer}:{name}", packed, Q8_0, inner, rows), rows)
            self.linears.append(w)
            self.vectors.append({n: sess.to_device((1 + rng.standard_normal(size) / 5).astype(np.float32))
                                 for n, size in (("norm1", HIDDEN), ("norm2", HIDDEN), ("q", DIM), ("k", DIM))})
        self.last = sess.to_device((1 + rng.standard_normal(HIDDEN) / 5).astype(np.float32))


class Run:
    """Buffers of `rows` tokens."""

    def __init__(self, sess, rows):
        self.sess, self.rows = sess, rows
        sizes = {"x": HIDDEN, "y": HIDDEN, "qkv": WIDTH, "q": HEADS * DIM, "k": KV * DIM, "v": KV * DIM, "t": HEADS * DIM, "att": HEADS * DIM, "branch": HIDDEN,
                 "gate": FFN, "up": FFN}
        self.b = {k: sess.alloc(4 * rows * n) for k, n in sizes.items()}

    def linear(self, model, layer, name, to, stage=True, src=None):
        h, _ = model.linears[layer][name]
        code = self.sess.matmul_stage(h, None, self.rows, self.b[to].ptr, _lib.STAGE_MULTIPLY) if stage else self.sess.matmul(h, self.b[src].ptr, self.rows,
                                                                                                                          self.b[to].ptr)
        _lib.check(code, name)

    def free(self):
        for b in self.b.values():
            b.free()


def layers(sess, model, caches, r, cos, sin, adapters, ranges, fused):
    """One pass of all layers over r.b["x"]; ranges [(begin, end, adapter's place, scale)]."""
    rows, b, ck = r.rows, r.b, _lib.check
    p = {k: v.ptr for k, v in b.items()}
    ck(sess.norm_quantize(Q8_0, p["x"], rows, HIDDEN, model.vectors[0]["norm1"].ptr, EPS, False, None, p["y"]), "norm")
    for layer in range(LAYERS):
        v = model.vectors[layer]
        r.linear(model, layer, "qkv", "qkv")
        ck(sess.adapters([(s, e, adapters[a].h, scale) for s, e, a, scale in ranges], p["y"], rows, p["qkv"], WIDTH, p["qkv"]), "adapters")
        q, k, val = p["qkv"], p["qkv"] + 4 * HEADS * DIM, p["qkv"] + 4 * (HEADS + KV) * DIM
        if fused:
            turn = sess.rotation(cos.ptr, sin.ptr, DIM, False, RMS, v["q"].ptr, v["k"].ptr, EPS)
            ck(sess.cache_append_rotated(caches, layer, q, k, val, rows, HEADS, turn, p["q"], ld=WIDTH), "append_rotated")
        else:
            for heads, feature, weight, to in ((HEADS, 0, "q", "q"), (KV, HEADS * DIM, "k", "k")):
                ck(sess.copy_rows(p["qkv"], rows, WIDTH, p["t"], rows, heads * DIM, rows, 0, feature, 0), "copy")
                ck(sess.norm_quantize(0, p["t"], rows * heads, DIM, v[weight].ptr, EPS, False, None, p[to]), "head norm")
                ck(sess.rope(p[to], rows, heads * DIM, heads, cos.ptr, sin.ptr, False), "rope")
            ck(sess.copy_rows(p["qkv"], rows, WIDTH, p["v"], rows, KV * DIM, rows, 0, (HEADS + KV) * DIM, 0), "copy")
            ck(sess.cache_append(caches, layer, p["k"], p["v"], rows), "append")
        ck(sess.cache_attention(caches, layer, p["q"], rows, HEADS, p["att"]), "attention")
        r.linear(model, layer, "out", "branch", False, "att")
        after = model.vectors[layer + 1]["norm1"] if layer + 1 < LAYERS else model.last
        for weight, step in ((v["norm2"], "attention"), (after, "ffn")):
            if step == "ffn":
                r.linear(model, layer, "gate", "gate")
                r.linear(model, layer, "up", "up")
                ck(sess.silu_gate_quantize(Q8_0, p["gate"], p["up"], rows, FFN), "silu gate")
                r.linear(model, layer, "down", "branch")
            if fused:
                ck(sess.residual_norm_quantize(Q8_0, p["x"], p["branch"], rows, HIDDEN, p["x"], p["y"], pre=RMS, pre_weight_ptr=weight.ptr, pre_eps=EPS),
                   "residual norm")
            else:
                ck(sess.pointwise(4, p["x"], p["branch"], rows, HIDDEN), "add")
                ck(sess.norm_quantize(Q8_0, p["x"], rows, HIDDEN, weight.ptr, EPS, False, None, p["y"]), "norm")
    return b["y"].download(np.float32, rows * HIDDEN).reshape(rows, HIDDEN)


def test_decoder_layers(sess):
    """Every output of a prompt's chunks and of the tokens behind it, bit for bit."""
    rng = np.random.default_rng(8)
    model = Model(sess, rng)
    adapters = [Adapter(sess, rng, BF16, 8, HIDDEN, WIDTH), Adapter(sess, rng, F16, 33, HIDDEN, WIDTH)]
    caches = [sess.cache(LAYERS, KV, DIM, 160) for _ in range(2)]
    at = 0
    for rows, ranges in ((37, [(0, 37, 0, 1.0)]), (64, [(0, 10, 0, 1.0), (10, 64, 1, 0.5)]), *((1, [(0, 1, i % 2, 1.0)]) for i in range(4)), (3, [])):
        x = rng.standard_normal((rows, HIDDEN)).astype(np.float32)
        angle = (at + np.arange(rows))[:, None] * 1e4 ** (-np.arange(DIM // 2) / (DIM // 2))
        cos, sin = (sess.to_device(f(angle).astype(np.float32)) for f in (np.cos, np.sin))
        got = []
        for fused, cache in zip((True, False), caches):
            r = Run(sess, rows)
            r.b["x"].upload(x)
            got.append(layers(sess, model, cache, r, cos, sin, adapters, ranges, fused))
            got.append(r.b["x"].download(np.float32, x.size))
            r.free()
        assert np.isfinite(got[0]).all() and np.abs(got[0]).max() > 0.1
        assert np.array_equal(got[0].view(np.uint32), got[2].view(np.uint32)) and np.array_equal(got[1].view(np.uint32), got[3].view(np.uint32))
        at += rows
        for b in (cos, sin):
            b.free()
    assert sess.cache_length(caches[0], 1) == at
    for c in caches:
        sess.cache_destroy(c)
    for a in adapters:
        a.free()


def small_block(sess, rng, modulated):
    linears = {}
    for key, (inner, rows) in zimage.ZBlockWeights.SHAPES.items():
        if key == "modulation" and not modulated:
            continue
        w = (rng.standard_normal((rows, inner)) * 0.02).astype(np.float32)
        linears[key] = (quantize(oracle(), "orc", w, "q8_0"), Q8_0) if key in ("w2", "modulation") else (synth.pack_q5_K(w), 13)
    vectors = {k: (1 + 0.1 * rng.standard_normal(zimage.HEAD_DIM if k in ("q_norm", "k_norm") else zimage.HIDDEN)).astype(np.float32)
               for k in ("attention_norm1", "attention_norm2", "ffn_norm1", "ffn_norm2", "q_norm", "k_norm")}
    if modulated:
        vectors["modulation_bias"] = (0.1 * rng.standard_normal(4 * zimage.HIDDEN)).astype(np.float32)
    return zimage.ZBlockWeights(sess, f"step:z{modulated}", linears, vectors)


@pytest.mark.parametrize("modulated", [True, False])
def test_dit_block(sess, modulated):
    """run() takes the steps between the linears together and gives what ops() gives; an adapter of zero changes nothing, others add up."""
    rows = 70
    rng = np.random.default_rng(30 + modulated)
    weights = small_block(sess, rng, modulated)
    block = zimage.ZBlock(sess, weights, rows)
    x = rng.standard_normal((rows, zimage.HIDDEN)).astype(np.float32)
    cos, sin = (sess.to_device(a) for a in zimage.rotary(rows, 0, 0, False))
    t = sess.to_device(rng.standard_normal((1, zimage.TIME_DIM)).astype(np.float32)) if modulated else None
    xb = sess.to_device(x)
    shapes = zimage.ZBlockWeights.SHAPES
    zero = {k: Adapter(sess, rng, BF16, 4, *shapes[k], up=np.zeros((shapes[k][1], 4))) for k in ("qkv", "out", "w1", "w3", "w2")}
    some = {k: Adapter(sess, rng, BF16, 4, *shapes[k]) for k in ("qkv", "w2")}

    def run(fn):
        xb.upload(x)
        fn()
        return xb.download(np.float32, x.size)

    args = (xb.ptr, cos.ptr, sin.ptr, t.ptr if t else None)
    single = run(lambda: [fn() for _, fn in block.ops(*args)])
    fused = run(lambda: block.run(*args))
    assert np.isfinite(single).all() and np.array_equal(single.view(np.uint32), fused.view(np.uint32))
    nothing = run(lambda: block.run(*args, adapters={k: [(a.h, 1.0)] for k, a in zero.items()}))
    assert np.array_equal(nothing, fused)
    once = run(lambda: block.run(*args, adapters={k: [(a.h, 1.0)] for k, a in some.items()}))
    halves = run(lambda: block.run(*args, adapters={k: [(a.h, 0.5), (a.h, 0.5)] for k, a in some.items()}))
    assert not np.allclose(once, fused, rtol=0, atol=1e-3)
    # (a code of the quantized input of a linear may fall on either side of a tie: the block's own tolerance)
    assert np.abs(once - halves).max() <= 2e-2 * np.abs(once).max()
    for a in [*zero.values(), *some.values()]:
        a.free()
    block.free()
    weights.free()
    for b in (xb, cos, sin, t):
        if b:
            b.free()
