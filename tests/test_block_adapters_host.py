"""ZBlock's calls of the session, recorded without a device: which buffers its adapters
have it write, and for how long."""
import types

import pytest

from pixelina_amd import _lib
from pixelina_amd.zimage import ZBlock, ZBlockWeights

ROWS = 3


class Recorder:
    """A session whose calls all succeed: (name, arguments) of each."""

    def __init__(self):
        self.calls, self.allocated, self.freed = [], 0, 0

    def alloc(self, nbytes):
        self.allocated += 1

        def free():
            self.freed += 1
        return types.SimpleNamespace(ptr=self.allocated << 32, nbytes=nbytes, free=free)

    def __getattr__(self, name):
        def call(*args, **kw):
            self.calls.append((name, args))
            return _lib.OK
        return call


def block(**kw):
    s = Recorder()
    vectors = {k: types.SimpleNamespace(ptr=1) for k in ("attention_norm1", "attention_norm2", "ffn_norm1", "ffn_norm2", "q_norm", "k_norm")}
    weights = types.SimpleNamespace(w={k: k for k in ZBlockWeights.SHAPES}, v=vectors, types={k: 13 for k in ZBlockWeights.SHAPES}, modulated=False)
    return s, ZBlock(s, weights, ROWS, **kw)


def products(s, fn):
    """Where the calls of fn() write the fp32 product of the feed-forward part, and what w2's adapters read."""
    s.calls.clear()
    fn()
    writes = [args[5] for name, args in s.calls if name == "silu_gate_quantize"]
    reads = [args[1] for name, args in s.calls if name == "adapters"]
    return writes, reads


def test_the_product_is_written_for_the_calls_that_read_it():
    s, b = block()
    args, adapters = (1, 2, 3), {"w2": [(77, 1.0)]}
    assert products(s, lambda: b.run(*args)) == ([None], [])
    (first,), reads = products(s, lambda: b.run(*args, adapters=adapters))
    assert first and reads == [first]
    assert products(s, lambda: b.run(*args)) == ([None], [])
    assert products(s, lambda: [fn() for _, fn in b.ops(*args)]) == ([None], [])
    assert products(s, lambda: b.run(*args, adapters={"w2": []})) == ([None], [])
    held = s.allocated
    assert products(s, lambda: b.run(*args, adapters=adapters)) == ([first], [first]) and s.allocated == held
    b.free()
    assert s.freed == s.allocated


@pytest.mark.parametrize("adapters", [None, {"w2": [(77, 1.0)]}, {"qkv": [(77, 1.0)]}])
def test_a_kept_product_is_always_written(adapters):
    s, b = block(keep_gated=True)
    writes, _ = products(s, lambda: b.run(1, 2, 3, adapters=adapters))
    assert writes == [b.gated.ptr]
    assert products(s, lambda: [fn() for _, fn in b.ops(1, 2, 3)])[0] == [b.gated.ptr]


@pytest.mark.parametrize("key", ["modulation", "ffn", "W1"])
def test_adapters_of_another_linear_are_refused(key):
    s, b = block()
    s.calls.clear()
    with pytest.raises(ValueError, match=key):
        b.run(1, 2, 3, adapters={"w1": [(77, 1.0)], key: [(78, 1.0)]})
    assert not s.calls


def test_no_adapters_of_another_linear_are_none():
    s, b = block()
    b.run(1, 2, 3, adapters={k: [] for k in ZBlockWeights.SHAPES})
    assert s.calls and "adapters" not in [name for name, _ in s.calls]
