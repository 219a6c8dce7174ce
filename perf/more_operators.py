"""Performance cases of what a transformer block does around its quantized linear
layers, and of adapters beside them.

  norms     pixhip_residual_norm_quantize: the norm of a block's output, its gate and
            scale, the residual sum and the norm (and modulation) in front of the
            next linear layers, in one pass.
  heads     pixhip_split_heads: q, k and v out of the rows of a fused projection,
            the heads of q and k normalized and rotated.
  append    pixhip_cache_append_rotated: the same with keys and values appended to
            the 8-bit cache on the way, and pixhip_cache_read of the blocks that
            they went to.
  adapters  pixhip_adapters: low-rank adapters of the requests of a batch added to
            the output of the linear layer that they share.

Sizes: 4608 rows of 3840 or 30 heads of 128, a feed-forward part of 10240 are the
image model's block, 8448 rows of 4096 the edit model's, 32 heads over 8 kv heads of
128 and chunks of 128 rows the chat model's; the others are generic.  `own` false
computes the same in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 32
EPS = 1e-6
NORMS = {"none": 0, "rms": 1, "layer": 2}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step's attention output added and normalized for the feed-forward part: nothing but latency
        {"name": "norms_step", "kind": "norms", "rows": 1, "inner": 4096, "post": "none", "pre": "rms", "gate": False, "modulated": False,
         "target": 0, "scale": 1.0},
        # the image model's block: both norms, gate and modulation
        {"name": "norms_image", "kind": "norms", "rows": 4608, "inner": 3840, "post": "rms", "pre": "rms", "gate": True, "modulated": True,
         "target": 0, "scale": 1.0},
        # the edit model's: parameters of their own for the reference image's rows
        {"name": "norms_edit", "kind": "norms", "rows": 8448, "inner": 4096, "post": "none", "pre": "layer", "gate": True, "modulated": True,
         "target": 4352, "scale": 1.0},
        # a decode step's fused projection
        {"name": "append_step", "kind": "append", "start": 2500, "rows": 1, "heads": 32, "kv_heads": 8, "dim": 128, "norm": "rms", "rotary": 128,
         "interleaved": False},
        # seven drafted tokens; heads of an odd size of which a part turns
        {"name": "append_draft", "kind": "append", "start": 1021, "rows": 7, "heads": 14, "kv_heads": 2, "dim": 90, "norm": "none", "rotary": 46,
         "interleaved": True},
        # a whole prompt behind a short system prompt
        {"name": "append_prompt", "kind": "append", "start": 77, "rows": 4099, "heads": 32, "kv_heads": 8, "dim": 128, "norm": "rms", "rotary": 128,
         "interleaved": False},
        # the captions of an image
        {"name": "heads_text", "kind": "heads", "rows": 333, "heads": 20, "kv_heads": 5, "dim": 80, "norm": "none", "rotary": 80, "interleaved": False},
        # the image model's joint sequence
        {"name": "heads_image", "kind": "heads", "rows": 4608, "heads": 30, "kv_heads": 30, "dim": 128, "norm": "rms", "rotary": 128,
         "interleaved": True},
        # one request's decode step
        {"name": "adapters_step", "kind": "adapters", "columns": 1, "inner": 4096, "rows": 4096, "type": "bf16", "requests": 1, "adapters": 1,
         "rank": 16, "ranks": 1, "bare": False},
        # a decode step of 64 requests that share 9 adapters of several ranks, some without any
        {"name": "adapters_batch", "kind": "adapters", "columns": 64, "inner": 3584, "rows": 18944, "type": "f16", "requests": 64, "adapters": 9,
         "rank": 8, "ranks": 4, "bare": True},
        # five prompts of unequal length in one batch, adapters as their trainer stored them
        {"name": "adapters_prompt", "kind": "adapters", "columns": 1501, "inner": 4096, "rows": 6144, "type": "f32", "requests": 5, "adapters": 3,
         "rank": 16, "ranks": 2, "bare": False},
        # a style adapter on the image model's feed-forward part
        {"name": "adapters_image", "kind": "adapters", "columns": 4608, "inner": 3840, "rows": 10240, "type": "bf16", "requests": 1, "adapters": 1,
         "rank": 64, "ranks": 1, "bare": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norms", "append", "heads", "adapters", "adapters"])
    if kind == "norms":
        rows, inner = rng.choice([1, _log(rng, 1, 8448), _log(rng, 1, 8448)]), rng.choice([_log(rng, 64, 20480), 4 * _log(rng, 16, 5120), 4096, 3840])
        while rows * inner > 8448 * 4096:
            rows //= 2
        return {"kind": kind, "rows": rows, "inner": inner, "post": rng.choice(["none", "rms", "layer"]), "pre": rng.choice(["rms", "layer", "none"]),
                "gate": rng.random() < 0.5, "modulated": rng.random() < 0.5, "target": rng.choice([0, 0, rng.randint(0, rows)]),
                "scale": rng.choice([1.0, 1.0, 0.22])}
    if kind == "adapters":
        inner, rows, columns = _log(rng, 64, 12288), _log(rng, 64, 18944), rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 4608)])
        while columns * (inner + 2 * rows) > 4608 * (3840 + 2 * 10240):
            columns //= 2
        requests = rng.choice([1, min(columns, rng.randint(1, 8)), min(columns, _log(rng, 1, 128))])
        return {"kind": kind, "columns": columns, "inner": inner, "rows": rows, "type": rng.choice(["f32", "f16", "bf16"]), "requests": requests,
                "adapters": rng.randint(1, min(requests, 12)), "rank": rng.choice([4, 8, 16, rng.randint(1, 32)]), "ranks": rng.randint(1, 3),
                "bare": rng.random() < 0.3}
    kv, dim = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 80, 96, 128, 128, 128, 2 * rng.randint(16, 64)])
    case = {"kind": kind, "rows": rng.choice([1, 128, _log(rng, 1, 4099)]), "heads": kv * rng.choice([1, 2, 4, 4, 7]), "kv_heads": kv, "dim": dim,
            "norm": rng.choice(["none", "rms", "rms", "layer"]), "rotary": rng.choice([dim, dim, dim // 4 * 2]), "interleaved": rng.random() < 0.4}
    if kind == "append":
        case["start"] = _log(rng, 1, 8192) - 1
    return case


# ---- inputs ----


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std


def _norms_inputs(case, seed):
    """A residual stream whose channels differ in magnitude, a block's output, and the parameters of both rows (the targets' first)."""
    g = _generator(seed)
    rows, inner = case["rows"], case["inner"]
    spread = torch.exp(_normal(g, (inner,), 1.0))
    t = {"x": _normal(g, (rows, inner)) * spread * 4, "branch": _normal(g, (rows, inner), 0.7) + 0.1}
    for name in ("post_weight", "pre_weight"):
        t[name] = 1 + _normal(g, (inner,), 0.2)
    for name in ("gate", "modulation"):
        t[name] = _normal(g, (2, inner), 0.5)
    return t


def _tables(case, first, g):
    """Cosines and sines of rows at positions first .. of a text, [rows][rotary / 2]."""
    half = case["rotary"] // 2
    frequency = torch.pow(1e6, -torch.arange(half, device="cuda", dtype=torch.float64) / max(1, half))
    angle = (first + torch.arange(case["rows"], device="cuda", dtype=torch.float64))[:, None] * frequency
    return torch.cos(angle).float(), torch.sin(angle).float()


def _heads_inputs(case, seed):
    """Rows of a fused projection (q, k, v side by side; some channels carry several times the others' magnitude), head norm weights and tables;
    for a cache the keys and values that it holds before."""
    g = _generator(seed)
    heads, kv, dim, start = case["heads"], case["kv_heads"], case["dim"], case.get("start", 0)
    spread = torch.exp(_normal(g, ((heads + 2 * kv) * dim,), 0.5))
    t = {"qkv": _normal(g, (case["rows"], (heads + 2 * kv) * dim)) * spread, "q_weight": 1 + _normal(g, (dim,), 0.2), "k_weight": 1 + _normal(g, (dim,), 0.2)}
    t["cosine"], t["sine"] = _tables(case, start, g)
    if start:
        t["k"], t["v"] = _normal(g, (start, kv * dim)), _normal(g, (start, kv * dim))
    return t


def _requests(case):
    """(first row, end, adapter or -1, scale) of the batch's requests: unequal parts, in order."""
    n, columns = case["requests"], case["columns"]
    cut = [round(columns * (i / n) ** 1.25) if n < columns else i for i in range(n)] + [columns]
    out = []
    for i in range(n):
        adapter = -1 if case["bare"] and i % 5 == 3 else (3 * i + i // 4) % case["adapters"]
        out.append((cut[i], cut[i + 1], adapter, 2.0 - 0.25 * (i % 3)))
    return [r for r in out if r[1] > r[0]]


def _rank(case, adapter):
    """Adapters' ranks: `rank` and its doubles, in turn."""
    return case["rank"] << (adapter % case["ranks"])


def _adapters_inputs(case, seed):
    g = _generator(seed)
    columns, inner, rows = case["columns"], case["inner"], case["rows"]
    spread = torch.exp(_normal(g, (inner,), 0.7))
    t = {"x": _normal(g, (columns, inner)) * spread, "base": _normal(g, (columns, rows), 2.0), "down": [], "up": []}
    for a in range(case["adapters"]):
        t["down"].append(_normal(g, (_rank(case, a), inner), 1 / math.sqrt(inner)).to(DTYPES[case["type"]]))
        t["up"].append(_normal(g, (rows, _rank(case, a)), 0.05).to(DTYPES[case["type"]]))
    return t


# ---- the state of a user's program ----

_streams = []


class _Owner:
    """A session that lives as long as anything that refers to its memory; all sessions run on one stream, in order."""

    def __init__(self):
        from pixelina_amd import Session, _lib
        if not _streams:
            _streams.append(torch.cuda.Stream())
        self.check = _lib.check
        self.types = {"f32": _lib.F32, "f16": _lib.F16, "bf16": _lib.BF16}
        self.session = Session(0)
        self.check(self.session.lib.pixhip_session_set_stream(self.session.handle, _streams[0].cuda_stream), "pixhip_session_set_stream")

    def __del__(self):
        self.session.close()


class _Memory:
    """One buffer of a session, as torch sees it."""

    def __init__(self, owner, shape, typestr):
        self.owner = owner
        self.buffer = owner.session.alloc(max(4, 4 * int(np.prod(shape))))
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (self.buffer.ptr, False), "version": 2}


def _tensor(owner, shape, values=None, typestr="<f4"):
    t = torch.as_tensor(_Memory(owner, shape, typestr), device="cuda")
    if values is not None:
        t.copy_(values)
    return t


def prepare(case, seed):
    kind = case["kind"]
    t = {"norms": _norms_inputs, "heads": _heads_inputs, "append": _heads_inputs, "adapters": _adapters_inputs}[kind](case, seed)
    state = {"case": case, "in": t}
    if not own:
        if kind == "append":
            # the rows of the block that is not full yet are kept as they came
            first = case["start"] // BLOCK * BLOCK
            for name in "kv":
                t[name] = t[name][first:].clone() if case["start"] else torch.zeros((0, case["kv_heads"] * case["dim"]), device="cuda")
        torch.cuda.synchronize()
        return state
    owner = state["owner"] = _Owner()
    s = owner.session
    state["in"] = {name: _tensor(owner, v.shape, v) for name, v in t.items() if not isinstance(v, list)}
    if kind == "norms":
        state["out"] = {"x": _tensor(owner, t["x"].shape)} | ({"y": _tensor(owner, t["x"].shape)} if case["pre"] != "none" else {})
    elif kind == "adapters":
        # each adapter once, as a server keeps them
        state["adapters"] = []
        torch.cuda.synchronize()
        for down, up in zip(t["down"], t["up"]):
            state["adapters"].append(s.adapter(owner.types[case["type"]], down.data_ptr(), up.data_ptr(), down.shape[0], case["inner"], case["rows"]))
        s.synchronize()
        state["ranges"] = [(a, b, state["adapters"][i], scale) for a, b, i, scale in _requests(case) if i >= 0]
        state["out"] = {"y": _tensor(owner, t["base"].shape)}
    else:
        rows, kv, dim = case["rows"], case["kv_heads"], case["dim"]
        i = state["in"]
        norm = NORMS[case["norm"]]
        state["rotation"] = s.rotation(i["cosine"].data_ptr(), i["sine"].data_ptr(), rotary=case["rotary"], interleaved=case["interleaved"], norm=norm,
                                       q_weight_ptr=i["q_weight"].data_ptr() if norm else None, k_weight_ptr=i["k_weight"].data_ptr() if norm else None,
                                       eps=EPS)
        out = state["out"] = {"q": _tensor(owner, (rows, case["heads"] * dim))}
        first = 0
        if kind == "append":
            first = case["start"] // BLOCK * BLOCK
            cache = state["cache"] = s.cache(1, kv, dim, case["start"] + rows)
            torch.cuda.synchronize()
            if case["start"]:
                owner.check(s.cache_append(cache, 0, i["k"].data_ptr(), i["v"].data_ptr(), case["start"]), "pixhip_cache_append")
            s.synchronize()
        for name in "kv":
            out[name] = _tensor(owner, (case.get("start", 0) + rows - first, kv * dim))
    torch.cuda.synchronize()
    return state


# ---- one pass ----


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norms": _norms_own, "heads": _heads_own, "append": _append_own, "adapters": _adapters_own}[kind](state)
    return {"norms": _norms_plain, "heads": _heads_plain, "append": _append_plain, "adapters": _adapters_plain}[kind](state)


def _norms_own(state):
    case, i, out, owner = state["case"], state["in"], state["out"], state["owner"]
    post, pre, target = NORMS[case["post"]], NORMS[case["pre"]], case["target"]
    gate, modulation = (i[t].data_ptr() if wanted else None for t, wanted in (("gate", case["gate"]), ("modulation", case["modulated"] and pre)))
    second = 4 * case["inner"]
    owner.check(owner.session.residual_norm_quantize(
        0, i["x"].data_ptr(), i["branch"].data_ptr(), case["rows"], case["inner"], out["x"].data_ptr(), out["y"].data_ptr() if pre else None,
        post=post, post_weight_ptr=i["post_weight"].data_ptr() if post else None, post_eps=EPS, gate_ptr=gate, scale=case["scale"],
        pre=pre, pre_weight_ptr=i["pre_weight"].data_ptr() if pre else None, pre_eps=EPS, modulation_ptr=modulation, target_begin=target,
        gate_before_ptr=gate + second if gate and target else None, modulation_before_ptr=modulation + second if modulation and target else None),
        "pixhip_residual_norm_quantize")
    return out


def _slices(state):
    """Addresses of q, k and v in the rows of the fused projection, and the rows' stride."""
    case, at = state["case"], state["in"]["qkv"].data_ptr()
    q, kv = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    return (at, at + 4 * q, at + 4 * (q + kv)), q + 2 * kv


def _heads_own(state):
    case, out, owner = state["case"], state["out"], state["owner"]
    (q, k, v), ld = _slices(state)
    owner.check(owner.session.split_heads(q, k, v, case["rows"], case["heads"], case["kv_heads"], case["dim"], state["rotation"], out["q"].data_ptr(),
                                          out["k"].data_ptr(), out["v"].data_ptr(), ld=ld), "pixhip_split_heads")
    return out


def _append_own(state):
    case, out, owner, cache = state["case"], state["out"], state["owner"], state["cache"]
    s, check = owner.session, owner.check
    (q, k, v), ld = _slices(state)
    start, first = case["start"], case["start"] // BLOCK * BLOCK
    check(s.cache_truncate(cache, 0, start), "pixhip_cache_truncate")
    check(s.cache_append_rotated(cache, 0, q, k, v, case["rows"], case["heads"], state["rotation"], out["q"].data_ptr(), ld=ld),
          "pixhip_cache_append_rotated")
    check(s.cache_read(cache, 0, first, start + case["rows"] - first, out["k"].data_ptr(), out["v"].data_ptr()), "pixhip_cache_read")
    return out


def _adapters_own(state):
    case, i, out, owner = state["case"], state["in"], state["out"], state["owner"]
    owner.check(owner.session.adapters(state["ranges"], i["x"].data_ptr(), case["columns"], out["y"].data_ptr(), rows=case["rows"],
                                       base_ptr=i["base"].data_ptr()), "pixhip_adapters")
    return out


def _norm(x, how, weight):
    """The statistics in 64 bits, as all norms of the framework have them; each product rounded to 32."""
    if how == "none":
        return x
    wide = x.double()
    if how == "layer":
        wide = wide - wide.mean(dim=-1, keepdim=True)
    inverse = (1 / torch.sqrt((wide * wide).mean(dim=-1, keepdim=True) + EPS)).float()
    return wide.float() * inverse * weight


def _norms_plain(state):
    case, i = state["case"], state["in"]
    before = (torch.arange(case["rows"], device="cuda") < case["target"]).long()
    add = _norm(i["branch"], case["post"], i["post_weight"])
    if case["gate"]:
        factor = torch.tanh(i["gate"].double()).float()
        add = add * (factor[before] if case["target"] else factor[0])
    if case["scale"] != 1.0:
        add = add * case["scale"]
    out = {"x": i["x"] + add}
    if case["pre"] != "none":
        out["y"] = _norm(out["x"], case["pre"], i["pre_weight"])
        if case["modulated"]:
            factor = 1 + i["modulation"]
            out["y"] = out["y"] * (factor[before] if case["target"] else factor[0])
    return out


def _rotate(x, case, cosine, sine):
    """Pairs of the leading `rotary` values of each head [rows][heads][dim] turned by their row's angles."""
    n = case["rotary"]
    c, s = cosine[:, None], sine[:, None]
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if case["interleaved"] else (x[..., :n // 2], x[..., n // 2:n])
    a, b = a * c - b * s, a * s + b * c
    turned = torch.stack((a, b), dim=-1).flatten(-2) if case["interleaved"] else torch.cat((a, b), dim=-1)
    return torch.cat((turned, x[..., n:]), dim=-1)


def _turned(state):
    case, i = state["case"], state["in"]
    rows, dim = case["rows"], case["dim"]
    q, k, v = torch.split(i["qkv"].reshape(rows, -1, dim), [case["heads"], case["kv_heads"], case["kv_heads"]], dim=1)
    q, k = (_rotate(_norm(x, case["norm"], i[w]), case, i["cosine"], i["sine"]).flatten(1) for x, w in ((q, "q_weight"), (k, "k_weight")))
    return q, k, v.flatten(1)


def _heads_plain(state):
    q, k, v = _turned(state)
    return {"q": q, "k": k, "v": v}


def _held(x, case):
    """What the cache holds of rows x: codes round(x / s) of 8 bits, s = max |x| / 127 of a block of 32 rows and a head."""
    n = x.shape[0]
    blocks = torch.zeros((-(-n // BLOCK) * BLOCK, x.shape[1]), device=x.device)
    blocks[:n] = x
    blocks = blocks.reshape(-1, BLOCK, case["kv_heads"], case["dim"])
    scale = (blocks.abs().amax(dim=(1, 3), keepdim=True).double() / 127).float()
    # in 64 bits: a quotient next to a half must not cross it
    codes = torch.round(blocks.double() / scale.double().clamp(min=1e-300))
    return (codes.float() * scale).reshape(-1, x.shape[1])[:n]


def _append_plain(state):
    case, i = state["case"], state["in"]
    q, k, v = _turned(state)
    return {"q": q, "k": _held(torch.cat((i["k"], k)), case), "v": _held(torch.cat((i["v"], v)), case)}


def _adapters_plain(state):
    case, i = state["case"], state["in"]
    y = i["base"].clone()
    for first, end, adapter, scale in _requests(case):
        if adapter >= 0:
            part = torch.matmul(i["x"][first:end], i["down"][adapter].float().T)
            y[first:end] += torch.matmul(part * scale, i["up"][adapter].float().T)
    return {"y": y}


# ---- what a pass cannot do without ----


def work(case):
    kind = case["kind"]
    if kind == "norms":
        values, pre = case["rows"] * case["inner"], case["pre"] != "none"
        rows = 2 if case["target"] else 1
        vectors = (case["post"] != "none") + pre + rows * (case["gate"] + (pre and case["modulated"]))
        return {"bytes": 4 * ((3 + pre) * values + vectors * case["inner"]), "flops": 12 * values}
    if kind == "adapters":
        inner, rows, width = case["inner"], case["rows"], 4 if case["type"] == "f32" else 2
        used = {a for _, _, a, _ in _requests(case) if a >= 0}
        ranks = sum(_rank(case, a) for a in used)
        served = [(end - first, _rank(case, a)) for first, end, a, _ in _requests(case) if a >= 0]
        return {"bytes": 4 * (sum(n for n, _ in served) * inner + 2 * case["columns"] * rows) + width * ranks * (inner + rows),
                "flops": 2.0 * sum(n * rank for n, rank in served) * (inner + rows)}
    rows, heads, kv, dim = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    read = 4 * rows * ((heads + 2 * kv) * dim + case["rotary"]) + (8 * dim if case["norm"] != "none" else 0)
    flops = rows * (heads + kv) * (3 * case["rotary"] + (6 * dim if case["norm"] != "none" else 0))
    if kind == "heads":
        return {"bytes": read + 4 * rows * (heads + 2 * kv) * dim, "flops": flops}
    # the rows of the block that is open come in as well, codes and scales go out, and come in again as values
    open_rows = case["start"] % BLOCK
    held = open_rows + rows
    codes = 2 * kv * (held * dim + 4 * -(-held // BLOCK))
    return {"bytes": read + 4 * rows * heads * dim + 8 * open_rows * kv * dim + codes + 8 * held * kv * dim, "flops": flops}


# ---- the same from the definitions, in 64 bits ----


def _norm64(x, how, weight):
    if how == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    if how == "none":
        return x
    return x / torch.sqrt(torch.mean(x * x, dim=-1, keepdim=True) + EPS) * weight.double()


def _norms64(case, seed):
    t = _norms_inputs(case, seed)
    out = {"x": torch.empty_like(t["x"], dtype=torch.float64)}
    if case["pre"] != "none":
        out["y"] = torch.empty_like(out["x"])
    for row, (first, end) in enumerate(((case["target"], case["rows"]), (0, case["target"]))):
        add = _norm64(t["branch"][first:end].double(), case["post"], t["post_weight"]) * case["scale"]
        out["x"][first:end] = t["x"][first:end].double() + (add * torch.tanh(t["gate"][row].double()) if case["gate"] else add)
        if "y" in out:
            y = _norm64(out["x"][first:end], case["pre"], t["pre_weight"])
            out["y"][first:end] = y * (1 + t["modulation"][row].double()) if case["modulated"] else y
    return out


def _turn64(x, case, cosine, sine, weight, rounded):
    """Heads [rows][heads][dim]; `rounded`: each operation rounded to 32 bits, which is how keys are defined before their codes are."""
    r = (lambda v: v.float().double()) if rounded else (lambda v: v)
    x = x.double()
    if case["norm"] != "none":
        if case["norm"] == "layer":
            x = x - x.mean(dim=-1, keepdim=True)
        inverse = 1 / torch.sqrt(torch.mean(x * x, dim=-1, keepdim=True) + EPS)
        x = r(r(r(x) * r(inverse)) * weight.double())
    n = case["rotary"]
    at = torch.arange(n // 2, device=x.device)
    first, second = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + n // 2)
    a, b, c, s = x[..., first], x[..., second], cosine.double()[:, None], sine.double()[:, None]
    out = x.clone()
    out[..., first] = r(r(a * c) - r(b * s))
    out[..., second] = r(r(a * s) + r(b * c))
    return out.flatten(1)


def _held64(x, case):
    """What a cache holds of rows x in the order they came."""
    n, kv, dim = x.shape[0], case["kv_heads"], case["dim"]
    out = torch.nn.functional.pad(x.double(), (0, 0, 0, -n % BLOCK)).reshape(-1, BLOCK, kv, dim)
    step = (out.abs().amax(dim=3, keepdim=True).amax(dim=1, keepdim=True) / 127).float().double()
    codes = torch.where(step > 0, out / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(out)).round()
    return (codes * step).reshape(-1, kv * dim)[:n]


def _heads64(case, seed):
    t = _heads_inputs(case, seed)
    heads, kv, dim, start = case["heads"], case["kv_heads"], case["dim"], case.get("start", 0)
    x = t["qkv"].reshape(case["rows"], -1, dim)
    cached = case["kind"] == "append"
    q = _turn64(x[:, :heads], case, t["cosine"], t["sine"], t["q_weight"], False)
    k = _turn64(x[:, heads:heads + kv], case, t["cosine"], t["sine"], t["k_weight"], cached)
    v = x[:, heads + kv:].double().flatten(1)
    if not cached:
        return {"q": q, "k": k, "v": v}
    first = start // BLOCK * BLOCK
    if start:
        k, v = (torch.cat((t[name][first:].double(), new)) for name, new in (("k", k), ("v", v)))
    return {"q": q, "k": _held64(k, case), "v": _held64(v, case)}


def _adapters64(case, seed):
    t = _adapters_inputs(case, seed)
    y = t["base"].double()
    for first, end, adapter, scale in _requests(case):
        if adapter >= 0:
            y[first:end] += (t["x"][first:end].double() @ t["down"][adapter].double().T) @ t["up"][adapter].double().T * scale
    return {"y": y}


def exact(case, seed):
    return {"norms": _norms64, "heads": _heads64, "append": _heads64, "adapters": _adapters64}[case["kind"]](case, seed)
