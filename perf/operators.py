"""Performance cases of the operators a chat runs around its linear layers: the
8-bit key/value cache with the attention that reads it, its eviction, and the
log probabilities of tokens.

  attention  pixhip_cache_attention over a cache of n tokens: one row (a decode
             step) or a chunk of rows, causal (the last rows of the cache see
             the keys up to their own) or not; `weigh` also adds up the
             attention weight that each token got, which eviction goes by.
  append     pixhip_cache_append of rows behind the tokens of a conversation, and
             pixhip_cache_read of the blocks they went to.
  evict      pixhip_cache_copy (a conversation forked), pixhip_cache_evict down to
             `keep` blocks per head, and pixhip_cache_read of what is left.
  log_probs  pixhip_log_probs: of given tokens, with the entropy and the most
             likely alternatives, rows of `pad` values more than the vocabulary.

The cache holds keys and values in blocks of 32 tokens of one kv head: a scale
s = max |x| / 127 (32 bits) and codes round(x / s) in 8 bits.

Sizes: 32 heads over 8 kv heads of 128 and chunks of 128 rows are the chat
model's, its cache holds up to 262144 rows, its vocabulary is read in 38 slices
of up to 4096 rows; the others are generic.  `own` false computes the same in
elementary torch operations on the codes and scales as plain tensors.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 32


def listed():
    return [
        # the first step after a one-line prompt: nothing but latency
        {"name": "step_first", "kind": "attention", "rows": 1, "n": 33, "heads": 28, "kv_heads": 4, "dim": 128, "causal": True, "weigh": False},
        # a decode step in the middle of a chat
        {"name": "step_chat", "kind": "attention", "rows": 1, "n": 2501, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "weigh": False},
        # a decode step over a cache that is kept small by eviction, so its weights are counted
        {"name": "step_weighed", "kind": "attention", "rows": 1, "n": 4099, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "weigh": True},
        # a decode step behind a whole book
        {"name": "step_long", "kind": "attention", "rows": 1, "n": 131072, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "weigh": False},
        # one 128-row chunk of a prefill
        {"name": "chunk", "kind": "attention", "rows": 128, "n": 1281, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "weigh": False},
        # a chunk far into a long document, its weights counted for the eviction that follows
        {"name": "chunk_weighed", "kind": "attention", "rows": 128, "n": 16401, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "weigh": True},
        # a decode step's key and value
        {"name": "append_step", "kind": "append", "start": 2500, "rows": 1, "kv_heads": 8, "dim": 128},
        # a whole prompt behind a short system prompt
        {"name": "append_prompt", "kind": "append", "start": 77, "rows": 4099, "kv_heads": 8, "dim": 128},
        # a chat cut down to its 2048 tokens
        {"name": "evict_chat", "kind": "evict", "n": 2565, "keep": 64, "recent": 4, "kv_heads": 8, "dim": 128},
        # a long document cut down to half
        {"name": "evict_long", "kind": "evict", "n": 16401, "keep": 256, "recent": 32, "kv_heads": 8, "dim": 128},
        # the token a step chose, with the alternatives a user is shown
        {"name": "log_probs_step", "kind": "log_probs", "rows": 1, "vocab": 151936, "pad": 0, "top": 20},
        # a given text scored
        {"name": "log_probs_score", "kind": "log_probs", "rows": 512, "vocab": 151936, "pad": 0, "top": 5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention"] * 5 + ["append", "append", "evict", "evict", "log_probs", "log_probs"])
    if kind == "log_probs":
        return {"kind": kind, "rows": rng.choice([1, _log(rng, 1, 512)]), "vocab": _log(rng, 1000, 151936), "pad": rng.choice([0, 0, rng.randint(1, 200)]),
                "top": rng.choice([0, 1, 5, 20, rng.randint(1, 64)])}
    kv, dim = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 80, 96, 128, 128, 128])
    if kind == "append":
        return {"kind": kind, "start": _log(rng, 1, 8192) - 1, "rows": rng.choice([1, 128, _log(rng, 1, 4099)]), "kv_heads": kv, "dim": dim}
    if kind == "evict":
        n = _log(rng, 64, 16401)
        blocks = (n + BLOCK - 1) // BLOCK
        keep = rng.randint(1, blocks)
        return {"kind": kind, "n": n, "keep": keep, "recent": rng.randint(1, max(1, keep // 4)), "kv_heads": kv, "dim": dim}
    heads = kv * rng.choice([1, 2, 4, 4, 7, 8])
    use = rng.choice(["step", "step", "few", "chunk", "chunk"])
    rows = {"step": 1, "few": rng.randint(2, 8), "chunk": rng.choice([128, _log(rng, 9, 512)])}[use]
    n = _log(rng, 1, 131072) if use == "step" else rows + _log(rng, 1, 16273) - 1
    while 4.0 * rows * n * heads * dim > 4.0 * 128 * 16401 * 32 * 128:
        n = max(rows, n // 2)
    return {"kind": kind, "rows": rows, "n": n, "heads": heads, "kv_heads": kv, "dim": dim, "causal": use == "step" or rng.random() < 0.8,
            "weigh": rng.random() < 0.4}


# ---- inputs ----


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std


def _keys(g, n, kv, dim):
    """Keys as attention sees them: some channels of a head carry several times the others' magnitude."""
    spread = torch.exp(_normal(g, (kv * dim,), 0.5))
    return _normal(g, (n, kv * dim)) * spread


def _attention_inputs(case, seed):
    g = _generator(seed)
    kv, dim = case["kv_heads"], case["dim"]
    q = _normal(g, (case["rows"], case["heads"] * dim), 1.2)
    return q, _keys(g, case["n"], kv, dim), _normal(g, (case["n"], kv * dim))


def _append_inputs(case, seed):
    g = _generator(seed)
    kv, dim, total = case["kv_heads"], case["dim"], case["start"] + case["rows"]
    return _keys(g, total, kv, dim), _normal(g, (total, kv * dim))


def _evict_inputs(case, seed):
    """Accumulated weights fall off over several orders of magnitude, as attention's do."""
    g = _generator(seed)
    kv, dim, n = case["kv_heads"], case["dim"], case["n"]
    weights = torch.exp(_normal(g, (n, kv), 1.5) + _normal(g, ((n + BLOCK - 1) // BLOCK, kv)).repeat_interleave(BLOCK, 0)[:n])
    return _keys(g, n, kv, dim), _normal(g, (n, kv * dim)), weights


def _log_probs_inputs(case, seed):
    """Logits of a language model: a few tokens stand out, some are banned."""
    g = _generator(seed)
    rows, vocab = case["rows"], case["vocab"]
    x = _normal(g, (rows, vocab + case["pad"]), 2.0)
    far = torch.randint(0, vocab, (rows, 12), generator=g, device="cuda")
    x.scatter_add_(1, far, 8 + _normal(g, far.shape, 2.0))
    x[:, torch.randint(0, vocab, (vocab // 500,), generator=g, device="cuda")] = -math.inf
    ids = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.7, far[:, 0], torch.randint(0, vocab, (rows,), generator=g, device="cuda"))
    return x, ids.to(torch.int32)


# ---- the state of a user's program ----

_streams = []


class _Owner:
    """A session that lives as long as anything that refers to its memory; all sessions run on one stream, in order."""

    def __init__(self):
        from pixelina_amd import Session, _lib
        if not _streams:
            _streams.append(torch.cuda.Stream())
        self.check = _lib.check
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


def _own_cache(owner, case, k, v, weights=None, more=0):
    """A cache of one layer with the rows k, v in it and room for `more`."""
    s = owner.session
    cache = s.cache(1, case["kv_heads"], case["dim"], k.shape[0] + more)
    torch.cuda.synchronize()
    if k.shape[0]:
        owner.check(s.cache_append(cache, 0, k.data_ptr(), v.data_ptr(), k.shape[0], weights_ptr=weights.data_ptr() if weights is not None else None),
                    "pixhip_cache_append")
    s.synchronize()
    return cache


def prepare(case, seed):
    kind = case["kind"]
    state = {"case": case}
    owner = state["owner"] = _Owner() if own else None
    if kind == "log_probs":
        x, ids = _log_probs_inputs(case, seed)
        if own:
            rows, top = case["rows"], case["top"]
            state["x"], state["ids"] = _tensor(owner, x.shape, x), _tensor(owner, ids.shape, ids, "<i4")
            state["out"] = {"log_probs": _tensor(owner, (rows,)), "entropy": _tensor(owner, (rows,))}
            if top:
                state["out"] |= {"top_ids": _tensor(owner, (rows, top), None, "<i4"), "top_log_probs": _tensor(owner, (rows, top))}
        else:
            state["x"], state["ids"] = x, ids
        torch.cuda.synchronize()
        return state
    if kind == "attention":
        q, k, v = _attention_inputs(case, seed)
        if own:
            state["q"], state["cache"] = _tensor(owner, q.shape, q), _own_cache(owner, case, k, v)
            state["out"] = {"out": _tensor(owner, q.shape)}
            if case["weigh"]:
                state["out"]["weights"] = _tensor(owner, (case["n"], case["kv_heads"]))
        else:
            state["q"], state["k"], state["v"] = q, _quantize(k, case), _quantize(v, case)
    elif kind == "append":
        k, v = _append_inputs(case, seed)
        start, first = case["start"], case["start"] // BLOCK * BLOCK
        if own:
            state["k"], state["v"] = (_tensor(owner, t[start:].shape, t[start:]) for t in (k, v))
            state["cache"] = _own_cache(owner, case, k[:start].contiguous(), v[:start].contiguous(), None, case["rows"])
            state["out"] = {"k": _tensor(owner, k[first:].shape), "v": _tensor(owner, v[first:].shape)}
        else:
            # the rows of the block that is not full yet are kept as they came
            state["k"], state["v"] = ((t[first:start], t[start:]) for t in (k, v))
    else:
        k, v, weights = _evict_inputs(case, seed)
        blocks = (case["n"] + BLOCK - 1) // BLOCK
        keep = min(case["keep"], blocks)
        left = case["n"] - (blocks - keep) * BLOCK
        if own:
            state["cache"] = _own_cache(owner, case, k, v, weights)
            state["work"] = owner.session.cache(1, case["kv_heads"], case["dim"], case["n"])
            state["left"] = left
            state["out"] = {"kept": _tensor(owner, (case["kv_heads"], keep), None, "<i4"), "k": _tensor(owner, (left, k.shape[1])),
                            "v": _tensor(owner, (left, k.shape[1])), "weights": _tensor(owner, (left, case["kv_heads"]))}
        else:
            state["k"], state["v"], state["weights"] = _quantize(k, case), _quantize(v, case), weights
    torch.cuda.synchronize()
    return state


# ---- one pass ----


def run(state):
    if own:
        return _run_own(state)
    return {"attention": _attention_plain, "append": _append_plain, "evict": _evict_plain, "log_probs": _log_probs_plain}[state["case"]["kind"]](state)


def _run_own(state):
    case, out, check = state["case"], state["out"], state["owner"].check
    s, kind = state["owner"].session, case["kind"]
    if kind == "log_probs":
        check(s.log_probs(state["x"].data_ptr(), case["rows"], case["vocab"], state["ids"].data_ptr(), out["log_probs"].data_ptr(),
                          out["entropy"].data_ptr(), case["top"], out["top_ids"].data_ptr() if case["top"] else None,
                          out["top_log_probs"].data_ptr() if case["top"] else None, ld=case["vocab"] + case["pad"]), "pixhip_log_probs")
        return out
    cache = state["cache"]
    if kind == "attention":
        # decay 0: the weights of this call alone
        check(s.cache_attention(cache, 0, state["q"].data_ptr(), case["rows"], case["heads"], out["out"].data_ptr(), causal=case["causal"],
                                weigh=case["weigh"], decay=0.0), "pixhip_cache_attention")
        if case["weigh"]:
            check(s.cache_read(cache, 0, 0, case["n"], weights_ptr=out["weights"].data_ptr()), "pixhip_cache_read")
        return out
    if kind == "append":
        start, first = case["start"], case["start"] // BLOCK * BLOCK
        check(s.cache_truncate(cache, 0, start), "pixhip_cache_truncate")
        check(s.cache_append(cache, 0, state["k"].data_ptr(), state["v"].data_ptr(), case["rows"]), "pixhip_cache_append")
        check(s.cache_read(cache, 0, first, start + case["rows"] - first, out["k"].data_ptr(), out["v"].data_ptr()), "pixhip_cache_read")
        return out
    work = state["work"]
    check(s.cache_copy(work, cache), "pixhip_cache_copy")
    check(s.cache_evict(work, 0, case["keep"], case["recent"], out["kept"].data_ptr()), "pixhip_cache_evict")
    check(s.cache_read(work, 0, 0, state["left"], out["k"].data_ptr(), out["v"].data_ptr(), out["weights"].data_ptr()), "pixhip_cache_read")
    return out


def _quantize(x, case):
    """Codes [blocks][32][kv_heads][dim] and scales [blocks][kv_heads] of rows x, and their count."""
    n = x.shape[0]
    blocks = torch.zeros((-(-n // BLOCK) * BLOCK, x.shape[1]), device=x.device)
    blocks[:n] = x
    blocks = blocks.reshape(-1, BLOCK, case["kv_heads"], case["dim"])
    scale = (blocks.abs().amax(dim=(1, 3)).double() / 127).float()
    # in 64 bits: a quotient next to a half must not cross it
    codes = torch.round(blocks.double() / scale.double().clamp(min=1e-300)[:, None, :, None]).to(torch.int8)
    return codes, scale, n


def _values(codes, scale, n):
    """The rows that codes and scales stand for: [n][kv_heads][dim]."""
    return (codes.float() * scale[:, None, :, None]).flatten(0, 1)[:n]


def _attention_plain(state):
    case = state["case"]
    rows, n, kv, dim = case["rows"], case["n"], case["kv_heads"], case["dim"]
    group = case["heads"] // kv
    k, v = (_values(*state[t]).transpose(0, 1).contiguous() for t in "kv")
    q = state["q"].reshape(rows, kv, group, dim).permute(1, 0, 2, 3).reshape(kv, rows * group, dim)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(1 / math.sqrt(dim)).reshape(kv, rows, group, n)
    if case["causal"]:
        at = torch.arange(n, device=q.device)
        s.masked_fill_((at[None] > (n - rows + torch.arange(rows, device=q.device))[:, None])[:, None], -math.inf)
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    p /= p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.reshape(kv, rows * group, n), v).reshape(kv, rows, group, dim).permute(1, 0, 2, 3).reshape(rows, -1)
    return {"out": o, "weights": p.sum(dim=(1, 2)).T.contiguous()} if case["weigh"] else {"out": o}


def _append_plain(state):
    case = state["case"]
    return {t: _values(*_quantize(torch.cat(state[t]), case)).flatten(1) for t in "kv"}


def _evict_plain(state):
    case, weights = state["case"], state["weights"]
    n, kv, recent = case["n"], case["kv_heads"], case["recent"]
    blocks = state["k"][1].shape[0]
    keep = min(case["keep"], blocks)
    padded = torch.zeros((blocks * BLOCK, kv), device=weights.device)
    padded[:n] = weights
    padded = padded.reshape(blocks, BLOCK, kv)
    score = padded.double().sum(dim=1)
    score[blocks - min(recent, keep):] = math.inf
    order = torch.sort(score, dim=0, descending=True, stable=True).indices[:keep]
    kept = torch.sort(order, dim=0).values
    left = n - (blocks - keep) * BLOCK
    head = torch.arange(kv, device=weights.device)
    out = {"kept": kept.T.to(torch.int32).contiguous(), "weights": padded.transpose(1, 2)[kept, head].transpose(1, 2).reshape(-1, kv)[:left]}
    for t in "kv":
        codes, scale, _ = state[t]
        chosen = codes.transpose(1, 2)[kept, head].transpose(1, 2)
        out[t] = _values(chosen, scale[kept, head], left).flatten(1)
    return out


def _log_probs_plain(state):
    case, ids = state["case"], state["ids"].long()
    x = state["x"][:, :case["vocab"]]
    shifted = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(dim=1)
    norm = torch.log(total)
    mean = torch.where(e > 0, e * shifted, torch.zeros_like(e)).sum(dim=1) / total
    out = {"log_probs": torch.gather(shifted, 1, ids[:, None])[:, 0] - norm, "entropy": norm - mean}
    if case["top"]:
        # one number that orders by value, then by the lower index
        bits = x.contiguous().view(torch.int32).long()
        rank = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 24) - torch.arange(case["vocab"], device=x.device)
        best = torch.topk(rank, case["top"], dim=1).indices
        out |= {"top_ids": best.to(torch.int32), "top_log_probs": torch.gather(shifted, 1, best) - norm[:, None]}
    return out


# ---- what a pass cannot do without ----


def _cache_bytes(n, kv, dim):
    """Keys and values of n tokens with their scales."""
    return 2 * kv * (n * dim + 4 * ((n + BLOCK - 1) // BLOCK))


def work(case):
    kind = case["kind"]
    if kind == "log_probs":
        return {"bytes": 4 * case["rows"] * (case["vocab"] + 3 + 2 * case["top"]), "flops": 0}
    kv, dim = case["kv_heads"], case["dim"]
    if kind == "attention":
        rows, n = case["rows"], case["n"]
        pairs = rows * (n - rows) + rows * (rows + 1) // 2 if case["causal"] else rows * n
        return {"bytes": _cache_bytes(n, kv, dim) + 8 * rows * case["heads"] * dim + (4 * n * kv if case["weigh"] else 0),
                "flops": 4.0 * pairs * case["heads"] * dim}
    if kind == "append":
        # the rows and the part of a block before them come in, codes and their values go out
        first = case["start"] // BLOCK * BLOCK
        total = case["start"] + case["rows"] - first
        return {"bytes": 8 * total * kv * dim + _cache_bytes(total, kv, dim) + 8 * total * kv * dim, "flops": 0}
    n = case["n"]
    blocks = (n + BLOCK - 1) // BLOCK
    keep = min(case["keep"], blocks)
    left = n - (blocks - keep) * BLOCK
    # the fork reads and writes the cache; what is left comes out as values
    return {"bytes": 2 * _cache_bytes(n, kv, dim) + 8 * n * kv + 4 * kv * keep + 8 * left * kv * dim + 4 * left * kv, "flops": 0}


# ---- the same from the definitions, in 64 bits ----


def _held64(x, case):
    """What a cache holds of rows x: [n][kv_heads][dim]."""
    n, kv, dim = x.shape[0], case["kv_heads"], case["dim"]
    out = torch.nn.functional.pad(x.double(), (0, 0, 0, -n % BLOCK)).reshape(-1, BLOCK, kv, dim)
    step = (out.abs().amax(dim=3, keepdim=True).amax(dim=1, keepdim=True) / 127).float().double()
    codes = torch.where(step > 0, out / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(out)).round()
    return (codes * step).reshape(-1, kv, dim)[:n]


def _attention64(case, seed):
    q, k, v = _attention_inputs(case, seed)
    rows, n, kv, dim = case["rows"], case["n"], case["kv_heads"], case["dim"]
    group = case["heads"] // kv
    out = torch.empty((rows, case["heads"], dim), dtype=torch.float64, device=q.device)
    weights = torch.zeros((n, kv), dtype=torch.float64, device=q.device)
    k, v = _held64(k, case), _held64(v, case)
    seen = torch.full((rows,), n, device=q.device)
    if case["causal"]:
        seen = n - rows + 1 + torch.arange(rows, device=q.device)
    hidden = torch.arange(n, device=q.device)[None] >= seen[:, None]
    for h in range(case["heads"]):
        kh, vh = k[:, h // group], v[:, h // group]
        score = q[:, h * dim:(h + 1) * dim].double() @ kh.T / math.sqrt(dim)
        p = torch.softmax(score.masked_fill(hidden, -math.inf), dim=1)
        out[:, h] = p @ vh
        weights[:, h // group] += p.sum(dim=0)
    return {"out": out.reshape(rows, -1), "weights": weights} if case["weigh"] else {"out": out.reshape(rows, -1)}


def exact(case, seed):
    kind = case["kind"]
    if kind == "attention":
        return _attention64(case, seed)
    if kind == "append":
        first = case["start"] // BLOCK * BLOCK
        return {name: _held64(t[first:], case).flatten(1) for name, t in zip("kv", _append_inputs(case, seed))}
    if kind == "evict":
        k, v, weights = _evict_inputs(case, seed)
        n, kv = case["n"], case["kv_heads"]
        blocks = -(-n // BLOCK)
        keep = min(case["keep"], blocks)
        recent = min(case["recent"], keep)
        sums = torch.stack([weights[b * BLOCK:(b + 1) * BLOCK].double().sum(dim=0) for b in range(blocks)]).tolist()
        kept = []
        for h in range(kv):
            best = sorted(range(blocks - recent), key=lambda b: (-sums[b][h], b))[:keep - recent]
            kept.append(sorted(best) + list(range(blocks - recent, blocks)))
        tokens = torch.tensor([[b * BLOCK + t for b in row for t in range(BLOCK) if b * BLOCK + t < n] for row in kept], device=k.device)
        head = torch.arange(kv, device=k.device)[:, None]
        held = [_held64(t, case)[tokens, head].transpose(0, 1).flatten(1) for t in (k, v)]
        return {"kept": torch.tensor(kept, dtype=torch.int32), "k": held[0], "v": held[1], "weights": weights.double()[tokens, head].T.contiguous()}
    x, ids = _log_probs_inputs(case, seed)
    logp = torch.log_softmax(x[:, :case["vocab"]].double(), dim=1)
    p = torch.exp(logp)
    out = {"log_probs": logp[torch.arange(case["rows"], device=x.device), ids.long()],
           "entropy": -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(dim=1)}
    if case["top"]:
        values, order = torch.sort(logp, dim=1, descending=True, stable=True)
        out |= {"top_ids": order[:, :case["top"]].to(torch.int32), "top_log_probs": values[:, :case["top"]]}
    return out
