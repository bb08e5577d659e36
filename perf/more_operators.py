"""Measured cases of a target's serving step on a paged key/value cache: new
tokens' rows rotated and written (``append_paged_context``), attention over a
cache held in 4 bits, of one new token (``paged_decode_attention_fp4``) and of
prompt and verify chunks (``paged_window_attention_fp4``), and the log
probabilities of given tokens (``token_logprobs``).

A case is a dict of plain values; ``prepare`` makes what a serving loop has in
hand before the call, ``run`` makes one call (the framework's operators when
``own`` is true, elementary torch operations otherwise), ``work`` counts the
bytes and operations one call cannot do without, and ``exact`` restates the
operators in 64 bits.

A 4-bit row of D values is D / 2 bytes of e2m1 codes (value 2 i in the low half
of byte i) and D / 16 e4m3 factors, one for each 16 values: the value is code
times factor.  Rotation: pairs (i, i + rotary / 2), or (2 i, 2 i + 1) where a
case says interleaved, of the first ``rotary`` values of a head.  A key at j is
visible to the query at p when j <= p and (no window, or p - j < window, or j <
sinks).  Query head h reads kv head h // (heads / kv_heads).
"""

import math

import numpy as np
import torch

own = False

#: rows of a case: "one" new token each, "same" (q_max each), "ragged" (1 .. q_max), "whole" (a prompt of which nothing is cached)
#: context lengths: evenly spread over len_min .. len_max, in an order drawn from the seed


def _cached(op, name, kw):
    base = dict(op=op, requests=1, heads=32, kv_heads=8, head_dim=128, page=16, len_min=1, len_max=1, pool="joint", q_max=1,
                q_kind="one")
    return dict(base, **kw, **({"name": name} if name else {}))


def _append(name, **kw):
    return _cached("append", name, dict(dict(dtype="fp4", rotary=kw.get("head_dim", 128), interleaved=False, descales=False,
                                             moved=0), **kw))


def _decode(name, **kw):
    return _cached("decode", name, dict(dict(window=0, sinks=0, descales=False), **kw))


def _window(name, **kw):
    return _cached("window", name, dict(dict(window=0, sinks=0, descales=False, q_kind="same"), **kw))


def _logprobs(name, **kw):
    return dict(dict(op="logprobs", rows=1, vocab=151936, pitch=0, dtype="bf16", top_k=0, temperature=1.0, hidden=0.0), **kw,
                **({"name": name} if name else {}))


def listed():
    return [
        # one user, one new token: latency alone counts
        _append("append one", len_min=1201, len_max=1201),
        # a decoding batch on an 8-bit pool of rows, half of each head rotated
        _append("append batch e4m3", requests=192, heads=40, len_min=512, len_max=4096, page=1, pool="split", dtype="e4m3",
                rotary=64, interleaved=True, descales=True),
        # the prompts of a few requests, none cached before
        _append("append prompts", requests=6, len_min=701, len_max=4800, q_max=4800, q_kind="whole"),
        # one user, the first tokens of an answer
        _decode("decode4 one short", len_min=201, len_max=201),
        # one user deep in a long document
        _decode("decode4 one long", len_min=100003, len_max=100003, page=64, pool="split"),
        # a serving batch
        _decode("decode4 batch", requests=128, len_min=1024, len_max=8192),
        # the target verifies 16 drafted tokens and the token before them
        _window("verify4 blocks", requests=24, len_min=512, len_max=4096, q_max=17),
        # prompts of a few hundred tokens, none cached before, streamed with a window; small heads
        _window("prompts4 ragged", requests=12, heads=16, kv_heads=4, head_dim=64, len_min=40, len_max=1500, q_max=1500,
                q_kind="whole", window=500, sinks=4),
        # chunks of long prompts, every earlier token visible
        _window("chunk4 long", requests=2, len_min=4100, len_max=6200, q_max=2048, page=64, pool="split", descales=True),
        # the token that one user's step just sampled, with a few alternatives
        _logprobs("logprobs one", top_k=5),
        # every row of a verified batch of 64 requests, 17 rows each
        _logprobs("logprobs verify", rows=1088, top_k=20),
        # a prompt's tokens scored at a sampling temperature, in fp32, half of the vocabulary closed; rows padded to a multiple of 64
        _logprobs("logprobs prompt", rows=1999, vocab=32003, pitch=32064, dtype="fp32", temperature=0.7, hidden=0.5),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(lo * (hi / lo) ** rng.random() + 0.5))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "window", "window", "logprobs"])
    if op == "logprobs":
        dtype = rng.choice(["bf16", "fp32"])
        vocab = _log_int(rng, 1000, 262144)
        rows = _log_int(rng, 1, min(4096, 1088 * 151936 * 2 // (vocab * (2 if dtype == "bf16" else 4))))
        return _logprobs(None, rows=rows, vocab=vocab, pitch=rng.choice([0, vocab + rng.randint(0, 100)]), dtype=dtype,
                         top_k=rng.choice([0, 1, 5, 20, 32]), temperature=rng.choice([1.0, 0.6, 1.3]),
                         hidden=rng.choice([0.0, 0.0, 0.8]))
    head_dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 10])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 16])
    while heads > 64:
        heads //= 2
        heads -= heads % kv_heads
    page = rng.choice([1, 16, 24, 32, 64, 128])
    pool = rng.choice(["joint", "split"])
    descales = rng.random() < 0.3
    shape = dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, pool=pool)
    len_max = _log_int(rng, 1, 65536)
    len_min = rng.randint(1, len_max)
    if op == "append":
        dtype = rng.choice(["fp4", "fp4", "bf16", "e4m3"])
        q_kind = rng.choice(["one", "same", "ragged"])
        q_max = 1 if q_kind == "one" else min(len_max, _log_int(rng, 1, 4096))
        requests = _log_int(rng, 1, max(1, min(256, 250000 * 8 // kv_heads // len_max, 600000 // (q_max * (heads + kv_heads)))))
        return _append(None, requests=requests, len_min=max(len_min, q_max), len_max=len_max, q_max=q_max, q_kind=q_kind, dtype=dtype,
                       rotary=rng.choice([0, 32, 64, head_dim]), interleaved=rng.random() < 0.3,
                       descales=descales and dtype != "bf16", moved=rng.choice([0, 0, 5000]), **shape)
    sinks = rng.choice([0, 1, 4, 16, 130])
    window = rng.choice([0, _log_int(rng, 1, 8192)])
    if op == "decode":
        requests = _log_int(rng, 1, max(1, min(256, 500000 * 8 // kv_heads // len_max)))
        return _decode(None, requests=requests, len_min=len_min, len_max=len_max, window=window, sinks=sinks, descales=descales, **shape)
    len_max = min(len_max, 16384)
    q_max = min(len_max, _log_int(rng, 1, 4096))
    scores = 2 * 32 * 2048 * 4200  # the largest listed case's score values
    q_max = max(1, min(q_max, scores // (heads * len_max)))
    requests = _log_int(rng, 1, max(1, min(64, 250000 * 8 // kv_heads // len_max, scores // (heads * q_max * len_max))))
    return _window(None, requests=requests, len_min=max(min(len_min, len_max), q_max), len_max=len_max, q_max=q_max,
                   q_kind=rng.choice(["same", "ragged"]), window=window, sinks=sinks, descales=descales, **shape)


# ------------------------------------------------------------------------------------- 4-bit rows

_CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantised(x):
    """(codes, factors) of fp32 or fp64 rows: the factor of 16 values is their largest magnitude / 6 as e4m3, a code
    the nearest e2m1 value of value / factor; both to even between two."""
    g = x.unflatten(-1, (-1, 16))
    top = g.abs().amax(-1)
    factors = (top / torch.full_like(top, 6.0)).clamp(max=448.0).float().to(torch.float8_e4m3fn)
    f = factors.to(x.dtype)[..., None]
    y = g.abs() / torch.where(f == 0, torch.ones_like(f), f)
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    code = (torch.where(f == 0, 0, code) + 8 * torch.signbit(g)).to(torch.uint8).flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] + 16 * code[..., 1], factors


def _values(codes, factors, dtype):
    """What codes and their factors stand for."""
    table = torch.tensor(_CODES + tuple(-c for c in _CODES), dtype=dtype, device=codes.device)
    halves = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    return (table[halves].unflatten(-1, (-1, 16)) * factors.to(dtype)[..., None]).flatten(-2)


class _Held(dict):
    """Outputs of which 4-bit pools are decoded when they are read: a pass leaves them in 4 bits, as its user does."""

    def __getitem__(self, key):
        held = dict.__getitem__(self, key)
        return _values(*held, torch.bfloat16) if isinstance(held, tuple) else held


# ------------------------------------------------------------------------------------- inputs


def _spread(lo, hi, n):
    """n whole numbers spread evenly over lo .. hi."""
    return np.linspace(lo, hi, n).round().astype(np.int64) if n > 1 else np.array([hi], dtype=np.int64)


def _lengths(case):
    return _spread(case["len_min"], case["len_max"], case["requests"])


def _queries(case, lengths):
    """New rows per request, in the order of `lengths`."""
    if case["q_kind"] == "whole":
        return lengths.copy()
    if case["q_kind"] in ("one", "same"):
        return np.minimum(lengths, case["q_max"])
    return np.minimum(lengths, _spread(1, case["q_max"], len(lengths))[::-1])


def _prepare_logprobs(case, g):
    dev, n, V = g.device, case["rows"], case["vocab"]
    pitch = case["pitch"] or V
    x = torch.randn(n, pitch, generator=g, device=dev) * 2.5
    likely = torch.randint(0, V, (n, 24), generator=g, device=dev)
    x.scatter_reduce_(1, likely, 4.0 + 3.0 * torch.randn(n, 24, generator=g, device=dev), "amax")  # an id may come twice
    tokens = torch.where(torch.rand(n, generator=g, device=dev) < 0.7, likely[:, 0], likely[:, 1] // 2)
    if case["hidden"]:  # tokens that the sampler may not choose, but the given ones
        closed = torch.rand(V, generator=g, device=dev) < case["hidden"]
        closed[tokens] = False
        x[:, :V].masked_fill_(closed, -math.inf)
    x[:, V:] = math.nan  # padding is no token
    return {"case": dict(case), "logits": x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)[:, :V],
            "tokens": tokens}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    if case["op"] == "logprobs":
        return _prepare_logprobs(case, g)
    host = np.random.RandomState(int(seed) % (1 << 31))
    order = host.permutation(case["requests"])
    lengths = _lengths(case)
    queries = _queries(case, lengths)[order]
    lengths = lengths[order]
    R, KH, D, page = case["requests"], case["kv_heads"], case["head_dim"], case["page"]
    cols = int(-(-lengths.max() // page))
    used = -(-lengths // page)
    total = int(used.sum())
    # page 0 is no request's: the tables' unused entries name it, and an attention must not see that its values are no numbers
    ids = torch.randperm(total, generator=g, device=dev).to(torch.int32) + 1
    first = torch.tensor(np.concatenate([[0], np.cumsum(used)])[:-1], device=dev)
    at = first[:, None] + torch.arange(cols, device=dev)[None]
    live = torch.arange(cols, device=dev)[None] < torch.tensor(used, device=dev)[:, None]
    state = {"case": dict(case), "table": torch.where(live, ids[at.clamp(max=total - 1)], 0).to(torch.int32),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev), "max_len": int(lengths.max()),
             "max_q": int(queries.max()), "descales": None, "k_scales": None, "v_scales": None,
             "cu": torch.tensor(np.concatenate([[0], np.cumsum(queries)]), dtype=torch.int32, device=dev)}
    if case["descales"]:
        state["descales"] = 0.5 + torch.rand(2, R, KH, generator=g, device=dev)
    pools = []
    for _ in range(1 if case["pool"] == "joint" else 2):
        pool = torch.randn(total + 1, KH, page, 2 * D if case["pool"] == "joint" else D, generator=g, device=dev, dtype=torch.bfloat16)
        pools.append(pool)
    kind = case.get("dtype", "fp4")
    if kind == "fp4":
        held = [_quantised(pool.float()) for pool in pools]
        for _, factors in held:
            factors[0] = math.nan
        state["k"], state["v"] = held[0][0][..., : D // 2], held[-1][0][..., -(D // 2):]
        state["k_scales"], state["v_scales"] = held[0][1][..., : D // 16], held[-1][1][..., -(D // 16):]
    else:
        pools = [pool.to(torch.float8_e4m3fn) if kind == "e4m3" else pool for pool in pools]
        state["k"], state["v"] = pools[0][..., :D], pools[-1][..., -D:]
    T = int(queries.sum())
    if case["op"] != "append":
        state["q"] = torch.randn(T, case["heads"], D, generator=g, device=dev).to(torch.bfloat16)
        # where the plain form puts a ragged batch's rows
        state["rows"] = torch.tensor(np.concatenate([r * state["max_q"] + np.arange(n) for r, n in enumerate(queries)]),
                                     device=dev)
        return state
    # a layer's projections of the new tokens: queries, keys and values side by side
    H = case["heads"]
    qkv = (2.0 * torch.randn(T, H + 2 * KH, D, generator=g, device=dev)).to(torch.bfloat16)
    state["q"], state["key"], state["value"] = qkv[:, :H], qkv[:, H: H + KH], qkv[:, H + KH:]
    # where contexts were cut the tokens stand further on in the text than in the cache
    state["positions"] = None
    if case["moved"]:
        index = np.concatenate([np.arange(L - n, L) for L, n in zip(lengths, queries)])
        state["positions"] = torch.tensor(index + np.repeat(host.randint(0, case["moved"] + 1, R), queries), device=dev)
    state["rope"] = None
    if case["rotary"]:
        far = state["max_len"] + case["moved"]
        inverse = 1e6 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64, device=dev) / case["rotary"])
        angle = torch.arange(far, dtype=torch.float64, device=dev)[:, None] * inverse
        state["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float()
    return state


# ------------------------------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if own:
        from flashmap_b200 import cache_ops, ops
        if case["op"] == "logprobs":
            got = ops.token_logprobs(state["logits"], state["tokens"], top_k=case["top_k"], temperature=case["temperature"])
            return {"logprobs": got.logprobs, "entropy": got.entropy, "top_ids": got.top_ids, "top_logprobs": got.top_logprobs}
        if case["op"] == "append":
            q = cache_ops.append_paged_context(state["key"], state["value"], state["k"], state["v"], state["lengths"],
                                               state["table"], cu_seqlens_q=None if case["q_kind"] == "one" else state["cu"],
                                               query=None if state["rope"] is None else state["q"], rope=state["rope"],
                                               interleaved=case["interleaved"], positions=state["positions"],
                                               k_scales=state["k_scales"], v_scales=state["v_scales"],
                                               descales=state["descales"])
            return _written(state, q)
        scale = case["head_dim"] ** -0.5
        if case["op"] == "decode":
            out = cache_ops.paged_decode_attention_fp4(state["q"], state["k"], state["v"], state["k_scales"], state["v_scales"],
                                                       state["lengths"], state["table"], state["max_len"], scale,
                                                       window=case["window"], sinks=case["sinks"], descales=state["descales"])
        else:
            out = cache_ops.paged_window_attention_fp4(state["q"], state["k"], state["v"], state["k_scales"], state["v_scales"],
                                                       state["cu"], state["lengths"], state["table"], state["max_q"],
                                                       state["max_len"], scale, window=case["window"], sinks=case["sinks"],
                                                       descales=state["descales"])
        return {"out": out}
    return {"append": _plain_append, "decode": _plain_attention, "window": _plain_attention,
            "logprobs": _plain_logprobs}[case["op"]](state, case)


def _written(state, q):
    """What an append leaves: the pools and the rotated queries."""
    if state["k_scales"] is None:
        pools = {"k": state["k"], "v": state["v"]}
    else:
        pools = {"k": (state["k"], state["k_scales"]), "v": (state["v"], state["v_scales"])}
    return _Held(pools if q is None else dict(pools, q=q))


def _rotated(x, rows, interleaved):
    """x (tokens, heads, D) rotated by each token's row (tokens, rotary / 2, 2) of cosines and sines."""
    n = 2 * rows.shape[1]
    cos, sin = rows[:, None, :, 0], rows[:, None, :, 1]
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., : n // 2], x[..., n // 2: n])
    u, w = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1), x[..., n:]], -1)


def _places(state):
    """Request and cache position of every new token."""
    cu = state["cu"].long()
    t = torch.arange(state["key"].shape[0], device=cu.device)
    r = torch.bucketize(t, cu[1:], right=True)
    return r, state["lengths"].long()[r] - cu[r + 1] + t


def _plain_append(state, case):
    r, j = _places(state)
    at = j if state["positions"] is None else state["positions"]
    key, value, q = state["key"].float(), state["value"].float(), None
    if state["rope"] is not None:
        rows = state["rope"][at]
        key = _rotated(key, rows, case["interleaved"])
        q = _rotated(state["q"].float(), rows, case["interleaved"]).to(torch.bfloat16)
    if state["descales"] is not None:
        key, value = key / state["descales"][0][r][..., None], value / state["descales"][1][r][..., None]
    page = case["page"]
    where = (state["table"][r, j // page].long()[:, None], torch.arange(case["kv_heads"], device=r.device)[None], (j % page)[:, None])
    if case["dtype"] == "fp4":
        for x, pool, scales in ((key, state["k"], state["k_scales"]), (value, state["v"], state["v_scales"])):
            codes, factors = _quantised(x)
            pool[where] = codes
            scales.view(torch.uint8)[where] = factors.view(torch.uint8)
    elif case["dtype"] == "e4m3":
        for x, pool in ((key, state["k"]), (value, state["v"])):
            pool.view(torch.uint8)[where] = x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        state["k"][where], state["v"][where] = key.to(torch.bfloat16), value.to(torch.bfloat16)
    return _written(state, q)


def _gathered(state, what, case, dtype):
    """(requests, kv_heads, max_len, head_dim) values of a 4-bit pool, zero past each request's length."""
    R, cols = state["table"].shape
    pages = state["table"].long()
    x = _values(state[what][pages], state[what + "_scales"][pages], dtype)  # requests, cols, heads, page, dim
    x = x.transpose(2, 3).reshape(R, cols * case["page"], case["kv_heads"], case["head_dim"])[:, : state["max_len"]].transpose(1, 2)
    if state["descales"] is not None:
        x = x * state["descales"][0 if what == "k" else 1].to(dtype)[:, :, None, None]
    held = torch.arange(state["max_len"], device=x.device)[None] < state["lengths"][:, None]
    return x.masked_fill(~held[:, None, :, None], 0.0)


def _plain_attention(state, case):
    k, v = _gathered(state, "k", case, torch.float32), _gathered(state, "v", case, torch.float32)
    T, H, D = state["q"].shape
    R, KH, Q, n = case["requests"], case["kv_heads"], state["max_q"], state["max_len"]
    G = H // KH
    q = torch.zeros(R * Q, H, D, device=k.device)
    q[state["rows"]] = state["q"].float()
    q = q.view(R, Q, KH, G, D).permute(0, 2, 3, 1, 4).reshape(R, KH, G * Q, D)
    count = state["cu"][1:] - state["cu"][:-1]
    p = (state["lengths"][:, None] - count[:, None] + torch.arange(Q, device=k.device)[None])[..., None]
    j = torch.arange(n, device=k.device)
    seen = (j <= p) & (j < state["lengths"][:, None, None])
    if case["window"] > 0:
        seen &= (p - j < case["window"]) | (j < case["sinks"])
    s = torch.matmul(q, k.transpose(2, 3)).mul_(D ** -0.5)
    s.view(R, KH, G, Q, n).masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = s.sum(-1, keepdim=True)
    s.div_(torch.where(total == 0, torch.ones_like(total), total))
    out = torch.matmul(s, v).view(R, KH, G, Q, D).permute(0, 3, 1, 2, 4).reshape(R * Q, H, D)
    return {"out": out[state["rows"]].to(torch.bfloat16)}


def _plain_logprobs(state, case):
    y = state["logits"].float() * (1.0 / case["temperature"])
    top = y.amax(-1, keepdim=True)
    d = y - top
    e = d.exp()
    total = e.sum(-1)
    log_total = total.log()
    given = d.gather(1, state["tokens"][:, None])[:, 0] - log_total
    entropy = log_total - (e * torch.where(e == 0, torch.zeros_like(d), d)).sum(-1) / total
    if case["top_k"] == 0:
        ids = state["tokens"].new_empty(y.shape[0], 0)
    else:
        ids = state["logits"].float().sort(dim=-1, descending=True, stable=True).indices[:, : case["top_k"]]
    return {"logprobs": given, "entropy": entropy, "top_ids": ids, "top_logprobs": d.gather(1, ids) - log_total[:, None]}


# ------------------------------------------------------------------------------------- work


def _seen(L, q, window, sinks):
    """(keys that some row sees, (row, key) pairs) of the last q rows of a context of L."""
    p = np.arange(L - q, L, dtype=np.int64)
    if window <= 0:
        return int(L), int((p + 1).sum())
    lo = np.maximum(p - window + 1, 0)
    pairs = p + 1 - lo + np.minimum(lo, sinks)
    edge = int(lo[0])
    return int(L - edge + min(edge, sinks)), int(pairs.sum())


def work(case):
    if case["op"] == "logprobs":
        n, k = case["rows"], case["top_k"]
        values = float(n * case["vocab"])
        return {"bytes": values * (2 if case["dtype"] == "bf16" else 4) + n * (8 + 8 + 12 * k), "flops": 6.0 * values}
    lengths = _lengths(case)
    queries = _queries(case, lengths)
    D, KH, H, T = case["head_dim"], case["kv_heads"], case["heads"], int(queries.sum())
    row = {"fp4": D // 2 + D // 16, "e4m3": D, "bf16": 2 * D}[case.get("dtype", "fp4")]
    if case["op"] == "append":
        q = 4 * H * D if case["rotary"] else 0
        return {"bytes": float(T * (2 * KH * (2 * D + row) + q + 4 * case["rotary"])), "flops": 3.0 * T * (H + KH) * case["rotary"]}
    seen = [_seen(int(L), int(q), case["window"], case["sinks"]) for L, q in zip(lengths, queries)]
    keys, pairs = sum(s[0] for s in seen), sum(s[1] for s in seen)
    return {"bytes": float(keys * KH * 2 * row + 4 * T * H * D), "flops": 4.0 * pairs * H * D}


# ------------------------------------------------------------------------------------- 64 bits


def _grid(x):
    """fp64 rows (n, D) as 4 bits hold them, by the distance to each code."""
    x = x.reshape(x.shape[0], -1, 16)
    f = (x.abs().amax(2, keepdim=True) / 6).clamp(max=448.0).to(torch.float8_e4m3fn).double()
    c = torch.tensor(_CODES, dtype=torch.float64, device=x.device)
    far = (x.abs()[..., None] - f[..., None] * c).abs()
    low = far.argmin(3)  # the lower of two that are as near
    up = (low + 1).clamp(max=7)
    tie = (far.gather(3, low[..., None]) == far.gather(3, up[..., None]))[..., 0] & (low % 2 == 1)
    return (torch.sign(x) * f * c[torch.where(tie, up, low)]).flatten(1)


def _exact_append(s, case):
    dev, D, page = s["key"].device, case["head_dim"], case["page"]
    lengths, cu = s["lengths"].tolist(), s["cu"].tolist()
    if case["dtype"] == "fp4":
        pools = [_values(s["k"], s["k_scales"], torch.float64), _values(s["v"], s["v_scales"], torch.float64)]
    else:
        pools = [s["k"].double(), s["v"].double()]
    if case["rotary"]:
        i = torch.arange(D, device=dev)
        half = case["rotary"] // 2
        pair = i // 2 if case["interleaved"] else i % half
        mate = i ^ 1 if case["interleaved"] else torch.where(i < half, i + half, i - half)
        sign = torch.where(i % 2 == 0 if case["interleaved"] else i < half, -1.0, 1.0).double()
        turned = i < case["rotary"]
        pair, mate = torch.where(turned, pair, 0), torch.where(turned, mate, i)

    def rotate(x, at):
        if not case["rotary"]:
            return x
        c, n = s["rope"][at].double()[:, None, pair, 0], s["rope"][at].double()[:, None, pair, 1]
        return torch.where(turned, x * c + sign * x[..., mate] * n, x)

    queries = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    for r, L in enumerate(lengths):
        a, b = cu[r], cu[r + 1]
        j = torch.arange(L - (b - a), L, device=dev)
        at = j if s["positions"] is None else s["positions"][a:b]
        queries[a:b] = rotate(s["q"][a:b].double(), at)
        for n, x in enumerate((rotate(s["key"][a:b].double(), at), s["value"][a:b].double())):
            if s["descales"] is not None:
                x = x / s["descales"][n, r].double()[:, None]
            if case["dtype"] == "fp4":
                x = _grid(x.reshape(-1, D)).view(x.shape)
            elif case["dtype"] == "e4m3":
                x = x.clamp(-448.0, 448.0)
            pools[n][s["table"][r, j // page].long(), :, j % page] = x
    return {"k": pools[0], "v": pools[1], "q": queries if case["rotary"] else None}


def _exact_logprobs(s, case):
    V, k, n = case["vocab"], case["top_k"], case["rows"]
    tokens = s["tokens"].tolist()
    got = {"logprobs": [], "entropy": [], "top_logprobs": []}
    for i in range(n):
        p = torch.log_softmax(s["logits"][i].double() / case["temperature"], 0)
        got["logprobs"].append(p[tokens[i]])
        got["entropy"].append(-torch.special.xlogy(p.exp(), p.exp()).sum())
        got["top_logprobs"].append(p.topk(k).values if k else p[:0])
    return dict({name: torch.stack(v) for name, v in got.items()}, top_ids=None)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s, case)
    if case["op"] == "logprobs":
        return _exact_logprobs(s, case)
    lengths, starts, page, D = s["lengths"].tolist(), s["cu"].tolist(), case["page"], case["head_dim"]
    G = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for r, L in enumerate(lengths):
        a, b = starts[r], starts[r + 1]
        j = torch.arange(L, device=out.device)
        at = s["table"][r, j // page].long(), slice(None), j % page
        k, v = (_values(s[x][at], s[x + "_scales"][at], torch.float64) for x in ("k", "v"))  # L, KH, D
        if s["descales"] is not None:
            k, v = k * s["descales"][0, r].double()[:, None], v * s["descales"][1, r].double()[:, None]
        p = torch.arange(L - (b - a), L, device=j.device)[:, None]
        hidden = j[None] > p
        if case["window"] > 0:
            hidden = hidden | ((j[None] <= p - case["window"]) & (j[None] >= case["sinks"]))
        for h in range(case["heads"]):
            score = s["q"][a:b, h].double() @ k[:, h // G].T / math.sqrt(D)
            out[a:b, h] = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1) @ v[:, h // G]
    return {"out": out}
