"""Measured cases of the operators on a paged key/value cache: attention of one
new token (``paged_decode_attention``), attention of prompt and verify chunks
with a sliding window and first tokens that stay visible
(``paged_window_attention``), and eviction of the positions that gathered the
least attention weight (``evict_paged_context``).

A case is a dict of plain values; ``prepare`` makes what a serving loop has in
hand before the call, ``run`` makes one call (the framework's operators when
``own`` is true, elementary torch operations otherwise), ``work`` counts the
bytes and operations one call cannot do without, and ``exact`` restates the
operators in 64 bits, request by request.

Positions of a request are 0 .. length - 1; the query rows of a request are its
last positions.  A key at j is visible to the query at p when j <= p and (no
window, or p - j < window, or j < sinks).  Query head h reads the keys and
values of head h // (heads / kv_heads).  A row that sees no key is zero.
"""

import math

import numpy as np
import torch

own = False

#: query lengths of a case: "one" (a new token each), "same" (q_max rows each), "ragged" (1 .. q_max)
#: context lengths of a case: evenly spread over len_min .. len_max, in an order drawn from the seed


def _decode(name, **kw):
    base = dict(op="decode", requests=1, heads=32, kv_heads=8, head_dim=128, page=16, len_min=1, len_max=1, dtype="bf16",
                pool="joint", window=0, sinks=0, sums=False)
    return dict(base, **kw, **({"name": name} if name else {}))


def _window(name, **kw):
    base = dict(op="window", requests=1, heads=32, kv_heads=8, head_dim=128, page=16, len_min=1, len_max=1, dtype="bf16",
                pool="joint", window=0, sinks=0, q_max=1, q_kind="same")
    return dict(base, **kw, **({"name": name} if name else {}))


def _evict(name, **kw):
    base = dict(op="evict", requests=1, kv_heads=8, head_dim=128, page=16, len_min=1, len_max=1, dtype="bf16", pool="joint",
                budget=1, sinks=4, recent=1, in_place=True)
    return dict(base, **kw, **({"name": name} if name else {}))


def listed():
    return [
        # one user, the first tokens of an answer: latency alone counts
        _decode("decode one short", len_min=201, len_max=201),
        # one user deep in a long document: the cache's length has to be split over the whole GPU
        _decode("decode one long", len_min=49157, len_max=49157, page=64),
        # a serving batch whose context will be evicted: every step also gathers the attention weights
        _decode("decode batch sums", requests=64, len_min=1024, len_max=8192, sums=True),
        # a large batch on an 8-bit cache with one row per slot, five query heads to a key/value head
        _decode("decode batch e4m3", requests=192, heads=40, len_min=512, len_max=4096, page=1, pool="split", dtype="e4m3"),
        # streaming over long contexts: a window and the first tokens, small heads
        _decode("decode window", requests=128, heads=64, head_dim=64, len_min=300, len_max=20000, page=32, window=2048,
                sinks=4),
        # the target verifies 16 drafted tokens and the token before them, as in the 64-request serving step
        _window("verify blocks", requests=24, len_min=512, len_max=4096, q_max=17),
        # prompts of a few hundred tokens each, none cached before, streamed with a window
        _window("prompts ragged", requests=12, heads=16, kv_heads=4, head_dim=64, len_min=40, len_max=1500, q_max=1500,
                q_kind="whole", window=500, sinks=4),
        # a chunk of a long document, windowed
        _window("chunk windowed", len_min=12300, len_max=12300, q_max=4096, window=4000, sinks=16, page=64),
        # chunks of long prompts on an 8-bit cache, every earlier token visible
        _window("chunk e4m3", requests=2, len_min=4100, len_max=6200, q_max=2048, page=64, dtype="e4m3"),
        # one request's cache cut to its budget, in place
        _evict("evict one", len_min=4096, len_max=4096, budget=2048, recent=256),
        # a serving batch's caches cut to their budget, in place
        _evict("evict batch", requests=64, len_min=2000, len_max=8192, budget=2048, recent=512),
        # long 8-bit contexts whose kept rows go to pages of their own (the old pages are shared with other requests)
        _evict("evict long copy", requests=8, len_min=20000, len_max=65000, budget=8192, sinks=16, recent=1024, page=64,
               dtype="e4m3", in_place=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(lo * (hi / lo) ** rng.random() + 0.5))


def draw(rng):
    op = rng.choice(["decode", "decode", "window", "window", "evict"])
    head_dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 10])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 16])
    while heads > 64:
        heads //= 2
        heads -= heads % kv_heads
    page = rng.choice([1, 16, 24, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "e4m3"])
    pool = rng.choice(["joint", "split"])
    len_max = _log_int(rng, 1, 32768)
    len_min = rng.randint(1, len_max)
    sinks = rng.choice([0, 1, 4, 16, 130])
    window = rng.choice([0, _log_int(rng, 1, 8192)])
    # the cache's rows over all requests, so that no drawn case is larger than the largest listed one
    rows = 250000 * 8 // kv_heads
    if op == "decode":
        requests = _log_int(rng, 1, max(1, min(256, rows // len_max)))
        return _decode(None, requests=requests, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, len_min=len_min,
                       len_max=len_max, dtype=dtype, pool=pool, window=window, sinks=sinks, sums=rng.random() < 0.4)
    if op == "window":
        q_max = min(len_max, _log_int(rng, 1, 4096))
        q_kind = rng.choice(["same", "ragged"])
        scores = 32 * 4096 * 12300  # the largest listed case's score values
        requests = _log_int(rng, 1, max(1, min(64, rows // len_max, scores // (heads * q_max * len_max))))
        return _window(None, requests=requests, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                       len_min=max(len_min, q_max), len_max=len_max, dtype=dtype, pool=pool, window=window, sinks=sinks,
                       q_max=q_max, q_kind=q_kind)
    requests = _log_int(rng, 1, max(1, min(64, rows // 2 // len_max)))
    budget = max(1, int(len_max * (0.1 + 0.8 * rng.random())))
    sinks = min(sinks, budget)
    recent = rng.randint(0, budget - sinks)
    return _evict(None, requests=requests, kv_heads=kv_heads, head_dim=head_dim, page=page, len_min=len_min, len_max=len_max,
                  dtype=dtype, pool=pool, budget=budget, sinks=sinks, recent=recent, in_place=rng.random() < 0.6)


# ------------------------------------------------------------------------------------- inputs


def _spread(lo, hi, n):
    """n whole numbers spread evenly over lo .. hi."""
    return np.linspace(lo, hi, n).round().astype(np.int64) if n > 1 else np.array([hi], dtype=np.int64)


def _lengths(case):
    return _spread(case["len_min"], case["len_max"], case["requests"])


def _queries(case, lengths):
    """Query rows per request, in the order of `lengths`."""
    if case["q_kind"] == "whole":
        return lengths.copy()
    if case["q_kind"] == "same":
        return np.minimum(lengths, case["q_max"])
    return np.minimum(lengths, _spread(1, case["q_max"], len(lengths))[::-1])


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    host = np.random.RandomState(int(seed) % (1 << 31))
    order = host.permutation(case["requests"])
    lengths = _lengths(case)
    queries = _queries(case, lengths) if case["op"] == "window" else None
    lengths = lengths[order]
    R, KH, D, page = case["requests"], case["kv_heads"], case["head_dim"], case["page"]
    cols = int(-(-lengths.max() // page))
    used = -(-lengths // page)
    out_cols = -(-case["budget"] // page) if case["op"] == "evict" and not case["in_place"] else 0
    total = int(used.sum()) + R * out_cols
    # page 0 is no request's: the tables' unused entries name it, and an attention must not see that its values are no numbers
    ids = torch.randperm(total, generator=g, device=dev).to(torch.int32) + 1
    first = torch.tensor(np.concatenate([[0], np.cumsum(used)])[:-1], device=dev)
    at = first[:, None] + torch.arange(cols, device=dev)[None]
    live = torch.arange(cols, device=dev)[None] < torch.tensor(used, device=dev)[:, None]
    table = torch.where(live, ids[at.clamp(max=total - 1)], 0).to(torch.int32)
    width = 2 * D if case["pool"] == "joint" else D
    pools = []
    for _ in range(1 if case["pool"] == "joint" else 2):
        pool = torch.randn(total + 1, KH, page, width, generator=g, device=dev, dtype=torch.bfloat16)
        pool[0] = 0.0 if case["op"] == "evict" else math.nan
        pools.append(pool.to(torch.float8_e4m3fn) if case["dtype"] == "e4m3" else pool)
    state = {"case": dict(case), "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev),
             "k": pools[0][..., :D], "v": pools[-1][..., -D:], "max_len": int(lengths.max()), "descales": None}
    if case["op"] != "evict" and case["dtype"] == "e4m3":
        state["descales"] = 0.5 + torch.rand(2, R, KH, generator=g, device=dev)
    if case["op"] == "decode":
        state["q"] = torch.randn(R, case["heads"], D, generator=g, device=dev).to(torch.bfloat16)
        # what earlier steps gathered
        state["sums"] = torch.rand(R, KH, state["max_len"], generator=g, device=dev) if case["sums"] else None
    elif case["op"] == "window":
        queries = queries[order]
        state["cu"] = torch.tensor(np.concatenate([[0], np.cumsum(queries)]), dtype=torch.int32, device=dev)
        state["max_q"] = int(queries.max())
        state["q"] = torch.randn(int(queries.sum()), case["heads"], D, generator=g, device=dev).to(torch.bfloat16)
        # what the plain form reads in place of a ragged batch: each request's rows, and each row's place
        state["rows"] = torch.tensor(np.concatenate([r * state["max_q"] + np.arange(n) for r, n in enumerate(queries)]),
                                     device=dev)
    else:
        # accumulated weights: a few positions hold most of them, and many hold the same small values
        w = torch.rand(R, KH, state["max_len"], generator=g, device=dev)
        state["sums"] = torch.where(w < 0.5, (w * 64).floor() / 64, 1.0 / (1.0001 - w))
        state["out_table"] = None if case["in_place"] else ids[int(used.sum()):].view(R, out_cols).contiguous()
    return state


# ------------------------------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if own:
        from flashmap_b200 import cache_ops
        scale = case["head_dim"] ** -0.5
        if case["op"] == "decode":
            out = cache_ops.paged_decode_attention(state["q"], state["k"], state["v"], state["lengths"], state["table"],
                                                   state["max_len"], scale, window=case["window"], sinks=case["sinks"],
                                                   descales=state["descales"], weight_sums=state["sums"])
            return {"out": out, "sums": state["sums"]}
        if case["op"] == "window":
            out = cache_ops.paged_window_attention(state["q"], state["k"], state["v"], state["cu"], state["lengths"],
                                                   state["table"], state["max_q"], state["max_len"], scale,
                                                   window=case["window"], sinks=case["sinks"], descales=state["descales"])
            return {"out": out}
        kept, lengths, sums = cache_ops.evict_paged_context(state["k"], state["v"], state["lengths"], state["table"],
                                                            state["sums"], case["budget"], sinks=case["sinks"],
                                                            recent=case["recent"], out_block_table=state["out_table"])
        return {"kept": kept, "lengths": lengths, "sums": sums, "k": state["k"], "v": state["v"]}
    return {"decode": _plain_decode, "window": _plain_window, "evict": _plain_evict}[case["op"]](state, case)


def _gathered(pool, table, n):
    """(requests, kv_heads, n, head_dim) rows of a paged pool, whatever the unused entries name."""
    R, cols = table.shape
    x = pool[table.long()].transpose(2, 3)  # requests, cols, page, heads, dim
    return x.reshape(R, cols * pool.shape[2], pool.shape[1], pool.shape[3])[:, :n].transpose(1, 2).float()


def _attend(q, k, v, visible, scale):
    """q (R, KH, rows, D), k and v (R, KH, n, D), visible (R, rows, n): the rows' outputs and weights."""
    s = torch.matmul(q, k.transpose(2, 3)).mul_(scale)
    s.masked_fill_(~visible[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = s.sum(-1, keepdim=True)
    s.div_(torch.where(total == 0, torch.ones_like(total), total))
    return torch.matmul(s, v), s


def _cache(state, case):
    k = _gathered(state["k"], state["table"], state["max_len"])
    v = _gathered(state["v"], state["table"], state["max_len"])
    if state["descales"] is not None:
        k = k * state["descales"][0][:, :, None, None]
        v = v * state["descales"][1][:, :, None, None]
    held = torch.arange(state["max_len"], device=k.device)[None] < state["lengths"][:, None]
    return k.masked_fill_(~held[:, None, :, None], 0.0), v.masked_fill_(~held[:, None, :, None], 0.0)


def _visible(positions, lengths, n, window, sinks):
    j = torch.arange(n, device=lengths.device)
    p = positions[..., None]
    ok = (j <= p) & (j < lengths[:, None, None])
    return ok & ((p - j < window) | (j < sinks)) if window > 0 else ok


def _plain_decode(state, case):
    k, v = _cache(state, case)
    R, H, D = state["q"].shape
    KH = case["kv_heads"]
    q = state["q"].float().view(R, KH, H // KH, D)
    visible = _visible(state["lengths"][:, None] - 1, state["lengths"], state["max_len"], case["window"], case["sinks"])
    out, w = _attend(q, k, v, visible, D ** -0.5)
    if state["sums"] is not None:
        state["sums"] += w.sum(2)
    return {"out": out.view(R, H, D).to(torch.bfloat16), "sums": state["sums"]}


def _plain_window(state, case):
    k, v = _cache(state, case)
    T, H, D = state["q"].shape
    R, KH, Q = case["requests"], case["kv_heads"], state["max_q"]
    G = H // KH
    q = torch.zeros(R * Q, H, D, device=k.device)
    q[state["rows"]] = state["q"].float()
    q = q.view(R, Q, KH, G, D).permute(0, 2, 3, 1, 4).reshape(R, KH, G * Q, D)
    count = state["cu"][1:] - state["cu"][:-1]
    p = state["lengths"][:, None] - count[:, None] + torch.arange(Q, device=k.device)[None]
    visible = _visible(p, state["lengths"], state["max_len"], case["window"], case["sinks"])
    out, _ = _attend(q, k, v, visible.repeat(1, G, 1), D ** -0.5)
    out = out.view(R, KH, G, Q, D).permute(0, 3, 1, 2, 4).reshape(R * Q, H, D)
    return {"out": out[state["rows"]].to(torch.bfloat16)}


def _plain_evict(state, case):
    R, KH, n, budget = case["requests"], case["kv_heads"], state["max_len"], case["budget"]
    L = state["lengths"].long()[:, None, None]
    j = torch.arange(n, device=L.device)[None, None]
    # the first and the last positions come before every other, and positions past the end come last
    rank = torch.where((j < case["sinks"]) | (j >= L - case["recent"]), math.inf, state["sums"])
    rank = torch.where(j < L, rank, -math.inf).expand(R, KH, n)
    best = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    m = best.shape[-1]
    best = torch.where(best < L, best, n).sort(dim=-1).values
    kept = torch.full((R, KH, budget), -1, dtype=torch.int32, device=L.device)
    kept[..., :m] = torch.where(best < n, best, -1).int()
    lengths = state["lengths"].clamp(max=budget)
    sums = torch.zeros(R, KH, budget, device=L.device)
    sums[..., :m] = torch.where(best < n, state["sums"].gather(2, best.clamp(max=n - 1)), 0.0)
    out_table = state["table"] if state["out_table"] is None else state["out_table"]
    r, h, i = (kept >= 0).nonzero(as_tuple=True)
    page = case["page"]
    src, dst = kept[r, h, i].long(), i
    from_page, to_page = state["table"][r, src // page].long(), out_table[r, dst // page].long()
    for pool in (state["k"], state["v"]):
        bits = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
        bits[to_page, h, dst % page] = bits[from_page, h, src % page]
    return {"kept": kept, "lengths": lengths, "sums": sums, "k": state["k"], "v": state["v"]}


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
    lengths = _lengths(case)
    esz = 1 if case["dtype"] == "e4m3" else 2
    row = case["kv_heads"] * case["head_dim"] * 2 * esz
    if case["op"] == "evict":
        moved = np.minimum(lengths, case["budget"]).astype(np.int64)
        if case["in_place"]:  # the first positions stay where they are, and so does a context within its budget
            moved = np.where(lengths <= case["budget"], 0, np.maximum(moved - case["sinks"], 0))
        kept = np.minimum(lengths, case["budget"])
        return {"bytes": float((2 * moved * row + 4 * case["kv_heads"] * (lengths + 2 * kept)).sum()), "flops": 0.0}
    queries = _queries(case, lengths) if case["op"] == "window" else np.ones_like(lengths)
    seen = [_seen(int(L), int(q), case["window"], case["sinks"]) for L, q in zip(lengths, queries)]
    keys, pairs = sum(s[0] for s in seen), sum(s[1] for s in seen)
    q_bytes = 2 * 2 * case["heads"] * case["head_dim"] * int(queries.sum())
    sums = 8 * case["kv_heads"] * keys if case.get("sums") else 0
    return {"bytes": float(keys * row + q_bytes + sums), "flops": 4.0 * pairs * case["heads"] * case["head_dim"]}


# ------------------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    lengths, table, page, D = s["lengths"].tolist(), s["table"].long(), case["page"], case["head_dim"]
    if case["op"] == "evict":
        # what moves is held as it is and whole numbers have no rounding; the kept sums are copies
        first = s["sums"].double().cpu().numpy()
        sums = np.zeros((case["requests"], case["kv_heads"], case["budget"]))
        for r, L in enumerate(lengths):
            n = min(L, case["budget"])
            for h in range(case["kv_heads"]):
                fixed = set(range(min(case["sinks"], L))) | set(range(max(0, L - case["recent"]), L))
                if L > case["budget"]:
                    middle = np.arange(case["sinks"], L - case["recent"])
                    by = middle[np.argsort(-first[r, h, middle], kind="stable")]
                    fixed |= set(by[: case["budget"] - len(fixed)].tolist())
                else:
                    fixed = range(L)
                sums[r, h, :n] = first[r, h, sorted(fixed)]
        return {"kept": None, "lengths": None, "sums": torch.tensor(sums), "k": None, "v": None}
    G = case["heads"] // case["kv_heads"]
    starts = s["cu"].tolist() if case["op"] == "window" else list(range(case["requests"] + 1))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    sums = s["sums"].double().clone() if s.get("sums") is not None else None
    for r, L in enumerate(lengths):
        a, b = starts[r], starts[r + 1]
        j = torch.arange(L, device=table.device)
        k = s["k"][table[r, j // page], :, j % page].double()  # L, KH, D
        v = s["v"][table[r, j // page], :, j % page].double()
        if s["descales"] is not None:
            k, v = k * s["descales"][0, r].double()[:, None], v * s["descales"][1, r].double()[:, None]
        p = torch.arange(L - (b - a), L, device=j.device)[:, None]
        hidden = j[None] > p
        if case["window"] > 0:
            hidden = hidden | ((j[None] <= p - case["window"]) & (j[None] >= case["sinks"]))
        for h in range(case["heads"]):
            score = s["q"][a:b, h].double() @ k[:, h // G].T / math.sqrt(D)
            w = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1)
            out[a:b, h] = w @ v[:, h // G]
            if sums is not None:
                sums[r, h // G, :L] += w.sum(0)
    return {"out": out, "sums": sums} if case["op"] == "decode" else {"out": out}
