"""The operators on a paged key/value cache against the 64-bit oracle.

Tolerances.  An output is sum_j w_j v_j: the kernels round each softmax
numerator once, to bf16 (8 significant bits: at most 2^-8 of it) or, for e4m3
caches, to f16 (11 bits: 2^-11), and the output once to bf16.  Everything else
is fp32: a score is off by at most 8 partial sums' rounding of 2^-22 of
sum |q k| scale, under 2^-16 for the unit-variance inputs here, and moves a
weight by that share.  So outputs are held to u sum_j w_j |v_j| + 2^-8 |out|
with u = 2^-8 or 2^-11, plus 2^-14 of both, and gathered weights to 2^-16 of the
weight plus the fp32 rounding of the sum they are added to.
"""

import math

import pytest
import torch

from oracle import cache_ops as O

pytestmark = pytest.mark.gpu

DEV = "cuda"
FP8 = torch.float8_e4m3fn


def ops():
    from flashmap_b200 import cache_ops
    return cache_ops


def close(got, want, mag, what, fp8=False):
    err = (got.double().cpu() - want).abs()
    tol = (2.0 ** (-11 if fp8 else -8) + 2.0 ** -14) * mag + (2.0 ** -8 + 2.0 ** -14) * want.abs() + 1e-30
    assert torch.isfinite(got.float()).all(), f"{what}: not finite"
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the tolerance"


def error_word():
    from flashmap_b200.serving_ops import _err
    torch.cuda.synchronize()
    w = _err(torch.device("cuda", torch.cuda.current_device()))
    code = int(w)
    w.zero_()
    return code


def make_cache(g, lengths, KH, D, page, dtype, layout, spare=3):
    """Pools (CPU), table and descales; unused table entries name page 0, whose values are NaN."""
    used = [-(-L // page) for L in lengths]
    cols = max(1, max(used, default=1))
    total = sum(used) + spare + 1
    ids = torch.randperm(total - 1, generator=g) + 1
    table = torch.zeros(len(lengths), cols, dtype=torch.int32)
    at = 0
    for r, n in enumerate(used):
        table[r, :n] = ids[at: at + n].int()
        at += n
    width = 2 * D if layout == "joint" else D
    pools = [torch.randn(total, KH, page, width, generator=g).to(torch.bfloat16) for _ in range(1 if layout == "joint" else 2)]
    for p in pools:
        p[0] = math.nan
    for r, L in enumerate(lengths):  # a page's slots past the length hold anything
        if L % page:
            for p in pools:
                p[table[r, used[r] - 1].item(), :, L % page:] = math.nan
    descales = None
    if dtype == FP8:
        pools = [p.to(FP8) for p in pools]
        descales = 0.5 + torch.rand(2, len(lengths), KH, generator=g)
    return pools, table, descales


def views(pools, D):
    dev = [p.to(DEV) for p in pools]
    return dev, dev[0][..., :D], dev[-1][..., -D:]


def cpu_views(pools, D):
    return pools[0][..., :D], pools[-1][..., -D:]


DECODE = [
    # heads, kv_heads, head_dim, page, dtype, layout, window, sinks, lengths
    (8, 2, 128, 16, "bf16", "joint", 0, 0, [1, 0, 17, 700, 64, 65, 3]),
    (8, 8, 128, 16, "bf16", "split", 0, 0, [33, 129, 2]),
    (10, 2, 64, 24, "bf16", "joint", 0, 0, [257, 1, 600]),
    (16, 1, 128, 1, "bf16", "split", 0, 0, [300, 77]),
    (40, 2, 64, 32, "bf16", "joint", 100, 4, [1000, 99, 100, 101, 104, 105, 0]),
    (8, 2, 128, 16, "bf16", "joint", 1, 0, [1, 2, 500]),
    (8, 2, 128, 128, "bf16", "joint", 130, 200, [5, 150, 331, 900]),
    (8, 2, 128, 16, "e4m3", "joint", 0, 0, [1, 0, 17, 700, 64, 65, 3]),
    (12, 1, 128, 1, "e4m3", "split", 64, 3, [400, 66, 67, 68]),
    (5, 1, 64, 24, "e4m3", "joint", 0, 0, [333, 16, 15]),
    (32, 2, 64, 16, "e4m3", "split", 70, 16, [512, 5]),
]


@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(map(str, c[:8])))
@pytest.mark.parametrize("gather", [False, True])
def test_decode(case, gather):
    H, KH, D, page, dt, layout, window, sinks, lengths = case
    g = torch.Generator().manual_seed(11)
    dtype = FP8 if dt == "e4m3" else torch.bfloat16
    pools, table, descales = make_cache(g, lengths, KH, D, page, dtype, layout)
    q = torch.randn(len(lengths), H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    top = max(lengths)
    before = torch.rand(len(lengths), KH, top + 5, generator=g)
    sums = before.to(DEV) if gather else None
    got = ops().paged_decode_attention(
        q.to(DEV), k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), top, D ** -0.5,
        window=window, sinks=sinks, descales=None if descales is None else descales.to(DEV), weight_sums=sums)
    want, mag, w = O.decode_attention(q, *cpu_views(pools, D), lengths, table, D ** -0.5, window, sinks, descales)
    close(got, want, mag, "decode", dt == "e4m3")
    assert error_word() == 0
    if gather:
        for r, L in enumerate(lengths):
            s = sums[r].double().cpu()
            add = torch.zeros_like(s)
            add[:, :L] = w[r]
            want_s = before[r].double() + add
            assert ((s - want_s).abs() <= 2.0 ** -16 * add + 2.0 ** -22 * want_s).all()
            assert torch.equal(s[:, L:].float(), before[r][:, L:])  # nothing past the length


def test_decode_many_chunks_repeats_bit_for_bit():
    g = torch.Generator().manual_seed(5)
    lengths, KH, H, D, page = [9001, 40, 5000], 2, 8, 128, 16
    pools, table, _ = make_cache(g, lengths, KH, D, page, torch.bfloat16, "joint")
    q = torch.randn(3, H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    L = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    runs = []
    for _ in range(2):
        sums = torch.zeros(3, KH, 9001, device=DEV)
        out = ops().paged_decode_attention(q.to(DEV), k, v, L, table.to(DEV), 9001, D ** -0.5, weight_sums=sums)
        runs.append((out, sums))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    want, mag, w = O.decode_attention(q, *cpu_views(pools, D), lengths, table, D ** -0.5)
    close(runs[0][0], want, mag, "decode")
    total = runs[0][1].double().sum(-1).cpu()  # every head's weights add up to one
    assert torch.allclose(total, torch.full_like(total, H / KH), atol=1e-4)


def test_decode_strided_query_sums_and_other_stream():
    g = torch.Generator().manual_seed(6)
    lengths, KH, H, D = [130, 50], 2, 4, 128
    pools, table, _ = make_cache(g, lengths, KH, D, 16, torch.bfloat16, "joint")
    _, k, v = views(pools, D)
    wide = torch.randn(2, H, 3, D, generator=g).to(torch.bfloat16)
    q = wide.to(DEV)[:, :, 1]
    big = torch.zeros(4, 3 * KH, 200, device=DEV)
    sums = big[::2, 1:1 + KH, :130]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops().paged_decode_attention(q, k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV),
                                           130, D ** -0.5, weight_sums=sums)
    side.synchronize()
    want, mag, w = O.decode_attention(wide[:, :, 1], *cpu_views(pools, D), lengths, table, D ** -0.5)
    close(out, want, mag, "decode")
    assert torch.allclose(sums[1, :, :50].double().cpu(), w[1], atol=1e-5)
    assert float(big[1].abs().max()) == 0.0 and float(big[:, 1 + KH:].abs().max()) == 0.0


def test_decode_extreme_scores():
    """Large scores, rows of zeros, infinite keys' scores of -inf and a query with an infinity."""
    g = torch.Generator().manual_seed(7)
    lengths, KH, D = [80, 80, 80], 1, 128
    for dtype in (torch.bfloat16, FP8):
        pools, table, descales = make_cache(g, lengths, KH, D, 16, dtype, "split")
        q = torch.randn(3, 2, D, generator=g)
        q[0] *= 1e4
        q[1] = 0.0
        q[2] *= 1e-30
        q = q.to(torch.bfloat16)
        _, k, v = views(pools, D)
        out = ops().paged_decode_attention(q.to(DEV), k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV),
                                           table.to(DEV), 80, D ** -0.5,
                                           descales=None if descales is None else descales.to(DEV))
        want, mag, _ = O.decode_attention(q, *cpu_views(pools, D), lengths, table, D ** -0.5, descales=descales)
        # scores of 1e4 carry an fp32 error of up to 1e4 2^-20, which moves weights by a percent
        assert ((out[0].double().cpu() - want[0]).abs() <= 0.03 * mag[0] + 2.0 ** -8 * want[0].abs()).all()
        close(out[1:], want[1:], mag[1:], "decode", dtype == FP8)
    k2 = pools[0].float().clone()
    k2[table[0, :5].long()] = -math.inf  # every score of request 0 is -inf (or the query is zero there)
    k2 = k2.to(torch.bfloat16).to(DEV)
    v2 = pools[1].float().to(torch.bfloat16).to(DEV)
    ones = torch.ones(3, 2, D, dtype=torch.bfloat16, device=DEV)
    out = ops().paged_decode_attention(ones, k2, v2, torch.tensor(lengths, dtype=torch.int32, device=DEV),
                                       table.to(DEV), 80, D ** -0.5)
    assert float(out[0].abs().max()) == 0.0 and torch.isfinite(out.float()).all()


WINDOW = [
    # heads, kv_heads, head_dim, page, dtype, layout, window, sinks, lengths, query rows
    (8, 2, 128, 16, "bf16", "joint", 0, 0, [1, 0, 17, 200, 64, 65, 300], [1, 0, 17, 5, 64, 3, 150]),
    (4, 4, 128, 16, "bf16", "split", 0, 0, [70, 129], [70, 129]),
    (10, 2, 64, 24, "bf16", "joint", 0, 0, [257, 1, 300], [33, 1, 299]),
    (16, 1, 128, 1, "bf16", "split", 0, 0, [300, 77], [17, 17]),
    (20, 1, 64, 32, "bf16", "joint", 100, 4, [500, 99, 100, 101, 104, 0], [200, 99, 100, 17, 1, 0]),
    (8, 2, 128, 16, "bf16", "joint", 1, 0, [1, 2, 200], [1, 2, 100]),
    (8, 2, 128, 16, "bf16", "joint", 1, 1, [300], [280]),
    (8, 2, 128, 128, "bf16", "joint", 130, 200, [5, 150, 331, 700], [5, 20, 331, 17]),
    (2, 1, 128, 16, "bf16", "joint", 37, 70, [900], [500]),
    (8, 2, 128, 16, "bf16", "joint", 0, 0, [20, 100], [30, 101]),  # more rows than positions: the first see nothing
    (8, 2, 128, 16, "e4m3", "joint", 0, 0, [1, 0, 17, 200, 64, 65, 300], [1, 0, 17, 5, 64, 3, 150]),
    (12, 1, 128, 1, "e4m3", "split", 64, 3, [400, 66, 67, 68], [17, 66, 1, 68]),
    (5, 1, 64, 24, "e4m3", "joint", 0, 0, [333, 16, 15], [300, 16, 2]),
    (3, 3, 64, 16, "e4m3", "split", 70, 16, [512, 5], [200, 5]),
]


@pytest.mark.parametrize("case", WINDOW, ids=lambda c: "-".join(map(str, c[:8])))
def test_window(case):
    H, KH, D, page, dt, layout, window, sinks, lengths, rows = case
    g = torch.Generator().manual_seed(12)
    dtype = FP8 if dt == "e4m3" else torch.bfloat16
    pools, table, descales = make_cache(g, lengths, KH, D, page, dtype, layout)
    cu = torch.tensor([0] + rows).cumsum(0).int()
    q = torch.randn(int(cu[-1]), H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    got = ops().paged_window_attention(
        q.to(DEV), k, v, cu.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), max(rows),
        max(lengths), D ** -0.5, window=window, sinks=sinks, descales=None if descales is None else descales.to(DEV))
    want, mag, _ = O.window_attention(q, *cpu_views(pools, D), cu, lengths, table, D ** -0.5, window, sinks, descales)
    close(got, want, mag, "window", dt == "e4m3")
    assert error_word() == 0


@pytest.mark.parametrize("dt", ["bf16", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5)])
def test_window_long(dt, window, sinks):
    """Contexts of thousands: long runs of key tiles, few rows (one verified block) and many."""
    H, KH, D, page, lengths, rows = 4, 1, 128, 16, [5003, 3100], [17, 600]
    g = torch.Generator().manual_seed(13)
    pools, table, descales = make_cache(g, lengths, KH, D, page, FP8 if dt == "e4m3" else torch.bfloat16, "joint")
    cu = torch.tensor([0] + rows).cumsum(0).int()
    q = torch.randn(int(cu[-1]), H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    got = ops().paged_window_attention(
        q.to(DEV), k, v, cu.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), max(rows),
        max(lengths), D ** -0.5, window=window, sinks=sinks, descales=None if descales is None else descales.to(DEV))
    want, mag, _ = O.window_attention(q, *cpu_views(pools, D), cu, lengths, table, D ** -0.5, window, sinks, descales)
    close(got, want, mag, "window", dt == "e4m3")


@pytest.mark.parametrize("dt", ["bf16", "e4m3"])
def test_window_many_short_items(dt):
    """More (row tile, kv head) items than SMs, each too short to be cut; some requests without rows."""
    H, KH, D, page = 16, 8, 64, 16
    lengths = [37 * (i % 13) + (i % 3) for i in range(40)]
    rows = [min(L, 5 * i % 211) for i, L in enumerate(lengths)]
    g = torch.Generator().manual_seed(21)
    pools, table, descales = make_cache(g, lengths, KH, D, page, FP8 if dt == "e4m3" else torch.bfloat16, "joint")
    cu = torch.tensor([0] + rows).cumsum(0).int()
    q = torch.randn(int(cu[-1]), H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    for window, sinks in ((0, 0), (100, 3)):
        got = ops().paged_window_attention(
            q.to(DEV), k, v, cu.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), max(rows),
            max(lengths), D ** -0.5, window=window, sinks=sinks, descales=None if descales is None else descales.to(DEV))
        want, mag, _ = O.window_attention(q, *cpu_views(pools, D), cu, lengths, table, D ** -0.5, window, sinks, descales)
        close(got, want, mag, "window", dt == "e4m3")
    assert error_word() == 0


def test_window_of_one_row_is_decode():
    g = torch.Generator().manual_seed(14)
    lengths, KH, H, D = [130, 50, 1], 2, 8, 128
    pools, table, _ = make_cache(g, lengths, KH, D, 16, torch.bfloat16, "joint")
    _, k, v = views(pools, D)
    q = torch.randn(3, H, D, generator=g).to(torch.bfloat16).to(DEV)
    L = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    a = ops().paged_decode_attention(q, k, v, L, table.to(DEV), 130, D ** -0.5, window=40, sinks=3)
    b = ops().paged_window_attention(q, k, v, torch.arange(4, dtype=torch.int32, device=DEV), L, table.to(DEV), 1, 130,
                                     D ** -0.5, window=40, sinks=3)
    assert torch.allclose(a.float(), b.float(), atol=2e-2)


def test_rows_past_32_bit_offsets():
    """A pool whose last pages lie more than 2^32 bytes, and 2^32 elements, from its start."""
    D, KH, page = 128, 1, 16
    pages, stride = 3, 2_200_000_000  # elements between pages
    pool = torch.empty(2 * stride + KH * page * 2 * D, dtype=torch.bfloat16, device=DEV)
    cache = pool.as_strided((pages, KH, page, 2 * D), (stride, page * 2 * D, 2 * D, 1))
    g = torch.Generator().manual_seed(15)
    host = torch.randn(pages, KH, page, 2 * D, generator=g).to(torch.bfloat16)
    cache.copy_(host.to(DEV))
    lengths, table = [40], torch.tensor([[2, 0, 1]], dtype=torch.int32)
    L = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q = torch.randn(1, 4, D, generator=g).to(torch.bfloat16)
    k, v = cache[..., :D], cache[..., D:]
    want, mag, _ = O.decode_attention(q, host[..., :D], host[..., D:], lengths, table, D ** -0.5)
    close(ops().paged_decode_attention(q.to(DEV), k, v, L, table.to(DEV), 40, D ** -0.5), want, mag, "decode")
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    close(ops().paged_window_attention(q.to(DEV), k, v, cu, L, table.to(DEV), 1, 40, D ** -0.5), want, mag, "window")
    sums = torch.arange(40, dtype=torch.float32, device=DEV).view(1, 1, 40)
    kept, n, _ = ops().evict_paged_context(k, v, L, table.to(DEV), sums, 20, sinks=2, recent=0)
    assert kept[0, 0].tolist() == [0, 1] + list(range(22, 40)) and int(n) == 20
    flat = torch.cat([host[2, 0], host[0, 0], host[1, 0]])[:40]
    now = torch.cat([cache[2, 0], cache[0, 0]])[:20].cpu()
    assert torch.equal(now, flat[kept[0, 0].cpu().long()])


def test_bad_indices_are_reported_and_not_seen():
    g = torch.Generator().manual_seed(16)
    KH, H, D, page = 2, 4, 128, 16
    pools, table, _ = make_cache(g, [64], KH, D, page, torch.bfloat16, "joint")
    _, k, v = views(pools, D)
    q = torch.randn(1, H, D, generator=g).to(torch.bfloat16)
    bad = table.clone()
    bad[0, 1] = 10_000
    L = torch.tensor([64], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    # the oracle on the 48 positions of the other pages
    sub = table[:, [0, 2, 3]]
    want, mag, _ = O.decode_attention(q, *cpu_views(pools, D), [48], sub, D ** -0.5)
    close(ops().paged_decode_attention(q.to(DEV), k, v, L, bad.to(DEV), 64, D ** -0.5), want, mag, "decode")
    assert error_word() == 4
    close(ops().paged_window_attention(q.to(DEV), k, v, cu, L, bad.to(DEV), 1, 64, D ** -0.5), want, mag, "window")
    assert error_word() == 4
    # a length past max_seqlen_k is cut, a negative one is none
    long = torch.tensor([100], dtype=torch.int32, device=DEV)
    want, mag, _ = O.decode_attention(q, *cpu_views(pools, D), [60], table, D ** -0.5)
    close(ops().paged_decode_attention(q.to(DEV), k, v, long, table.to(DEV), 60, D ** -0.5), want, mag, "decode")
    assert error_word() == 4
    none = torch.tensor([-3], dtype=torch.int32, device=DEV)
    out = ops().paged_decode_attention(q.to(DEV), k, v, none, table.to(DEV), 60, D ** -0.5)
    assert float(out.abs().max()) == 0.0 and error_word() == 4
    sums = torch.rand(1, KH, 64, device=DEV)
    kept, n, _ = ops().evict_paged_context(k, v, L, bad.to(DEV), sums, 32, recent=4)
    assert error_word() == 4 and int(n) == 32


EVICT = [
    # kv_heads, head_dim, page, dtype, layout, budget, sinks, recent, lengths
    (2, 128, 16, "bf16", "joint", 40, 4, 8, [100, 40, 41, 39, 0, 1, 700]),
    (1, 64, 24, "bf16", "split", 33, 0, 0, [500, 34, 3]),
    (4, 64, 1, "e4m3", "split", 50, 10, 40, [300, 51, 50]),  # nothing between is kept
    (2, 128, 32, "e4m3", "joint", 1, 0, 0, [5, 1, 2000]),
    (2, 128, 16, "bf16", "joint", 600, 1, 100, [1500, 601, 20]),
]


@pytest.mark.parametrize("case", EVICT, ids=lambda c: "-".join(map(str, c[:8])))
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("values", ["ties", "spread", "odd"])
def test_evict(case, in_place, values):
    KH, D, page, dt, layout, budget, sinks, recent, lengths = case
    g = torch.Generator().manual_seed(17)
    R = len(lengths)
    out_cols = -(-budget // page)
    pools, table, _ = make_cache(g, lengths, KH, D, page, FP8 if dt == "e4m3" else torch.bfloat16, layout,
                                 spare=R * out_cols)
    free = sorted(set(range(1, pools[0].shape[0])) - set(table.flatten().tolist()))
    out_table = torch.tensor(free[: R * out_cols], dtype=torch.int32).view(R, out_cols)
    top = max(lengths)
    sums = torch.rand(R, KH, top + 3, generator=g)
    if values == "ties":
        sums = (sums * 5).floor()
    if values == "odd":
        pick = torch.randint(0, 6, sums.shape, generator=g)
        for i, x in enumerate([math.nan, math.inf, -math.inf, -0.0, 0.0, -1.5]):
            sums[pick == i] = x
    dev, k, v = views(pools, D)
    kept, n, got = ops().evict_paged_context(
        k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), sums.to(DEV), budget, sinks=sinks,
        recent=recent, out_block_table=None if in_place else out_table.to(DEV))
    assert error_word() == 0
    want = O.evict(sums, lengths, budget, sinks, recent)
    to = table if in_place else out_table
    untouched = [p.clone().view(torch.uint8) for p in pools]
    for r, L in enumerate(lengths):
        m = min(L, budget)
        assert int(n[r]) == m
        for h in range(KH):
            assert kept[r, h].tolist() == want[r][h] + [-1] * (budget - m)
            assert torch.equal(got[r, h, :m].cpu().nan_to_num(7.0), sums[r, h, want[r][h]].nan_to_num(7.0))
            assert float(got[r, h, m:].abs().sum()) == 0.0
            for i, j in enumerate(want[r][h]):
                a, b = int(table[r, j // page]), int(to[r, i // page])
                for p, u in zip(pools, untouched):
                    u[b, h, i % page] = p.view(torch.uint8)[a, h, j % page]
    for p, u in zip(dev, untouched):  # the moved rows, and no other byte of the pool
        assert torch.equal(p.view(torch.uint8).cpu(), u)


def test_evict_long_rows():
    """A selection over many positions, where the threshold lies in the last byte of the keys."""
    g = torch.Generator().manual_seed(18)
    L, budget, KH = 50_001, 20_000, 2
    page, D = 16, 64
    cols = -(-L // page)
    table = torch.randperm(cols, generator=g).int().view(1, cols)
    pool = torch.randint(-100, 100, (cols, KH, page, 2 * D), generator=g, dtype=torch.int8).to(torch.bfloat16)
    sums = 1.0 + torch.randint(0, 4000, (1, KH, L), generator=g).float() * 2.0 ** -23
    dev = pool.to(DEV)
    kept, n, _ = ops().evict_paged_context(dev[..., :D], dev[..., D:], torch.tensor([L], dtype=torch.int32, device=DEV),
                                           table.to(DEV), sums.to(DEV), budget, sinks=4, recent=100)
    want = O.evict(sums, [L], budget, 4, 100)
    for h in range(KH):
        assert kept[0, h].tolist() == want[0][h]
        src = torch.tensor(want[0][h])
        i = torch.arange(budget)
        moved = dev[table[0, i // page].long().to(DEV), h, (i % page).to(DEV)].cpu()
        assert torch.equal(moved, pool[table[0, src // page].long(), h, src % page])


def test_decode_in_a_cuda_graph():
    g = torch.Generator().manual_seed(19)
    lengths, KH, H, D = [900, 300], 2, 8, 128
    pools, table, _ = make_cache(g, lengths, KH, D, 16, torch.bfloat16, "joint")
    _, k, v = views(pools, D)
    q = torch.randn(2, H, D, generator=g).to(torch.bfloat16).to(DEV)
    L = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    t = table.to(DEV)
    sums = torch.zeros(2, KH, 900, device=DEV)
    eager = ops().paged_decode_attention(q, k, v, L, t, 900, D ** -0.5, weight_sums=sums)
    want_sums = sums.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops().paged_decode_attention(q, k, v, L, t, 900, D ** -0.5, weight_sums=sums)
    sums.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager) and torch.equal(sums, want_sums)
    L.copy_(torch.tensor([450, 0], dtype=torch.int32))  # lengths are read when the graph runs
    graph.replay()
    want, mag, _ = O.decode_attention(q.cpu(), *cpu_views(pools, D), [450, 0], table, D ** -0.5)
    close(out, want, mag, "decode")


def test_refusals():
    c = ops()
    KH, D, page = 2, 128, 16
    cache = torch.zeros(4, KH, page, 2 * D, dtype=torch.bfloat16, device=DEV)
    k, v = cache[..., :D], cache[..., D:]
    L = torch.tensor([5], dtype=torch.int32, device=DEV)
    t = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 4, D, dtype=torch.bfloat16, device=DEV)
    sums = torch.zeros(1, KH, 5, device=DEV)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)

    def decode(**kw):
        a = dict(query=q, k_cache=k, v_cache=v, seqused_k=L, block_table=t, max_seqlen_k=5, softmax_scale=1.0)
        return c.paged_decode_attention(**dict(a, **kw))

    def chunk(**kw):
        a = dict(query=q, k_cache=k, v_cache=v, cu_seqlens_q=cu, seqused_k=L, block_table=t, max_seqlen_q=1,
                 max_seqlen_k=5, softmax_scale=1.0)
        return c.paged_window_attention(**dict(a, **kw))

    def evict(**kw):
        a = dict(k_cache=k, v_cache=v, seqused_k=L, block_table=t, weight_sums=sums, budget=4)
        return c.evict_paged_context(**dict(a, **kw))

    decode(), chunk(), evict()
    bad = [
        (decode, dict(query=q.float())), (decode, dict(query=q[:, :3])), (decode, dict(query=q[..., :64])),
        (decode, dict(query=q.expand(2, 4, D))), (decode, dict(query=q.cpu())), (decode, dict(window=-1)),
        (decode, dict(sinks=-1)), (decode, dict(weight_sums=sums[..., :4])), (decode, dict(weight_sums=sums.double())),
        (decode, dict(descales=torch.ones(2, 1, KH, device=DEV))), (decode, dict(seqused_k=L.long())),
        (decode, dict(block_table=t.long())), (decode, dict(block_table=t[:0])), (decode, dict(v_cache=v[:2])),
        (decode, dict(k_cache=cache[..., :96], v_cache=cache[..., 96:192])), (decode, dict(k_cache=k.float(), v_cache=v.float())),
        (decode, dict(max_seqlen_k=-1)), (chunk, dict(cu_seqlens_q=cu[:1])), (chunk, dict(cu_seqlens_q=cu.long())),
        (chunk, dict(max_seqlen_q=-1)), (chunk, dict(sinks=-2)), (evict, dict(budget=0)),
        (evict, dict(sinks=3, recent=2)), (evict, dict(sinks=-1)), (evict, dict(weight_sums=sums[:, :1])),
        (evict, dict(out_block_table=t[:, :0])), (evict, dict(out_block_table=t.long())),
    ]
    for fn, kw in bad:
        with pytest.raises(c.OpArgumentError):
            fn(**kw)
    from flashmap_b200._lib import FlashMapError
    odd = torch.zeros(4, KH, page, 2 * D + 4, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(FlashMapError, match="16-byte"):
        decode(k_cache=odd[..., 4:4 + D], v_cache=odd[..., 4 + D:])
    with pytest.raises(FlashMapError, match="in place"):
        evict(out_block_table=t)
    assert error_word() == 0
    # nothing to do
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert decode(query=q[:0], seqused_k=none, block_table=t[:0]).shape == (0, 4, D)
    assert chunk(query=q[:0], cu_seqlens_q=torch.zeros(2, dtype=torch.int32, device=DEV)).shape == (0, 4, D)
    assert evict(seqused_k=none, block_table=t[:0], weight_sums=sums[:0])[0].shape == (0, KH, 4)


def test_evict_slices_past_shared_memory():
    """So many positions of one kv head that a CTA's slice of them does not fit its shared memory."""
    g = torch.Generator().manual_seed(20)
    L, budget, page, D = 600_000, 100_000, 128, 64
    cols = -(-L // page)
    table = torch.randperm(cols, generator=g).int().view(1, cols)
    pool = torch.randint(-100, 100, (cols, 1, page, 2 * D), generator=g, dtype=torch.int8).to(torch.bfloat16)
    sums = torch.randint(0, 50, (1, 1, L), generator=g).float()
    dev = pool.to(DEV)
    kept, n, got = ops().evict_paged_context(dev[..., :D], dev[..., D:], torch.tensor([L], dtype=torch.int32, device=DEV),
                                             table.to(DEV), sums.to(DEV), budget, sinks=4, recent=1000)
    want = O.evict(sums, [L], budget, 4, 1000)
    assert int(n) == budget and kept[0, 0].tolist() == want[0][0]
    src = torch.tensor(want[0][0])
    assert torch.equal(got[0, 0].cpu(), sums[0, 0, src])
    i = torch.arange(budget)
    moved = dev[table[0, i // page].long().to(DEV), 0, (i % page).to(DEV)].cpu()
    assert torch.equal(moved, pool[table[0, src // page].long(), 0, src % page])


@pytest.mark.parametrize("max_len", [64, 4096])
def test_window_bounds_that_run_back_are_reported(max_len):
    """Bounds 0, T, 0, T, .. give the same rows to several requests, more row
    tiles than T rows can have: with shares nothing is done, without them no
    more than fit; the next call is as ever."""
    g = torch.Generator().manual_seed(23)
    KH, H, D, page, T, R = 1, 16, 128, 16, 64, 9
    pools, table, _ = make_cache(g, [max_len], KH, D, page, torch.bfloat16, "joint")
    _, k, v = views(pools, D)
    q = torch.randn(T, H, D, generator=g).to(torch.bfloat16)
    L = torch.tensor([max_len] * R, dtype=torch.int32, device=DEV)
    many = table.expand(R, -1).contiguous().to(DEV)
    back = torch.tensor([0, T] * (R // 2) + [0, T], dtype=torch.int32, device=DEV)
    ops().paged_window_attention(q.to(DEV), k, v, back, L, many, T, max_len, D ** -0.5)
    assert error_word() == 4
    cu = torch.tensor([0] + [T] * R, dtype=torch.int32, device=DEV)
    want, mag, _ = O.window_attention(q, *cpu_views(pools, D), [0, T], [max_len], table, D ** -0.5)
    close(ops().paged_window_attention(q.to(DEV), k, v, cu, L, many, T, max_len, D ** -0.5), want, mag, "window")
    assert error_word() == 0


def test_sums_that_share_memory_are_refused():
    """Sums are added to in place: two rows of them in the same memory would lose additions."""
    c = ops()
    KH, D, page, R = 2, 128, 16, 3
    cache = torch.zeros(4, KH, page, 2 * D, dtype=torch.bfloat16, device=DEV)
    L = torch.full((R,), 5, dtype=torch.int32, device=DEV)
    t = torch.zeros(R, 1, dtype=torch.int32, device=DEV)
    q = torch.zeros(R, 4, D, dtype=torch.bfloat16, device=DEV)

    def decode(sums):
        return c.paged_decode_attention(q, cache[..., :D], cache[..., D:], L, t, 5, 1.0, weight_sums=sums)

    base = torch.zeros(64, device=DEV)
    for strides in ((0, 5, 1), (10, 0, 1), (10, 4, 1), (5, 5, 1), (9, 5, 1)):
        with pytest.raises(c.OpArgumentError, match="share memory"):
            decode(base.as_strided((R, KH, 5), strides))
    assert float(base.abs().max()) == 0.0 and error_word() == 0
    for strides in ((10, 5, 1), (5, 15, 1), (12, 6, 1), (15, 10, 1)):
        base.zero_()
        decode(base.as_strided((R, KH, 5), strides))
        assert torch.allclose(base.as_strided((R, KH, 5), strides), torch.full((R, KH, 5), 0.4, device=DEV))  # 2 heads / 5
    # rows that are only read may share memory
    kept, _, sums = c.evict_paged_context(cache[..., :D], cache[..., D:], L[:1], t[:1], base[:5].expand(1, KH, 5), 4)
    assert kept.shape == (1, KH, 4) and error_word() == 0


RUNS_OF_NOTHING = [
    # heads, kv_heads, lengths, query rows
    # a verify batch padded with requests that hold nothing: items one by one, then in shares
    (8, 8, [37 * i % 290 + 1 if i % 8 == 3 else 0 for i in range(150)], [17] * 150),
    (8, 8, [171 * i % 890 + 11 if i % 8 == 3 else 0 for i in range(200)], [17] * 200),
    # requests that hold nothing, or less than their rows, between chunks
    (16, 8, [2304, 0, 2304, 0, 2304], [800, 1, 900, 1, 1000]),
    (32, 8, [900, 30, 900, 25, 700], [700, 3000, 800, 4000, 600]),
    # long enough for shares among many items, too
    (8, 8, [171 * i % 890 + 911 if i % 8 == 3 else 0 for i in range(200)], [17] * 200),
    (32, 8, [1900, 30, 1900, 25, 1700], [300, 3000, 400, 4000, 200]),
]


@pytest.mark.parametrize("dt", ["bf16", "e4m3"])
@pytest.mark.parametrize("case", RUNS_OF_NOTHING, ids=["padded", "padded_shares", "between", "rows_before", "padded_long", "rows_before_long"])
def test_window_runs_of_items_that_see_nothing(case, dt):
    """Several items of a CTA in a row whose rows see no key, after one that has keys: what it still waits for
    must not be held back by them."""
    H, KH, lengths, rows = case
    D, page = 64, 16
    g = torch.Generator().manual_seed(24)
    pools, table, descales = make_cache(g, lengths, KH, D, page, FP8 if dt == "e4m3" else torch.bfloat16, "joint")
    cu = torch.tensor([0] + rows).cumsum(0).int()
    q = torch.randn(int(cu[-1]), H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    got = ops().paged_window_attention(
        q.to(DEV), k, v, cu.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), max(rows),
        max(lengths), D ** -0.5, descales=None if descales is None else descales.to(DEV))
    assert error_word() == 0
    want, mag, _ = O.window_attention(q, *cpu_views(pools, D), cu, lengths, table, D ** -0.5, descales=descales)
    close(got, want, mag, "window", dt == "e4m3")


def evicted(pools, table, to, want, lengths, budget, page):
    """The pools' bytes with each (request, kv head)'s kept rows moved to the first slots of `to`."""
    now = [p.view(torch.uint8).clone() for p in pools]
    for r, L in enumerate(lengths):
        i = torch.arange(min(L, budget))
        dst = to[r, i // page].long()
        for h, rows in enumerate(want[r]):
            src = torch.tensor(rows, dtype=torch.long)
            for p, u in zip(pools, now):
                u[dst, h, i % page] = p.view(torch.uint8)[table[r, src // page].long(), h, src % page]
    return now


def spread(n, top, odd=37):
    return [odd * i * i % top for i in range(n)]


EVICT_MANY = [
    # kv_heads, head_dim, page, dtype, layout, budget, sinks, recent, in place, lengths
    # 148 (request, kv head) pairs or more, moved by the CTA that chose them
    (4, 128, 16, "bf16", "joint", 50, 4, 8, True, [0, 1, 49, 50, 51, 52, 900] + spread(33, 400)),
    (8, 64, 24, "e4m3", "split", 33, 0, 0, True, [0, 1, 33, 34] + spread(16, 300)),
    (4, 128, 1, "e4m3", "joint", 300, 16, 100, True, [299, 300, 301, 1800] + spread(33, 900)),
    (4, 64, 16, "bf16", "split", 700, 0, 64, True, [700, 701, 2500, 2040] + spread(33, 1100)),
    # one CTA to a pair however long the context, and more slots than its shared memory stages
    (4, 64, 32, "e4m3", "split", 5000, 4, 4900, True, [6000, 5001, 5000, 4999] + spread(52, 100)),
    # copies to other pages: one, two and four CTAs to a pair
    (4, 128, 16, "bf16", "joint", 50, 4, 8, False, [0, 1, 49, 50, 51, 52, 900] + spread(33, 400)),
    (4, 128, 32, "bf16", "split", 600, 4, 100, False, [5000, 4097, 601, 600, 599, 1] + spread(14, 3000)),
    (4, 64, 24, "e4m3", "joint", 1100, 1, 0, False, [9000, 8191, 1101, 1100] + spread(6, 6000)),
    # too few pairs for that: two launches, four CTAs choosing for a pair
    (4, 128, 16, "bf16", "joint", 1100, 4, 300, True, [9000, 1101, 8200, 40, 3000]),
]


@pytest.mark.parametrize("case", EVICT_MANY, ids=lambda c: "-".join(map(str, c[:9])))
@pytest.mark.parametrize("values", ["ties", "spread", "odd"])
def test_evict_many(case, values):
    KH, D, page, dt, layout, budget, sinks, recent, in_place, lengths = case
    g = torch.Generator().manual_seed(25)
    R, out_cols = len(lengths), -(-budget // page)
    pools, table, _ = make_cache(g, lengths, KH, D, page, FP8 if dt == "e4m3" else torch.bfloat16, layout,
                                 spare=0 if in_place else R * out_cols)
    to = table
    if not in_place:
        free = sorted(set(range(1, pools[0].shape[0])) - set(table.flatten().tolist()))
        to = torch.tensor(free, dtype=torch.int32)[torch.randperm(len(free), generator=g)][: R * out_cols].view(R, out_cols)
    sums = torch.rand(R, KH, max(lengths) + 3, generator=g)
    if values == "ties":
        sums = (sums * 5).floor()
    if values == "odd":
        pick = torch.randint(0, 6, sums.shape, generator=g)
        for i, x in enumerate([math.nan, math.inf, -math.inf, -0.0, 0.0, -1.5]):
            sums[pick == i] = x
    dev, k, v = views(pools, D)
    kept, n, got = ops().evict_paged_context(
        k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), sums.to(DEV), budget, sinks=sinks,
        recent=recent, out_block_table=None if in_place else to.to(DEV))
    assert error_word() == 0
    want = O.evict(sums, lengths, budget, sinks, recent)
    assert n.tolist() == [min(L, budget) for L in lengths]
    for r, L in enumerate(lengths):
        m = min(L, budget)
        for h in range(KH):
            assert kept[r, h].tolist() == want[r][h] + [-1] * (budget - m)
            assert torch.equal(got[r, h, :m].cpu().nan_to_num(7.0), sums[r, h, want[r][h]].nan_to_num(7.0))
            assert float(got[r, h, m:].abs().sum()) == 0.0
    for p, u in zip(dev, evicted(pools, table, to, want, lengths, budget, page)):
        assert torch.equal(p.view(torch.uint8).cpu(), u)


VERIFY = [
    # heads, kv_heads, most rows, page, layout, lengths: at most 128 (row, head of the group) rows to a request
    (8, 2, 17, 16, "joint", [1, 2, 17, 100, 128, 129, 200, 256, 257, 300, 384, 385, 500, 513, 640, 800, 1000, 1500, 2049,
                             3000, 4096, 5, 64, 700]),  # one key tile to many, shares and cut items
    (32, 8, 17, 64, "split", [4096, 1, 129, 2500, 257, 60, 900, 385, 3333, 128, 1700, 30, 513, 641, 2048, 1, 200, 300, 256, 4000]),
    (16, 8, 5, 24, "joint", [(97 * i) % 520 + 1 for i in range(60)]),  # many short items, one by one
    (8, 1, 16, 1, "split", [1000, 127, 300, 16]),  # all 128 rows
    (3, 1, 1, 16, "joint", [700, 1, 129, 0, 5000]),  # a new token each
]


@pytest.mark.parametrize("dt", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 5)])
@pytest.mark.parametrize("case", VERIFY, ids=["shares", "groups", "short", "full", "one"])
def test_window_verify(case, window, sinks, D, dt):
    H, KH, most, page, layout, lengths = case
    g = torch.Generator().manual_seed(26)
    rows = [min(L, most - i % 3 if most > 3 else most) for i, L in enumerate(lengths)]
    pools, table, descales = make_cache(g, lengths, KH, D, page, FP8 if dt == "e4m3" else torch.bfloat16, layout)
    cu = torch.tensor([0] + rows).cumsum(0).int()
    q = torch.randn(int(cu[-1]), H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    got = ops().paged_window_attention(
        q.to(DEV), k, v, cu.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), most,
        max(lengths), D ** -0.5, window=window, sinks=sinks, descales=None if descales is None else descales.to(DEV))
    assert error_word() == 0
    want, mag, _ = O.window_attention(q, *cpu_views(pools, D), cu, lengths, table, D ** -0.5, window, sinks, descales)
    close(got, want, mag, "window", dt == "e4m3")


@pytest.mark.parametrize("dt", ["bf16", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (3500, 20)])
def test_decode_joins_many_chunks_at_head_dim_64(dt, window, sinks):
    """Few requests with long contexts: more than 16 chunks to a row."""
    H, KH, D, page, lengths = 12, 1, 64, 16, [5003, 300, 0, 4000]
    g = torch.Generator().manual_seed(27)
    pools, table, descales = make_cache(g, lengths, KH, D, page, FP8 if dt == "e4m3" else torch.bfloat16, "joint")
    q = torch.randn(len(lengths), H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    want, mag, w = O.decode_attention(q, *cpu_views(pools, D), lengths, table, D ** -0.5, window, sinks, descales)
    for gather in (False, True):
        sums = torch.zeros(len(lengths), KH, 5003, device=DEV) if gather else None
        got = ops().paged_decode_attention(
            q.to(DEV), k, v, torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), 5003, D ** -0.5,
            window=window, sinks=sinks, descales=None if descales is None else descales.to(DEV), weight_sums=sums)
        assert error_word() == 0
        close(got, want, mag, "decode", dt == "e4m3")
    for r, L in enumerate(lengths):
        s = sums[r].double().cpu()
        assert ((s[:, :L] - w[r]).abs() <= (2.0 ** -16 + 2.0 ** -22) * w[r]).all() and float(s[:, L:].abs().sum()) == 0.0


@pytest.mark.parametrize("dt", ["bf16", "e4m3"])
def test_window_of_many_row_tiles(dt):
    """More than 512 row tiles and requests, dealt out in shares."""
    H, KH, D, page = 16, 1, 64, 16
    lengths = [(53 * i) % 90 + 1 + (800 if i % 61 == 7 else 0) for i in range(530)]
    rows = [min(L, 1 + (7 * i) % 40) for i, L in enumerate(lengths)]
    g = torch.Generator().manual_seed(28)
    pools, table, descales = make_cache(g, lengths, KH, D, page, FP8 if dt == "e4m3" else torch.bfloat16, "split")
    cu = torch.tensor([0] + rows).cumsum(0).int()
    q = torch.randn(int(cu[-1]), H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    for window, sinks in ((0, 0), (600, 3)):
        got = ops().paged_window_attention(
            q.to(DEV), k, v, cu.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), max(rows),
            max(lengths), D ** -0.5, window=window, sinks=sinks, descales=None if descales is None else descales.to(DEV))
        assert error_word() == 0
        want, mag, _ = O.window_attention(q, *cpu_views(pools, D), cu, lengths, table, D ** -0.5, window, sinks, descales)
        close(got, want, mag, "window", dt == "e4m3")


@pytest.mark.parametrize("rows", [[17, 9], [300, 40]], ids=["verify", "chunk"])
def test_window_in_a_cuda_graph(rows):
    g = torch.Generator().manual_seed(29)
    lengths, KH, H, D = [900, 300], 2, 8, 128
    pools, table, _ = make_cache(g, lengths, KH, D, 16, torch.bfloat16, "joint")
    _, k, v = views(pools, D)
    q = torch.randn(sum(rows), H, D, generator=g).to(torch.bfloat16)
    dq, t = q.to(DEV), table.to(DEV)
    L = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, rows[0], sum(rows)], dtype=torch.int32, device=DEV)

    def call():
        return ops().paged_window_attention(dq, k, v, cu, L, t, max(rows), 900, D ** -0.5, window=500, sinks=4)

    eager = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    out.fill_(math.nan)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    L.copy_(torch.tensor([450, 0], dtype=torch.int32))  # lengths and bounds are read when the graph runs
    cu.copy_(torch.tensor([0, rows[0] - 3, sum(rows)], dtype=torch.int32))
    graph.replay()
    assert error_word() == 0
    want, mag, _ = O.window_attention(q, *cpu_views(pools, D), cu.tolist(), [450, 0], table, D ** -0.5, 500, 4)
    close(out, want, mag, "window")


@pytest.mark.parametrize("case", [(2, [900, 300, 200], True), (50, [900, 300, 200], True), (50, [900, 300, 200], False),
                                  (5, [9000, 300, 200], True)], ids=["few", "many", "copied", "clusters"])
def test_evict_in_a_cuda_graph(case):
    times, some, in_place = case
    lengths, KH, D, page, budget = some * times, 2, 64, 16, 250
    g = torch.Generator().manual_seed(30)
    R, out_cols = len(lengths), -(-budget // page)
    pools, table, _ = make_cache(g, lengths, KH, D, page, torch.bfloat16, "joint", spare=0 if in_place else R * out_cols)
    to = table
    if not in_place:
        free = sorted(set(range(1, pools[0].shape[0])) - set(table.flatten().tolist()))
        to = torch.tensor(free, dtype=torch.int32)[: R * out_cols].view(R, out_cols)
    dev, k, v = views(pools, D)
    first = dev[0].clone()
    L, t, dto = torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), to.to(DEV)
    values = torch.rand(R, KH, max(lengths), generator=g)
    sums = values.to(DEV)

    def call():
        return ops().evict_paged_context(k, v, L, t, sums, budget, sinks=4, recent=30,
                                         out_block_table=None if in_place else dto)

    call()
    dev[0].copy_(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, n, got = call()
    for now in (lengths, [max(0, x - 270) for x in lengths]):  # lengths and sums are read when the graph runs
        dev[0].copy_(first)
        values = torch.rand(R, KH, max(lengths), generator=g)
        sums.copy_(values.to(DEV))
        L.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        assert error_word() == 0
        want = O.evict(values, now, budget, 4, 30)
        assert n.tolist() == [min(x, budget) for x in now]
        assert kept.tolist() == [[w + [-1] * (budget - len(w)) for w in per] for per in want]
        assert torch.equal(dev[0].view(torch.uint8).cpu(), evicted(pools, table, to, want, now, budget, page)[0])


def test_window_and_eviction_of_strided_tensors_on_another_stream():
    g = torch.Generator().manual_seed(31)
    lengths, rows, KH, H, D, page, budget = [130, 50, 300], [20, 50, 7], 2, 4, 128, 16, 40
    pools, table, _ = make_cache(g, lengths, KH, D, page, torch.bfloat16, "joint", spare=12)
    dev, k, v = views(pools, D)
    wide = torch.randn(sum(rows), H, 3, D, generator=g).to(torch.bfloat16)
    q = wide.to(DEV)[:, :, 1]
    tables = torch.full((6, table.shape[1] + 3), 10_000, dtype=torch.int32)  # rows of a wider table, every other one
    tables[::2, : table.shape[1]] = table
    t = tables.to(DEV)[::2, : table.shape[1]]
    free = sorted(set(range(1, pools[0].shape[0])) - set(table.flatten().tolist()))
    to = torch.tensor(free[:9], dtype=torch.int32).view(3, 3)
    wide_to = torch.full((3, 5), 10_000, dtype=torch.int32)
    wide_to[:, :3] = to
    big = torch.rand(3, 3 * KH, 310, generator=g)
    dbig = big.to(DEV)
    L = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0] + rows).cumsum(0).int()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops().paged_window_attention(q, k, v, cu.to(DEV), L, t, 50, 300, D ** -0.5, window=60, sinks=2)
        kept, n, got = ops().evict_paged_context(k, v, L, t, dbig[:, 1:1 + KH, :300], budget, sinks=1, recent=5,
                                                 out_block_table=wide_to.to(DEV)[:, :3])
    side.synchronize()
    assert error_word() == 0
    want, mag, _ = O.window_attention(wide[:, :, 1], *cpu_views(pools, D), cu, lengths, table, D ** -0.5, 60, 2)
    close(out, want, mag, "window")
    rows_kept = O.evict(big[:, 1:1 + KH], lengths, budget, 1, 5)
    assert kept.tolist() == rows_kept and n.tolist() == [40, 40, 40]
    for r in range(3):
        for h in range(KH):
            assert torch.equal(got[r, h].cpu(), big[r, 1 + h, rows_kept[r][h]])
    assert torch.equal(dev[0].view(torch.uint8).cpu(), evicted(pools, table, to, rows_kept, lengths, budget, page)[0])


def test_strides_of_dimensions_of_one():
    g = torch.Generator().manual_seed(32)
    D, page = 128, 48
    pool = torch.randn(page * 2 * D + 16, generator=g).to(torch.bfloat16)
    cache = pool.as_strided((1, 1, page, 2 * D), (5, 3, 2 * D, 1))
    q = torch.randn(4 * D, generator=g).to(torch.bfloat16).as_strided((1, 4, D), (3, D, 1))
    table, L, cu = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([40], dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    dc = pool.to(DEV).as_strided((1, 1, page, 2 * D), (5, 3, 2 * D, 1))
    dq = q.contiguous().to(DEV).as_strided((1, 4, D), (3, D, 1))
    want, mag, _ = O.decode_attention(q, cache[..., :D], cache[..., D:], [40], table, D ** -0.5)
    a = ops().paged_decode_attention(dq, dc[..., :D], dc[..., D:], L.to(DEV), table.to(DEV), 40, D ** -0.5)
    b = ops().paged_window_attention(dq, dc[..., :D], dc[..., D:], cu.to(DEV), L.to(DEV), table.to(DEV), 1, 40, D ** -0.5)
    close(a, want, mag, "decode")
    close(b, want, mag, "window")
    kept, n, _ = ops().evict_paged_context(dc[..., :D], dc[..., D:], L.to(DEV), table.to(DEV),
                                           torch.arange(40.0, device=DEV).view(1, 1, 40), 20)
    assert kept[0, 0].tolist() == list(range(20, 40)) and error_word() == 0


@pytest.mark.parametrize("dt", ["bf16", "e4m3"])
def test_caches_that_hold_nothing(dt):
    """Requests without a position yet: empty tables, sums and pools; their rows see nothing and are zero."""
    KH, H, D, page, R = 2, 4, 64, 16, 3
    L = torch.zeros(R, dtype=torch.int32, device=DEV)
    q = torch.randn(R, H, D, device=DEV).to(torch.bfloat16)
    cu = torch.arange(R + 1, dtype=torch.int32, device=DEV)
    for pages, cols in ((4, 0), (0, 0), (0, 2)):
        cache = torch.zeros(pages, KH, page, 2 * D, dtype=torch.bfloat16, device=DEV)
        cache = cache.to(FP8) if dt == "e4m3" else cache
        k, v = cache[..., :D], cache[..., D:]
        t = torch.zeros(R, cols, dtype=torch.int32, device=DEV)
        for most in (0, 20):
            sums = torch.zeros(R, KH, most, device=DEV)
            for gather in (None, sums, torch.zeros(R, KH, 30, device=DEV)):
                out = ops().paged_decode_attention(q, k, v, L, t, most, 0.1, weight_sums=gather)
                assert out.shape == q.shape and float(out.float().abs().max()) == 0.0
            out = ops().paged_window_attention(q, k, v, cu, L, t, 1, most, 0.1, window=5, sinks=1)
            assert out.shape == q.shape and float(out.float().abs().max()) == 0.0
            kept, n, got = ops().evict_paged_context(k, v, L, t, sums, 8, sinks=1)
            assert int((kept != -1).sum()) == 0 and n.tolist() == [0] * R and float(got.abs().sum()) == 0.0
    assert error_word() == 0


def attention_calls(KH=2, H=8, D=128, page=16, lengths=(90, 33)):
    """(query, one call of each attention on it) over one small cache."""
    g = torch.Generator().manual_seed(33)
    pools, table, _ = make_cache(g, list(lengths), KH, D, page, torch.bfloat16, "joint")
    _, k, v = views(pools, D)
    L, t = torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV)
    cu = torch.arange(len(lengths) + 1, dtype=torch.int32, device=DEV)
    q = torch.randn(len(lengths), H, D, generator=g).to(torch.bfloat16).to(DEV)

    def decode(q, sums=None, k=k):
        return ops().paged_decode_attention(q, k, v, L, t, max(lengths), D ** -0.5, weight_sums=sums)

    def chunk(q, sums=None, k=k):
        return ops().paged_window_attention(q, k, v, cu, L, t, 1, max(lengths), D ** -0.5, window=50, sinks=2)

    return q, k, (decode, chunk)


def test_no_gradient_is_an_error_and_not_a_constant():
    q, k, calls = attention_calls()
    for call in calls:
        plain = call(q)
        assert not plain.requires_grad
        for kw in (dict(q=q.clone().requires_grad_()), dict(q=q, k=k.detach().clone().requires_grad_())):
            out = call(**kw)
            assert torch.equal(out, plain) and out.requires_grad
            with pytest.raises(RuntimeError):
                out.float().sum().backward()
            with torch.no_grad():
                assert not call(**kw).requires_grad
    a, b = torch.zeros(2, 2, 90, device=DEV), torch.zeros(2, 2, 90, device=DEV)
    assert torch.equal(calls[0](q, a), calls[0](q.clone().requires_grad_(), b)) and torch.equal(a, b)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_attentions_stay_whole_in_a_compiled_graph(backend):
    q, _, calls = attention_calls()
    for call in calls:
        def layer(q, sums):
            return call(q * 2, sums) + 1

        compiled = torch.compile(layer, backend=backend, fullgraph=True)
        for scale in (1.0, 0.5):
            a, b = torch.zeros(2, 2, 90, device=DEV), torch.zeros(2, 2, 90, device=DEV)
            with torch.no_grad():
                assert torch.equal(compiled(q * scale, a), layer(q * scale, b))
            assert torch.equal(a, b)
    assert error_word() == 0


@pytest.mark.parametrize("dt", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows_most", [8, 40])
def test_window_of_many_row_tiles_in_shares(dt, rows_most):
    """More than 512 row tiles, some of them long enough that all are dealt out in shares."""
    H, KH, D, page = 16, 1, 64, 16
    lengths = [(53 * i) % 90 + 1 + (1900 if i % 61 == 7 else 0) for i in range(530)]
    rows = [min(L, 1 + (7 * i) % rows_most) for i, L in enumerate(lengths)]
    g = torch.Generator().manual_seed(34)
    pools, table, descales = make_cache(g, lengths, KH, D, page, FP8 if dt == "e4m3" else torch.bfloat16, "joint")
    cu = torch.tensor([0] + rows).cumsum(0).int()
    q = torch.randn(int(cu[-1]), H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    for window, sinks in ((0, 0), (1700, 3)):
        got = ops().paged_window_attention(
            q.to(DEV), k, v, cu.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), max(rows),
            max(lengths), D ** -0.5, window=window, sinks=sinks, descales=None if descales is None else descales.to(DEV))
        assert error_word() == 0
        want, mag, _ = O.window_attention(q, *cpu_views(pools, D), cu, lengths, table, D ** -0.5, window, sinks, descales)
        close(got, want, mag, "window", dt == "e4m3")


@pytest.mark.parametrize("dt", ["bf16", "e4m3"])
def test_window_of_many_requests(dt):
    """So many requests that their short items are dealt out in shares; some have no rows, some no positions."""
    H, KH, D, page = 4, 2, 64, 16
    lengths = [(53 * i) % 90 + (400 if i % 61 == 7 else 0) for i in range(1100)]
    rows = [min(L + i % 2, (7 * i) % 6) for i, L in enumerate(lengths)]
    g = torch.Generator().manual_seed(35)
    pools, table, descales = make_cache(g, lengths, KH, D, page, FP8 if dt == "e4m3" else torch.bfloat16, "joint")
    cu = torch.tensor([0] + rows).cumsum(0).int()
    q = torch.randn(int(cu[-1]), H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    got = ops().paged_window_attention(
        q.to(DEV), k, v, cu.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), table.to(DEV), max(rows),
        max(lengths), D ** -0.5, descales=None if descales is None else descales.to(DEV))
    assert error_word() == 0
    want, mag, _ = O.window_attention(q, *cpu_views(pools, D), cu, lengths, table, D ** -0.5, descales=descales)
    close(got, want, mag, "window", dt == "e4m3")


def test_recorded_errors_are_raised_once():
    from flashmap_b200._lib import FlashMapError
    _, k, (decode, _) = attention_calls()
    c = ops()
    q = torch.zeros(2, 8, 128, dtype=torch.bfloat16, device=DEV)
    c.check_device_errors()
    decode(q)
    c.check_device_errors()
    bad = torch.full((1, 1), 10_000, dtype=torch.int32, device=DEV)
    c.paged_decode_attention(q[:1], k, k, torch.tensor([5], dtype=torch.int32, device=DEV), bad, 5, 1.0)
    with pytest.raises(FlashMapError, match="device error 4"):
        c.check_device_errors(torch.device("cuda", torch.cuda.current_device()))
    c.check_device_errors()


@pytest.mark.parametrize("dt", ["bf16", "e4m3"])
@pytest.mark.parametrize("H,KH", [(300, 1), (514, 2)])
def test_head_groups_wider_than_a_row_tile(H, KH, dt):
    D, page, lengths, rows = 64, 16, [150, 1, 0, 700], [5, 1, 2, 3]
    g = torch.Generator().manual_seed(36)
    pools, table, descales = make_cache(g, lengths, KH, D, page, FP8 if dt == "e4m3" else torch.bfloat16, "joint")
    cu = torch.tensor([0] + rows).cumsum(0).int()
    q = torch.randn(int(cu[-1]), H, D, generator=g).to(torch.bfloat16)
    _, k, v = views(pools, D)
    L, dd = torch.tensor(lengths, dtype=torch.int32, device=DEV), None if descales is None else descales.to(DEV)
    got = ops().paged_window_attention(q.to(DEV), k, v, cu.to(DEV), L, table.to(DEV), max(rows), max(lengths), D ** -0.5,
                                       window=200, sinks=3, descales=dd)
    want, mag, _ = O.window_attention(q, *cpu_views(pools, D), cu, lengths, table, D ** -0.5, 200, 3, descales)
    close(got, want, mag, "window", dt == "e4m3")
    sums = torch.zeros(4, KH, 700, device=DEV)
    got = ops().paged_decode_attention(q[:4].to(DEV), k, v, L, table.to(DEV), max(lengths), D ** -0.5, descales=dd,
                                       weight_sums=sums)
    want, mag, w = O.decode_attention(q[:4], *cpu_views(pools, D), lengths, table, D ** -0.5, descales=descales)
    close(got, want, mag, "decode", dt == "e4m3")
    for r, n in enumerate(lengths):
        assert ((sums[r, :, :n].double().cpu() - w[r]).abs() <= (2.0 ** -16 + 2.0 ** -20) * w[r]).all()
    assert error_word() == 0


@pytest.mark.parametrize("rows", [1, 40])  # chunks of one row tile, of two
@pytest.mark.parametrize("heavy", [0, 700])
def test_window_many_keys_far_below_one_e4m3(rows, heavy):
    """One key takes nearly all of the weight and has a value of 0, 1599 others 2^-22 to 2^-26 of it each: what they add
    is the output.  As many requests (the same context) as leave the items whole.

    Numerators are f16 with the row's largest at 2^11 or more: one of 2^-26 is 2^-15, whose steps are 2^-24: off by 2^-25
    at most, 2^-36 of the largest.  n keys: n 2^-36 max |v| beside the rest."""
    g = torch.Generator().manual_seed(71)
    L, D, R, H = 1600, 64, 160, 4
    pools, table, _ = make_cache(g, [L], 1, D, 16, FP8, "split")
    j = torch.arange(L)
    page = table[0, j // 16].long()
    K, V = torch.zeros(L, D), torch.randn(L, D, generator=g).abs()
    K[heavy], V[heavy] = 6.0, 0.0
    for pool, x in zip(pools, (K, V)):
        pool.view(torch.uint8)[page, 0, j % 16] = x.to(FP8).view(torch.uint8)
    _, k, v = views(pools, D)
    vmax = float(V.max())
    lengths = torch.full((R,), L, dtype=torch.int32, device=DEV)
    many = table.to(DEV).expand(R, -1)
    for size in (0.3125, 0.328125, 0.375):  # e^-15, e^-15.75, e^-18
        q = torch.full((rows, H, D), size).to(torch.bfloat16)
        want, mag, _ = O.window_attention(q, *cpu_views(pools, D), torch.tensor([0, rows]), [L], table, D ** -0.5)
        cu = rows * torch.arange(R + 1, dtype=torch.int32, device=DEV)
        got = ops().paged_window_attention(q.to(DEV).repeat(R, 1, 1), k, v, cu, lengths, many, rows, L, D ** -0.5)
        for r in (0, 77, 159):
            err = (got[r * rows: (r + 1) * rows].double().cpu() - want).abs()
            tol = (2.0 ** -11 + 2.0 ** -14) * mag + (2.0 ** -8 + 2.0 ** -14) * want.abs() + L * 2.0 ** -36 * vmax
            assert (err <= tol).all(), (size, (err / tol).max().item())
    assert error_word() == 0


@pytest.mark.parametrize("heavy", [0, 700, 1599])
@pytest.mark.parametrize("R", [1, 160])  # cut into chunks and joined, whole
def test_decode_many_keys_far_below_one_e4m3(heavy, R):
    """As above for one new token, with its gathered weights; numerators are f16 with a warp's largest at 2^15, so one of
    2^-26 is 2^-11, within f16's ordinary steps."""
    g = torch.Generator().manual_seed(72)
    L, D, H = 1600, 64, 4
    pools, table, _ = make_cache(g, [L], 1, D, 16, FP8, "split")
    j = torch.arange(L)
    page = table[0, j // 16].long()
    K, V = torch.zeros(L, D), torch.randn(L, D, generator=g).abs()
    K[heavy], V[heavy] = 6.0, 0.0
    for pool, x in zip(pools, (K, V)):
        pool.view(torch.uint8)[page, 0, j % 16] = x.to(FP8).view(torch.uint8)
    _, k, v = views(pools, D)
    lengths = torch.full((R,), L, dtype=torch.int32, device=DEV)
    for size in (0.3125, 0.328125, 0.375):  # e^-15, e^-15.75, e^-18
        q = torch.full((1, H, D), size).to(torch.bfloat16)
        want, mag, w = O.decode_attention(q, *cpu_views(pools, D), [L], table, D ** -0.5)
        sums = torch.zeros(R, 1, L, device=DEV)
        args = (q.to(DEV).expand(R, -1, -1), k, v, lengths, table.to(DEV).expand(R, -1), L, D ** -0.5)
        for kw in ({}, dict(weight_sums=sums)):
            close(ops().paged_decode_attention(*args, **kw)[R - 1:], want, mag, "decode", True)
        assert ((sums[R - 1].double().cpu() - w[0]).abs() <= 2.0 ** -16 * w[0] + 2.0 ** -22 * w[0]).all()
    assert error_word() == 0
