"""Attention over a 4-bit cache against the 64-bit oracle.

Tolerances.  A cache value is exact in f16, a query row too (times a power of
two; values under 2^-24 of its largest come within 2^-38 of it).  The softmax
numerators are rounded once to f16: 11 bits, 2^-11 of each, as long as they are
not under 2^-14 of the type's unit; for the decoding kernel that is 2^-25 of the
largest, for chunks 2^-14 of it, where steps of 2^-24 are off by 2^-25 of the
largest numerator a key at most.  The output is rounded once to bf16 (2^-8),
and scores and sums are fp32 (under 2^-14 of both, as for the wider caches).
So outputs are held to (2^-11 + 2^-14) sum w |v| + (2^-8 + 2^-14) |out|, and
where a row sees n keys of which one outweighs the rest, to n 2^-25 max |v| more.
"""

import math

import pytest
import torch

from oracle import cache_ops as C
from oracle import serving_step as O

pytestmark = pytest.mark.gpu

DEV = "cuda"
FP8 = torch.float8_e4m3fn


def ops():
    from flashmap_b200 import cache_ops
    return cache_ops


def error_word():
    from flashmap_b200.ops import error_word as word
    torch.cuda.synchronize()
    w = word(torch.device("cuda", torch.cuda.current_device()))
    code = int(w)
    w.zero_()
    return code


def close(got, want, mag, what, more=0.0):
    assert torch.isfinite(got.float()).all(), f"{what}: not finite"
    err = (got.double().cpu() - want).abs()
    tol = (2.0 ** -11 + 2.0 ** -14) * mag + (2.0 ** -8 + 2.0 ** -14) * want.abs() + more + 1e-30
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the tolerance"


class Cache:
    """A 4-bit cache; unused table entries name page 0, and slots past a length hold factors that are no number."""

    def __init__(self, g, lengths, KH, D, page, layout, scaled=False, spread=1.0):
        used = [-(-L // page) for L in lengths]
        cols, total = max(1, max(used, default=1)), sum(used) + 4
        ids = torch.randperm(total - 1, generator=g) + 1
        self.table = torch.zeros(len(lengths), cols, dtype=torch.int32)
        at = 0
        for r, n in enumerate(used):
            self.table[r, :n] = ids[at: at + n].int()
            at += n
        n = 2 if layout == "joint" else 1
        pools = [O.quantise4(spread * torch.randn(total, KH, page, n * D, generator=g)) for _ in range(3 - n)]
        for _, f in pools:
            f[0] = math.nan
            for r, L in enumerate(lengths):
                if L % page:
                    f[self.table[r, used[r] - 1].item(), :, L % page:] = math.nan
        self.lengths, self.D = lengths, D
        self.descales = 0.5 + torch.rand(2, len(lengths), KH, generator=g) if scaled else None
        self.values = [O.values4(*p) for p in pools]
        self.dev = [(c.to(DEV), f.to(DEV)) for c, f in pools]

    def host(self):
        return self.values[0][..., : self.D], self.values[-1][..., -self.D:]

    def tensors(self):
        D = self.D
        (kc, kf), (vc, vf) = self.dev[0], self.dev[-1]
        return kc[..., : D // 2], vc[..., -(D // 2):], kf[..., : D // 16], vf[..., -(D // 16):]

    def rest(self):
        return torch.tensor(self.lengths, dtype=torch.int32, device=DEV), self.table.to(DEV)

    def kw(self, **kw):
        return dict(kw, descales=None if self.descales is None else self.descales.to(DEV))

    def decode(self, q, top=None, **kw):
        L, table = self.rest()
        return ops().paged_decode_attention_fp4(q.to(DEV), *self.tensors(), L, table, top or max(self.lengths), self.D ** -0.5, **self.kw(**kw))

    def window(self, q, rows, **kw):
        L, table = self.rest()
        cu = torch.tensor([0] + rows).cumsum(0).int()
        got = ops().paged_window_attention_fp4(q.to(DEV), *self.tensors(), cu.to(DEV), L, table, max(rows), max(self.lengths),
                                               self.D ** -0.5, **self.kw(**kw))
        want, mag, _ = C.window_attention(q, *self.host(), cu, self.lengths, self.table, self.D ** -0.5, kw.get("window", 0),
                                          kw.get("sinks", 0), self.descales)
        return got, want, mag

    def want(self, q, window=0, sinks=0):
        want, mag, _ = C.decode_attention(q, *self.host(), self.lengths, self.table, self.D ** -0.5, window, sinks, self.descales)
        return want, mag


DECODE = [
    # heads, kv_heads, head_dim, page, layout, scaled, window, sinks, lengths
    (8, 2, 128, 16, "joint", False, 0, 0, [1, 0, 17, 700, 64, 65, 3]),
    (8, 8, 128, 16, "split", True, 0, 0, [33, 129, 2]),
    (10, 2, 64, 24, "joint", True, 0, 0, [257, 1, 600]),
    (16, 1, 128, 1, "split", False, 0, 0, [300, 77]),
    (40, 2, 64, 32, "joint", False, 100, 4, [1000, 99, 100, 101, 104, 105, 0]),
    (20, 1, 128, 16, "joint", True, 1, 0, [1, 2, 500]),
    (8, 2, 128, 128, "joint", False, 130, 200, [5, 150, 331, 900]),
    (12, 1, 128, 1, "split", True, 64, 3, [400, 66, 67, 68]),
    (5, 1, 64, 24, "joint", False, 0, 0, [333, 16, 15]),
    (32, 2, 64, 16, "split", False, 70, 16, [512, 5]),
    (4, 1, 128, 64, "split", False, 0, 0, [9001, 40, 5000]),
    (3, 1, 64, 16, "joint", True, 3000, 40, [7000, 3041, 2999]),
]


@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(map(str, c[:8])))
def test_decode(case):
    H, KH, D, page, layout, scaled, window, sinks, lengths = case
    g = torch.Generator().manual_seed(51)
    cache = Cache(g, lengths, KH, D, page, layout, scaled)
    q = torch.randn(len(lengths), H, D, generator=g).to(torch.bfloat16)
    got = cache.decode(q, window=window, sinks=sinks)
    close(got, *cache.want(q, window, sinks), "decode")
    assert torch.equal(got, cache.decode(q, window=window, sinks=sinks))
    # sized for far longer contexts than there are (the table cuts it)
    close(cache.decode(q, top=1 << 20, window=window, sinks=sinks), *cache.want(q, window, sinks), "decode")
    assert error_word() == 0


def test_decode_extreme_scores():
    """Scores of thousands, queries of zero, tiny and huge ones, factors at both ends, infinite queries."""
    g = torch.Generator().manual_seed(52)
    D = 128
    for spread in (1.0, 1e-3, 400.0):
        cache = Cache(g, [80] * 4, 1, D, 16, "split", True, spread)
        q = torch.randn(4, 2, D, generator=g)
        q[0] *= 1e3 / spread
        q[1] = 0.0
        q[2] *= 1e-30
        q = q.to(torch.bfloat16)
        got, (want, mag) = cache.decode(q), cache.want(q)
        # A score of s is off by s 2^-20, which moves weights by that share.  Where the key that outweighs the rest
        # holds an exact 0, what is left has weights under 2^-126 of it, which fp32 has not: 80 of them times values
        # of 2688 * 1.5 at most are under 80 * 2^-126 * 4032 = 3.8e-33.
        err = (got[0].double().cpu() - want[0]).abs()
        assert (err <= 0.01 * mag[0] + 2.0 ** -8 * want[0].abs() + 80 * 2.0 ** -126 * 4032).all()
        close(got[1:3], want[1:3], mag[1:3], "decode")
    q[3, :, 5] = math.inf
    assert torch.isfinite(cache.decode(q)[:3].float()).all()


def test_one_key_outweighs_many():
    """A long context of equal scores far below one: numerators where f16 has its coarsest steps."""
    g = torch.Generator().manual_seed(53)
    L, D = 6000, 64
    cache = Cache(g, [L], 1, D, 16, "split")
    K = torch.zeros(L, D)
    K[3000] = 6.0
    codes, factors = O.quantise4(K)
    kc, kf = cache.dev[0]
    j = torch.arange(L)
    page = cache.table[0, j // 16].long()
    kc[page.to(DEV), 0, (j % 16).to(DEV)] = codes.to(DEV)
    kf.view(torch.uint8)[page.to(DEV), 0, (j % 16).to(DEV)] = factors.view(torch.uint8).to(DEV)
    cache.values[0][page, 0, j % 16] = O.values4(codes, factors)
    for size in (0.2, 0.25, 0.3):  # e^-9.6 to e^-14.4 of the one
        q = torch.full((1, 4, D), size).to(torch.bfloat16)
        want, mag = cache.want(q)
        close(cache.decode(q), want, mag, "decode")
        vmax = float(cache.host()[1][page, 0, j % 16].abs().max())
        close(cache.window(q, [1])[0], want, mag, "window", more=L * 2.0 ** -25 * vmax)


WINDOW = [
    # heads, kv_heads, head_dim, page, layout, scaled, window, sinks, lengths, query rows
    (8, 2, 128, 16, "joint", False, 0, 0, [1, 0, 17, 200, 64, 65, 300], [1, 0, 17, 5, 64, 3, 150]),
    (4, 4, 128, 16, "split", True, 0, 0, [70, 129], [70, 129]),
    (10, 2, 64, 24, "joint", False, 0, 0, [257, 1, 300], [33, 1, 299]),
    (16, 1, 128, 1, "split", False, 0, 0, [300, 77], [17, 17]),
    (20, 1, 64, 32, "joint", True, 100, 4, [500, 99, 100, 101, 104, 0], [200, 99, 100, 17, 1, 0]),
    (8, 2, 128, 16, "joint", False, 1, 1, [300], [280]),
    (8, 2, 128, 128, "split", False, 130, 200, [5, 150, 331, 700], [5, 20, 331, 17]),
    (2, 1, 128, 16, "joint", False, 37, 70, [900], [500]),
    (8, 2, 128, 16, "joint", False, 0, 0, [20, 100], [30, 101]),  # more rows than positions: the first see nothing
    (5, 1, 64, 24, "joint", False, 0, 0, [333, 16, 15], [300, 16, 2]),
    (3, 3, 64, 1, "split", True, 70, 16, [512, 5], [200, 5]),
    (4, 1, 128, 16, "joint", True, 0, 0, [5003, 3100], [17, 600]),
    (4, 1, 128, 16, "joint", False, 700, 5, [5003, 3100], [17, 600]),
    (300, 1, 64, 16, "split", False, 0, 0, [200], [3]),
]


@pytest.mark.parametrize("case", WINDOW, ids=lambda c: "-".join(map(str, c[:8])))
def test_window(case):
    H, KH, D, page, layout, scaled, window, sinks, lengths, rows = case
    g = torch.Generator().manual_seed(54)
    cache = Cache(g, lengths, KH, D, page, layout, scaled)
    q = torch.randn(sum(rows), H, D, generator=g).to(torch.bfloat16)
    got, want, mag = cache.window(q, rows, window=window, sinks=sinks)
    close(got, want, mag, "window")
    assert torch.equal(got, cache.window(q, rows, window=window, sinks=sinks)[0])
    assert error_word() == 0


def test_window_many_short_items():
    H, KH, D, page = 16, 8, 64, 16
    lengths = [37 * (i % 13) + (i % 3) for i in range(40)]
    rows = [min(L, 5 * i % 211) for i, L in enumerate(lengths)]
    g = torch.Generator().manual_seed(55)
    cache = Cache(g, lengths, KH, D, page, "joint")
    q = torch.randn(sum(rows), H, D, generator=g).to(torch.bfloat16)
    for window, sinks in ((0, 0), (100, 3)):
        close(*cache.window(q, rows, window=window, sinks=sinks), "window")
    assert error_word() == 0


def test_bad_indices_are_reported_and_not_seen():
    g = torch.Generator().manual_seed(56)
    cache = Cache(g, [64], 2, 128, 16, "joint")
    q = torch.randn(1, 4, 128, generator=g).to(torch.bfloat16)
    good = cache.table.clone()
    cache.table, cache.lengths = good[:, [0, 2, 3]], [48]
    want, mag = cache.want(q)
    cache.table, cache.lengths = good.clone(), [64]
    cache.table[0, 1] = 10_000
    for got in (cache.decode(q), None):
        if got is None:
            L, table = cache.rest()
            got = ops().paged_window_attention_fp4(q.to(DEV), *cache.tensors(), torch.tensor([0, 1], dtype=torch.int32, device=DEV), L,
                                                   table, 1, 64, 128 ** -0.5)
        close(got, want, mag, "attention")
        assert error_word() == 4
    cache.table, cache.lengths = good, [60]
    want, mag = cache.want(q)
    cache.lengths = [100]  # past the call's size: cut
    close(cache.decode(q, top=60), want, mag, "decode")
    assert error_word() == 4
    cache.lengths = [-3]
    assert float(cache.decode(q, top=60).abs().max()) == 0.0 and error_word() == 4


def test_more_rows_than_the_call_is_sized_for():
    """max_seqlen_q says 10 rows of 4 heads (one row tile), a request has 50: recorded; the other request is as it should be."""
    g = torch.Generator().manual_seed(60)
    cache = Cache(g, [300, 200], 1, 128, 16, "joint")
    q = torch.randn(60, 4, 128, generator=g).to(torch.bfloat16)
    L, table = cache.rest()
    cu = torch.tensor([0, 50, 60], dtype=torch.int32)
    got = ops().paged_window_attention_fp4(q.to(DEV), *cache.tensors(), cu.to(DEV), L, table, 10, 300, 128 ** -0.5)
    want, mag, _ = C.window_attention(q, *cache.host(), cu, cache.lengths, cache.table, 128 ** -0.5)
    assert error_word() == 4
    close(got[50:], want[50:], mag[50:], "window")


def test_strides_streams_graphs_and_far_pages():
    g = torch.Generator().manual_seed(57)
    D, KH, page = 64, 2, 16
    cache = Cache(g, [130, 50], KH, D, page, "joint")
    wide = torch.randn(2, 4, 3, D, generator=g).to(torch.bfloat16)
    want, mag = cache.want(wide[:, :, 1])
    L, table = cache.rest()
    t = cache.tensors()
    q = wide.to(DEV)[:, :, 1]
    cu = torch.arange(3, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = ops().paged_decode_attention_fp4(q, *t, L, table, 130, D ** -0.5)
        b = ops().paged_window_attention_fp4(q, *t, cu, L, table, 1, 130, D ** -0.5)
    side.synchronize()
    close(a, want, mag, "decode")
    close(b, want, mag, "window")
    static = torch.zeros(2, 4, D, dtype=torch.bfloat16, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = ops().paged_decode_attention_fp4(static, *t, L, table, 4000, D ** -0.5)
        b = ops().paged_window_attention_fp4(static, *t, cu, L, table, 1, 4000, D ** -0.5)
    static.copy_(q)
    for lengths in ([100, 50], [1, 0]):
        L.copy_(torch.tensor(lengths, dtype=torch.int32))
        cache.lengths = lengths
        want, mag = cache.want(wide[:, :, 1])
        graph.replay()
        torch.cuda.synchronize()
        close(a, want, mag, "decode")
        if min(lengths):
            close(b, want, mag, "window")
    assert error_word() == 0


@pytest.mark.parametrize("reach", [2_200_000_000, 8_600_000_000])  # offsets past 32 bits in bytes, and in rows of factors
def test_far_pages(reach):
    g = torch.Generator().manual_seed(57)
    D, KH, page = 64, 2, 16
    cache = Cache(g, [130, 50], KH, D, page, "joint")
    wide = torch.randn(2, 4, 3, D, generator=g).to(torch.bfloat16)
    q = wide.to(DEV)[:, :, 1]
    cu = torch.arange(3, dtype=torch.int32, device=DEV)
    stride = 2_200_000_000
    pool = torch.empty(2 * stride + KH * page * D, dtype=torch.uint8, device=DEV)
    far = pool.as_strided((3, KH, page, D), (stride, page * D, D, 1))
    factors = torch.empty(2 * reach + KH * page * D // 8, dtype=torch.uint8, device=DEV)
    far_f = factors.as_strided((3, KH, page, D // 8), (reach, page * D // 8, D // 8, 1))
    used = cache.table[1, :3].long().to(DEV)
    far.copy_(cache.dev[0][0][used])
    far_f.copy_(cache.dev[0][1].view(torch.uint8)[used])
    far_f = far_f.view(FP8)
    views = (far[..., : D // 2], far[..., D // 2:], far_f[..., : D // 16], far_f[..., D // 16:])
    order = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV)
    one = torch.tensor([40], dtype=torch.int32, device=DEV)
    cache.lengths = [1, 40]
    want, mag = (x[1:] for x in cache.want(wide[:, :, 1]))
    close(ops().paged_decode_attention_fp4(q[1:], *views, one, order, 40, D ** -0.5), want, mag, "decode")
    close(ops().paged_window_attention_fp4(q[1:], *views, cu[:2], one, order, 1, 40, D ** -0.5), want, mag, "window")
    assert error_word() == 0


def test_empty_and_traced_calls():
    g = torch.Generator().manual_seed(58)
    cache = Cache(g, [5, 0], 1, 64, 16, "split")
    q = torch.randn(2, 2, 64, generator=g).to(torch.bfloat16).to(DEV)
    L, table = cache.rest()
    t = cache.tensors()
    cu = torch.arange(3, dtype=torch.int32, device=DEV)
    assert ops().paged_decode_attention_fp4(q[:0], *t, L[:0], table[:0], 5, 0.1).shape == (0, 2, 64)
    assert ops().paged_window_attention_fp4(q[:0], *t, cu * 0, L, table, 0, 5, 0.1).shape == (0, 2, 64)
    assert float(ops().paged_decode_attention_fp4(q, *t, L * 0, table, 0, 0.1).abs().max()) == 0.0
    assert float(ops().paged_decode_attention_fp4(q, *t, L * 0, table[:, :0], 5, 0.1).abs().max()) == 0.0

    def f(q):
        a = ops().paged_decode_attention_fp4(q, *t, L, table, 5, 0.1, window=3, sinks=1)
        return a + ops().paged_window_attention_fp4(q, *t, cu, L, table, 1, 5, 0.1)

    assert torch.equal(torch.compile(f, backend="aot_eager")(q), f(q))
    out = ops().paged_decode_attention_fp4(q.clone().requires_grad_(), *t, L, table, 5, 0.1)
    with pytest.raises(RuntimeError):
        out.float().sum().backward()
    assert error_word() == 0


def test_refusals():
    from flashmap_b200 import _lib
    from flashmap_b200.cache_ops import OpArgumentError
    g = torch.Generator().manual_seed(59)
    cache = Cache(g, [5, 3], 2, 64, 16, "split")
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    L, table = cache.rest()
    kc, vc, kf, vf = cache.tensors()
    f = ops().paged_decode_attention_fp4
    cu = torch.arange(3, dtype=torch.int32, device=DEV)
    for args in ((q.float(), kc, vc, kf, vf, L, table, 5, 0.1), (q[:, :3], kc, vc, kf, vf, L, table, 5, 0.1),
                 (q[:1], kc, vc, kf, vf, L, table, 5, 0.1), (q, kc, vc, kf, None, L, table, 5, 0.1),
                 (q, kc, vc, kf, vf.float(), L, table, 5, 0.1), (q, kc, vc, kf[:, :, :8], vf, L, table, 5, 0.1),
                 (q, kc.view(torch.int8), vc, kf, vf, L, table, 5, 0.1), (q, kc, vc[:1], kf, vf, L, table, 5, 0.1),
                 (q, kc[..., :16], vc[..., :16], kf, vf, L, table, 5, 0.1), (q, kc, vc, kf, vf, L.long(), table, 5, 0.1),
                 (q, kc, vc, kf, vf, L, table.long(), 5, 0.1), (q, kc, vc, kf, vf, L, table, -1, 0.1),
                 (q.cpu(), kc, vc, kf, vf, L, table, 5, 0.1), (q, kc, vc, kf.cpu(), vf, L, table, 5, 0.1)):
        with pytest.raises(OpArgumentError):
            f(*args)
    with pytest.raises(OpArgumentError):
        f(q, kc, vc, kf, vf, L, table, 5, 0.1, window=-1)
    with pytest.raises(OpArgumentError):
        f(q, kc, vc, kf, vf, L, table, 5, 0.1, descales=torch.ones(2, 1, 2, device=DEV))
    with pytest.raises(OpArgumentError):
        ops().paged_window_attention_fp4(q, kc, vc, kf, vf, cu[:2], L, table, 1, 5, 0.1)
    odd = torch.zeros(kc.numel() + 8, dtype=torch.uint8, device=DEV)[8:].view(kc.shape)
    with pytest.raises(_lib.FlashMapError):
        f(q, odd, vc, kf, vf, L, table, 5, 0.1)


@pytest.mark.parametrize("rows", [1, 40])  # one row tile with both softmax warpgroups, two row tiles
@pytest.mark.parametrize("heavy", [0, 700, 1599])
def test_many_keys_far_below_one(rows, heavy):
    """One key takes nearly all of the weight and has a value of 0, 1599 others 2^-22 to 2^-26 of it each: what they add
    is the output.  As many requests (the same context) as leave the items whole.

    A numerator of a row is at least 2^11 times its share of the row's largest, so one of 2^-26 is 2^-15 in f16, whose
    steps there are 2^-24: off by 2^-25 at most, 2^-36 of the largest.  n keys: n 2^-36 max |v| beside the rest."""
    g = torch.Generator().manual_seed(61)
    L, D, R, H = 1600, 64, 160, 4
    cache = Cache(g, [L], 1, D, 16, "split")
    j = torch.arange(L)
    page = cache.table[0, j // 16].long()
    K, V = torch.zeros(L, D), torch.randn(L, D, generator=g).abs()
    K[heavy], V[heavy] = 6.0, 0.0
    for which, x in ((0, K), (1, V)):
        codes, factors = O.quantise4(x)
        kc, kf = cache.dev[which]
        kc[page.to(DEV), 0, (j % 16).to(DEV)] = codes.to(DEV)
        kf.view(torch.uint8)[page.to(DEV), 0, (j % 16).to(DEV)] = factors.view(torch.uint8).to(DEV)
        cache.values[which][page, 0, j % 16] = O.values4(codes, factors)
    vmax = float(cache.host()[1][page, 0, j % 16].abs().max())
    table = cache.table.to(DEV).expand(R, -1)
    lengths = torch.full((R,), L, dtype=torch.int32, device=DEV)
    cu = rows * torch.arange(R + 1, dtype=torch.int32, device=DEV)
    for size in (0.3125, 0.328125, 0.375):  # e^-15, e^-15.75, e^-18
        q = torch.full((rows, H, D), size).to(torch.bfloat16)
        want, mag, _ = C.window_attention(q, *cache.host(), torch.tensor([0, rows]), [L], cache.table, D ** -0.5)
        got = ops().paged_window_attention_fp4(q.to(DEV).repeat(R, 1, 1), *cache.tensors(), cu, lengths, table, rows, L, D ** -0.5)
        more = L * 2.0 ** -36 * vmax
        for r in (0, 77, 159):
            close(got[r * rows: (r + 1) * rows], want, mag, f"window, request {r}", more=more)
        if rows == 1:
            one = ops().paged_decode_attention_fp4(q.to(DEV).expand(R, -1, -1), *cache.tensors(), lengths, table, L, D ** -0.5)
            close(one[159:], want, mag, "decode", more=more)
    assert error_word() == 0


def test_short_and_long_contexts_in_a_call_sized_for_more():
    """Requests of one chunk, of a few and of many beside one another, where rows are joined by a block each."""
    g = torch.Generator().manual_seed(62)
    lengths = [5, 300, 20003, 0, 200]
    cache = Cache(g, lengths, 2, 64, 16, "joint")
    q = torch.randn(5, 8, 64, generator=g).to(torch.bfloat16)
    want, mag = cache.want(q)
    L = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    table = torch.zeros(5, 8192, dtype=torch.int32)
    table[:, : cache.table.shape[1]] = cache.table
    got = [ops().paged_decode_attention_fp4(q.to(DEV), *cache.tensors(), L, table.to(DEV), 131072, 64 ** -0.5) for _ in range(3)]
    close(got[0], want, mag, "decode")
    assert all(torch.equal(got[0], x) for x in got[1:]) and error_word() == 0
