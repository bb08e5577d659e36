"""``append_paged_context`` against the oracle.

Rotation is fp32 with every product and sum rounded, which the CPU repeats bit
for bit; so do the divisions and roundings behind it.  The cache is therefore
held to equal bytes, slots that nothing was written to included, and queries to
equal bits.  Apart from that the values are held to the formula in 64 bits: a
rotated value has three roundings of 2^-24 of |a c| + |b s|, the cache's type
adds half a step of its own (bf16 2^-8, e4m3 2^-4 or 2^-10 where steps are
absolute; a 4-bit value half the distance of its codes, at most one factor).
"""

import math

import pytest
import torch

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


def table_of(n, D, theta=1e4):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    return torch.stack([angle.cos(), angle.sin()], -1).float()


class Cache:
    """A cache of random bytes on the CPU; ``gpu`` its tensors on the GPU."""

    def __init__(self, g, lengths, KH, D, page, kind, layout, spare=2):
        used = [max(1, -(-L // page)) for L in lengths]
        self.cols = max(used)
        total = sum(used) + spare
        ids = torch.randperm(total, generator=g).int()
        self.table = torch.full((len(lengths), self.cols), 1 << 30, dtype=torch.int32)  # unused entries name no page
        at = 0
        for r, n in enumerate(used):
            self.table[r, :n] = ids[at: at + n]
            at += n
        self.lengths = torch.tensor(lengths, dtype=torch.int32)
        self.kind, self.page, self.D = kind, page, D
        n = 1 if layout == "joint" else 2

        def pool(width):
            w = n == 1 and 2 * width or width
            return [torch.randint(0, 256, (total, KH, page, w), generator=g, dtype=torch.uint8) for _ in range(n)]

        self.row = {"bf16": 2 * D, "e4m3": D, "fp4": D // 2}[kind]
        self.pools = pool(self.row)
        self.factors = pool(D // 16) if kind == "fp4" else None
        self.dev = [p.to(DEV) for p in self.pools]
        self.dev_factors = [p.to(DEV) for p in self.factors] if self.factors else None

    def typed(self, x):
        return x.view(torch.bfloat16) if self.kind == "bf16" else x.view(FP8) if self.kind == "e4m3" else x

    def cut(self, pools, width):
        return pools[0][..., :width], pools[-1][..., -width:]

    def args(self):
        k, v = self.cut(self.dev, self.row)
        kw = {}
        if self.kind == "fp4":
            fk, fv = self.cut(self.dev_factors, self.D // 16)
            kw = dict(k_scales=fk.view(FP8), v_scales=fv.view(FP8))
        return (self.typed(k), self.typed(v), self.lengths.to(DEV), self.table.to(DEV)), kw

    def write(self, which, r, j, x):
        """What x (KH, D) fp32 becomes at position j of request r, in the CPU's pools."""
        page, tok = int(self.table[r, j // self.page]), j % self.page
        to = self.cut(self.pools, self.row)[which][page, :, tok]
        if self.kind == "bf16":
            to.copy_(x.to(torch.bfloat16).view(torch.uint8))
        elif self.kind == "e4m3":
            to.copy_(x.clamp(-448.0, 448.0).to(FP8).view(torch.uint8))
        else:
            codes, factors = O.quantise4(x)
            to.copy_(codes)
            self.cut(self.factors, self.D // 16)[which][page, :, tok].copy_(factors.view(torch.uint8))

    def same(self):
        torch.cuda.synchronize()
        ok = all(torch.equal(a, b.cpu()) for a, b in zip(self.pools, self.dev))
        return ok and (self.factors is None or all(torch.equal(a, b.cpu()) for a, b in zip(self.factors, self.dev_factors)))


def expect(cache, key, value, rows, rope=None, interleaved=False, at=None, descales=None, query=None):
    """Writes what the call should into the CPU's pools; the queries it should return."""
    out = None if query is None else torch.zeros_like(query)
    t = 0
    for r, n in enumerate(rows):
        L = int(cache.lengths[r])
        for i in range(n):
            j = L - n + i
            if j >= 0:
                k, v = key[t].float(), value[t].float()
                p = j if at is None else int(at[t])
                if rope is not None:
                    k = O.rotate(k[None], rope[p][None], interleaved)[0]
                    if query is not None:
                        out[t] = O.rotate(query[t].float()[None], rope[p][None], interleaved)[0].to(torch.bfloat16)
                if descales is not None:
                    k, v = k / descales[0, r][:, None], v / descales[1, r][:, None]
                cache.write(0, r, j, k)
                cache.write(1, r, j, v)
            t += 1
    return out


CASES = [
    # heads, kv_heads, head_dim, page, kind, layout, rotary, interleaved, descales, lengths, rows (None: one each), moved
    (8, 2, 128, 16, "fp4", "joint", 128, False, False, [1, 17, 40, 33], None, False),
    (8, 2, 128, 16, "fp4", "split", 128, False, True, [5, 40, 0, 33], [5, 17, 0, 2], True),
    (6, 3, 64, 24, "fp4", "joint", 64, True, False, [100, 1], [70, 1], False),
    (5, 5, 64, 1, "fp4", "split", 32, False, False, [9, 3, 50], [9, 1, 33], True),
    (16, 1, 128, 64, "fp4", "joint", 48, True, True, [64, 65, 130], [64, 65, 66], False),
    (4, 4, 128, 16, "fp4", "split", 0, False, False, [20], [20], False),
    (8, 2, 128, 16, "bf16", "joint", 128, False, False, [1, 17, 40], [1, 16, 3], False),
    (10, 2, 64, 24, "bf16", "split", 16, False, False, [30, 2], None, True),
    (2, 1, 64, 1, "bf16", "joint", 0, False, False, [7], [7], False),
    (8, 8, 128, 16, "e4m3", "joint", 64, True, True, [40, 3], [33, 3], False),
    (40, 10, 64, 1, "e4m3", "split", 64, False, False, [12, 200, 1], None, True),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:9])))
def test_append(case):
    H, KH, D, page, kind, layout, rot, inter, scaled, lengths, rows, moved = case
    g = torch.Generator().manual_seed(31)
    cache = Cache(g, lengths, KH, D, page, kind, layout)
    each = rows if rows is not None else [1] * len(lengths)
    T = sum(each)
    qkv = (3.0 * torch.randn(T, H + 2 * KH, D, generator=g)).to(torch.bfloat16)
    dev = qkv.to(DEV)
    q, k, v = qkv[:, :H], qkv[:, H: H + KH], qkv[:, H + KH:]
    rope = table_of(max(lengths) + 300, rot) if rot else None
    at = torch.randint(0, 300, (T,), generator=g) if moved and rot else None
    descales = 0.5 + torch.rand(2, len(lengths), KH, generator=g) if scaled else None
    want_q = expect(cache, k, v, each, rope, inter, at, descales, q if rot else None)
    (kc, vc, L, table), kw = cache.args()
    got = ops().append_paged_context(
        dev[:, H: H + KH], dev[:, H + KH:], kc, vc, L, table, query=dev[:, :H] if rot else None,
        cu_seqlens_q=None if rows is None else torch.tensor([0] + rows).cumsum(0).int().to(DEV),
        rope=None if rope is None else rope.to(DEV), interleaved=inter, positions=None if at is None else at.to(DEV),
        descales=None if descales is None else descales.to(DEV), **kw)
    assert cache.same()
    assert (got is None) == (want_q is None) and (got is None or torch.equal(got.cpu(), want_q))
    assert error_word() == 0


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "fp4"])
def test_positions_of_rows_that_are_not_rotated(kind):
    """Layers without a rotation take the positions of those that have one; values outside any table mean nothing."""
    g = torch.Generator().manual_seed(38)
    cache = Cache(g, [40, 17], 2, 64, 16, kind, "joint")
    k, v = ((3.0 * torch.randn(8, 2, 64, generator=g)).to(torch.bfloat16) for _ in range(2))
    expect(cache, k, v, [5, 3], None, False, None, None, None)
    (kc, vc, L, table), kw = cache.args()
    at = torch.tensor([0, 1, 900, -1, 7, 1 << 40, 2, 3], device=DEV)
    assert ops().append_paged_context(k.to(DEV), v.to(DEV), kc, vc, L, table, positions=at,
                                      cu_seqlens_q=torch.tensor([0, 5, 8], dtype=torch.int32, device=DEV), **kw) is None
    assert cache.same() and error_word() == 0


def test_formula_in_64_bits():
    g = torch.Generator().manual_seed(32)
    D, KH, L = 128, 2, 200
    k, v = ((3.0 * torch.randn(L, KH, D, generator=g)).to(torch.bfloat16) for _ in range(2))
    rope = table_of(70000, D)
    at = torch.randint(60000, 70000, (L,), generator=g)
    turned = O.rotate(k.double(), rope[at].double(), False)
    mag = O.rotate(k.double().abs(), rope[at].double().abs() * torch.tensor([1.0, -1.0]), False).abs() + turned.abs()
    for kind in ("bf16", "e4m3", "fp4"):
        cache = Cache(g, [L], KH, D, 16, kind, "split")
        (kc, vc, n, table), kw = cache.args()
        ops().append_paged_context(k.to(DEV), v.to(DEV), kc, vc, n, table, rope=rope.to(DEV), positions=at.to(DEV).int(),
                                   cu_seqlens_q=torch.tensor([0, L], dtype=torch.int32, device=DEV), **kw)
        j = torch.arange(L)
        where = (cache.table[0, j // 16].long(), slice(None), j % 16)
        for pool, factors, x in ((kc, kw.get("k_scales"), turned), (vc, kw.get("v_scales"), v.double())):
            if kind == "fp4":
                f = factors.cpu()[where]
                got = O.values4(pool.cpu()[where], f)
                y = (x.unflatten(-1, (-1, 16)) / f.double()[..., None]).abs().flatten(-2)
                # half the distance of the codes about y; above 6 (a factor rounded down by 2^-4 at most) what is cut off
                half = torch.where(y <= 2, 0.25, torch.where(y <= 4, 0.5, 1.0))
                tol = half * f.double().repeat_interleave(16, -1) + 3 * 2.0 ** -24 * (mag if x is turned else 0.0)
                assert (y <= 6 * (1 + 2.0 ** -4) + 1e-6).all()
            else:
                got = pool.cpu()[where].double()
                tol = (2.0 ** -8 if kind == "bf16" else 2.0 ** -4) * x.abs() + (0.0 if kind == "bf16" else 2.0 ** -10)
                tol = tol + 3 * 2.0 ** -24 * (mag if x is turned else 0.0)
            assert ((got - x).abs() <= tol).all(), kind


def test_values_at_the_edge_of_4_bits():
    """Zeros, ties between codes, values far too large or small, infinities and NaN."""
    D, KH = 64, 1
    rows = torch.zeros(8, KH, D)
    rows[1, 0, :16] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -0.0])
    rows[1, 0, 16:32] = 2.0 ** -12 * torch.arange(16)  # below every factor's step
    rows[1, 0, 32:48] = 2.0 ** -7 * (1 + torch.arange(16) / 16)  # factors whose steps are absolute
    rows[2, 0, 3] = 1e5  # past the largest value
    rows[2, 0, 4] = 1000.0
    rows[3, 0, 5] = math.inf
    rows[3, 0, 6] = 1.0
    rows[4, 0, 20] = -math.inf
    rows[5, 0, 40] = math.nan
    rows[5, 0, 41] = 3.0
    rows[6] = torch.randn(KH, D, generator=torch.Generator().manual_seed(3)) * 1e-20
    rows[7] = torch.randn(KH, D, generator=torch.Generator().manual_seed(4)) * 1e30
    x = rows.to(torch.bfloat16)
    g = torch.Generator().manual_seed(33)
    cache = Cache(g, [8], KH, D, 16, "fp4", "joint")
    (kc, vc, n, table), kw = cache.args()
    ops().append_paged_context(x.to(DEV), x.to(DEV), kc, vc, n, table, cu_seqlens_q=torch.tensor([0, 8], dtype=torch.int32, device=DEV),
                               **kw)
    where = (int(table[0, 0]), 0, slice(0, 8))
    got = O.values4(kc.cpu()[where], kw["k_scales"].cpu()[where])
    codes, factors = O.quantise4(x[:, 0].float())
    want = O.values4(codes, factors)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isnan(got[5, 32:48]).all() and torch.isnan(got).sum() == 16
    assert torch.equal(got.nan_to_num(), want.nan_to_num())
    assert got[2, 3] == 448 * 6 and got[3, 5] == 448 * 6 and got[4, 20] == -448 * 6
    assert torch.equal(got[1, :16].float(), torch.tensor([6.0, 0, 1, 1, 2, 2, 4, 4, 0, -1, -1, -2, -2, -4, -4, 0]))
    assert (got[0] == 0).all() and (got[6] == 0).all() and (got[1, 16:32] == 0).all()
    assert torch.equal(kc.cpu()[where], vc.cpu()[where])


def test_rows_without_a_place():
    """Padding behind the last request, more rows than positions, lengths and positions out of range."""
    g = torch.Generator().manual_seed(34)
    H, KH, D = 4, 2, 128
    cache = Cache(g, [3, 20, 40], KH, D, 16, "fp4", "joint")
    rows = [5, 2, 3]  # the first two rows of request 0 have no position
    T = sum(rows) + 4
    q, k, v = ((torch.randn(T, n, D, generator=g)).to(torch.bfloat16) for n in (H, KH, KH))
    rope = table_of(64, D)
    want = expect(cache, k, v, rows, rope, query=q)
    (kc, vc, L, table), kw = cache.args()
    cu = torch.tensor([0] + rows).cumsum(0).int().to(DEV)
    got = ops().append_paged_context(k.to(DEV), v.to(DEV), kc, vc, L, table, cu_seqlens_q=cu, query=q.to(DEV),
                                     rope=rope.to(DEV), **kw)
    assert cache.same() and torch.equal(got[:10].cpu(), want[:10]) and float(got[:2].abs().max()) == 0.0
    assert error_word() == 0
    # a length past the table, a negative one, a position past the rope's rows, a bad page
    before = [p.clone() for p in cache.dev]
    far = torch.tensor([1000, -4, 40], dtype=torch.int32, device=DEV)
    got = ops().append_paged_context(k[:3].to(DEV), v[:3].to(DEV), kc, vc, far, table, query=q[:3].to(DEV), rope=rope.to(DEV),
                                     positions=torch.tensor([0, 0, 64], device=DEV), **kw)
    torch.cuda.synchronize()
    assert float(got.abs().max()) == 0.0 and all(torch.equal(a, b) for a, b in zip(before, cache.dev))
    with pytest.raises(RuntimeError):
        ops().check_device_errors()
    ops().check_device_errors()
    bad = table.clone()
    bad[0, 0], bad[1, 1], bad[2, 2] = -1, 1 << 20, 99
    ops().append_paged_context(k[:3].to(DEV), v[:3].to(DEV), kc, vc, L, bad, **kw)
    assert all(torch.equal(a, b) for a, b in zip(before, cache.dev)) and error_word() == 4
    # row bounds that run back or past the rows
    for bounds in ([0, 5, 2, 3], [0, 2, 4, 400], [-3, 2, 4, 6]):
        ops().append_paged_context(k.to(DEV), v.to(DEV), kc, vc, L, table,
                                   cu_seqlens_q=torch.tensor(bounds, dtype=torch.int32, device=DEV), **kw)
        assert error_word() == 4, bounds


def test_many_requests():
    """Rows found among more requests than a warp has lanes, and than its square; some without rows."""
    g = torch.Generator().manual_seed(38)
    for n in (33, 700, 1500):
        rows = [int(x) for x in torch.randint(0, 3, (n,), generator=g)]
        rows[0], rows[-1] = 0, 2
        lengths = [r + int(x) for r, x in zip(rows, torch.randint(0, 4, (n,), generator=g))]
        cache = Cache(g, lengths, 1, 64, 4, "fp4", "joint")
        T = sum(rows)
        k, v = (torch.randn(T + 3, 1, 64, generator=g).to(torch.bfloat16) for _ in range(2))
        expect(cache, k, v, rows)
        (kc, vc, L, table), kw = cache.args()
        ops().append_paged_context(k.to(DEV), v.to(DEV), kc, vc, L, table, cu_seqlens_q=torch.tensor([0] + rows).cumsum(0).int().to(DEV), **kw)
        assert cache.same() and error_word() == 0


def test_strides_streams_graphs_and_far_pages():
    g = torch.Generator().manual_seed(35)
    H, KH, D, page = 4, 2, 64, 16
    # heads between other heads, rows that start between two 16-byte lines
    cache = Cache(g, [30, 7], KH, D, page, "fp4", "split")
    wide = torch.randn(2, 3, KH, D, generator=g).to(torch.bfloat16)
    odd = torch.randn(2 * KH * D + 3, generator=g).to(torch.bfloat16)
    rope = table_of(64, D)
    k, v = wide[:, 1], odd[3:].view(2, KH, D)
    expect(cache, k, v, [1, 1], rope)
    (kc, vc, L, table), kw = cache.args()
    dk, dv, dr = wide.to(DEV)[:, 1], odd.to(DEV)[3:].view(2, KH, D), rope.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops().append_paged_context(dk, dv, kc, vc, L, table, rope=dr, **kw)
    side.synchronize()
    assert cache.same()
    # captured, and replayed on other rows and lengths
    static = torch.zeros(2, H + 2 * KH, D, dtype=torch.bfloat16, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops().append_paged_context(static[:, H: H + KH], static[:, H + KH:], kc, vc, L, table, query=static[:, :H],
                                         rope=dr, **kw)
    for lengths in ([12, 1], [20, 0]):
        rows = torch.randn(2, H + 2 * KH, D, generator=g).to(torch.bfloat16)
        static.copy_(rows)
        L.copy_(torch.tensor(lengths, dtype=torch.int32))
        cache.lengths = torch.tensor(lengths)
        want = expect(cache, rows[:, H: H + KH], rows[:, H + KH:], [1, 1], rope, query=rows[:, :H])
        graph.replay()
        assert cache.same() and torch.equal(out.cpu(), want)
    # pages whose offset passes 32 bits
    stride = 2_200_000_000
    pool = torch.zeros(2 * stride + KH * page * D, dtype=torch.uint8, device=DEV)
    far = pool.as_strided((3, KH, page, D // 2), (stride, page * D, D, 1))
    far_v = pool.as_strided((3, KH, page, D // 2), (stride, page * D, D, 1), D // 2)
    f = torch.zeros(3, KH, page, D // 8, dtype=torch.uint8, device=DEV).view(FP8)
    t = torch.tensor([[2]], dtype=torch.int32, device=DEV)
    ops().append_paged_context(dk[:1], dv[:1], far, far_v, torch.tensor([3], dtype=torch.int32, device=DEV), t,
                               k_scales=f[..., : D // 16], v_scales=f[..., D // 16:])
    codes, factors = O.quantise4(k[0].float())
    assert torch.equal(far[2, :, 2].cpu(), codes) and torch.equal(f[2, :, 2, : D // 16].cpu().view(torch.uint8), factors.view(torch.uint8))
    assert torch.equal(far_v[2, :, 2].cpu(), O.quantise4(v[0].float())[0])
    assert error_word() == 0


def test_empty_calls():
    g = torch.Generator().manual_seed(36)
    cache = Cache(g, [3], 2, 64, 16, "fp4", "joint")
    (kc, vc, L, table), kw = cache.args()
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    ops().append_paged_context(none, none, kc, vc, L, table, cu_seqlens_q=torch.zeros(2, dtype=torch.int32, device=DEV), **kw)
    ops().append_paged_context(none, none, kc, vc, L[:0], table[:0], **kw)
    q = ops().append_paged_context(none, none, kc, vc, L[:0], table[:0], query=none, rope=table_of(4, 64).to(DEV), **kw)
    assert q.shape == none.shape and cache.same() and error_word() == 0


def test_refusals():
    from flashmap_b200.cache_ops import OpArgumentError
    g = torch.Generator().manual_seed(37)
    cache = Cache(g, [3, 4], 2, 64, 16, "fp4", "joint")
    (kc, vc, L, table), kw = cache.args()
    rows = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    rope = table_of(32, 64).to(DEV)
    f = ops().append_paged_context

    def refused(*a, **k):
        with pytest.raises(OpArgumentError):
            f(*a, **k)

    refused(rows, rows, kc, vc, L, table)  # no factors
    refused(rows, rows, kc, vc, L, table, k_scales=kw["k_scales"], v_scales=None)
    refused(rows, rows, kc, vc, L, table, k_scales=kw["k_scales"][:, :, :, :2], v_scales=kw["v_scales"])
    refused(rows.float(), rows, kc, vc, L, table, **kw)
    refused(rows[:, :1], rows, kc, vc, L, table, **kw)
    refused(rows[:1], rows[:1], kc, vc, L, table, **kw)  # one row for two requests
    refused(rows, rows, kc, vc, L, table, query=rows, **kw)  # without rope
    refused(rows, rows, kc, vc, L, table, query=rows[:, :1], rope=rope, **kw)
    refused(rows, rows, kc, vc, L, table, rope=rope[:, :4], **kw)
    refused(rows, rows, kc, vc, L, table, rope=rope.double(), **kw)
    refused(rows, rows, kc, vc, L, table, rope=table_of(32, 128).to(DEV), **kw)
    refused(rows, rows, kc, vc, L, table, positions=L.float(), **kw)
    refused(rows, rows, kc, vc, L, table, rope=rope, positions=L[:1], **kw)
    refused(rows, rows, kc, vc, L.long(), table, **kw)
    refused(rows, rows, kc, vc, L, table, cu_seqlens_q=L, **kw)
    refused(rows.requires_grad_(), rows, kc, vc, L, table, **kw)
    rows = rows.detach()
    wide = torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    refused(rows, rows, wide, wide, L, table, **kw)  # factors of a bf16 cache
    refused(rows, rows, wide, wide, L, table, descales=torch.ones(2, 2, 2, device=DEV))
    assert cache.same()
