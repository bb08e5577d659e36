"""``token_logprobs`` against 64 bits.

Tolerances.  A thread adds up to V / 256 exponentials one after the other, and
about 40 sums are joined after that, each addition off by 2^-24; an exponential
is off by 2^-22 and by 2^-24 of its exponent d, a join's factor likewise.  So S
is off by (V / 256 + 300) 2^-24 and by 2^-22 of the mean |d|, which is under
log2 V + 2 for the rows here or carries no weight.  A log probability adds 2^-22
of itself and of log S (the constants' and the result's roundings); the entropy
sum |p d| is off by the same share of its own size.
"""

import math

import pytest
import torch

from oracle import serving_step as O

pytestmark = pytest.mark.gpu

DEV = "cuda"


def call(*a, **k):
    from flashmap_b200 import ops
    return ops.token_logprobs(*a, **k)


def error_word():
    from flashmap_b200.ops import error_word as word
    torch.cuda.synchronize()
    w = word(torch.device("cuda", torch.cuda.current_device()))
    code = int(w)
    w.zero_()
    return code


def check(got, logits, tokens, k, T):
    V = logits.shape[-1]
    lp, ent, ids, top = O.token_logprobs(logits.cpu(), tokens.cpu().tolist(), k, T)
    tol = (V / 256 + 300) * 2.0 ** -24 + 2.0 ** -22 * (math.log2(V) + 2)
    assert torch.equal(got.top_ids.cpu(), ids)
    for a, b, more in ((got.logprobs, lp, 0.0), (got.top_logprobs, top, 0.0), (got.entropy, ent, tol * math.log2(V))):
        a, b = a.double().cpu(), b.float().double()  # past fp32's range (3e38 above -3e38): -inf
        live = torch.isfinite(b)
        assert torch.equal(a[~live], b[~live]) and torch.isfinite(a[live]).all()
        err, lim = (a - b).abs()[live], tol + more + 2.0 ** -21 * (b.abs()[live] + math.log(V))
        assert (err <= lim).all(), (err / lim).max().item()


CASES = [
    # rows, V, pitch, dtype, top_k, temperature
    (1, 1, 1, torch.float32, 1, 1.0),
    (3, 2, 9, torch.bfloat16, 2, 0.5),
    (5, 33, 33, torch.bfloat16, 32, 1.0),
    (2, 255, 256, torch.float32, 0, 1.7),
    (7, 1000, 1003, torch.bfloat16, 20, 1.0),
    (4, 4097, 4100, torch.float32, 5, 0.3),
    (1, 32003, 32064, torch.float32, 32, 1.0),
    (37, 32003, 32003, torch.bfloat16, 1, 2.0),
    (2, 151936, 151936, torch.bfloat16, 20, 1.0),
    (700, 5001, 5001, torch.bfloat16, 7, 0.8),
    (1, 1500001, 1500001, torch.bfloat16, 32, 1.0),
    (2, 700001, 700001, torch.float32, 3, 1.0),
    (300, 9001, 9001, torch.bfloat16, 4, 1.0),
    (597, 140001, 140001, torch.float32, 3, 1.0),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_logprobs(case):
    n, V, pitch, dtype, k, T = case
    g = torch.Generator().manual_seed(41)
    x = torch.full((n, pitch), math.nan)
    x[:, :V] = 3.0 * torch.randn(n, V, generator=g)
    x[:, V // 2] += 8.0
    x = x.to(dtype).to(DEV)[:, :V]
    tokens = torch.randint(0, V, (n,), generator=g).to(DEV)
    tokens[0] = V - 1
    check(call(x, tokens, top_k=k, temperature=T), x, tokens, k, T)
    assert error_word() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_masks_and_empty_rows(dtype):
    """All values equal (more ties than are sorted at once), few that differ, all but some -inf, -inf alone, -0 and 0."""
    V = 9000
    x = torch.zeros(7, V)
    x[1, 4000:] = 1.0
    x[2] = -math.inf
    x[2, [8999, 17, 4096]] = torch.tensor([1.0, 2.0, 1.0])
    x[3] = -math.inf
    x[4, ::2] = -0.0
    x[5] = torch.arange(V) % 3
    x[6] = -1e4
    x[6, 5000] = 1e4
    x = x.to(dtype).to(DEV)
    tokens = torch.tensor([5, 4000, 0, 3, 1, 2, 1], device=DEV)
    for k in (0, 4, 32):
        got = call(x, tokens, top_k=k)
        check(got, x, tokens, k, 1.0)
        assert float(got.logprobs[3]) == -math.inf and float(got.entropy[3]) == 0.0 and float(got.logprobs[2]) == -math.inf
    assert error_word() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lowest_values_and_temperatures(dtype):
    """Masks of the type's lowest value (alone in a row, beside -inf, beside logits), logits at both ends, tiny and huge T."""
    V, low = 3001, torch.finfo(dtype).min
    x = 2.0 * torch.randn(8, V, generator=torch.Generator().manual_seed(45))
    x[0] = low
    x[1] = -math.inf
    x[1, 100:300] = low
    x[2, ::2] = low
    x[3] = -math.inf
    x[3, 7], x[3, 8] = 3e38, low
    x[4] *= 1e35
    x[5, 5] = 1e30
    x = x.to(dtype).to(DEV)
    tokens = torch.tensor([0, 150, 1, 7, 3, 5, 6, 3000], device=DEV)
    check(call(x, tokens, top_k=6), x, tokens, 6, 1.0)
    y, t = x[6:], tokens[6:]
    check(call(y, t, top_k=3, temperature=1e6), y, t, 3, 1e6)
    lp, ent, ids, top = O.token_logprobs(y.cpu(), t.cpu().tolist(), 3, 1e-30)  # numbers of 1e30: by their share
    got = call(y, t, top_k=3, temperature=1e-30)
    assert torch.equal(got.top_ids.cpu(), ids) and torch.equal(got.entropy.double().cpu(), ent)
    assert ((got.logprobs.double().cpu() - lp).abs() <= 2.0 ** -21 * lp.abs()).all()
    assert ((got.top_logprobs.double().cpu() - top).abs() <= 2.0 ** -21 * top.abs()).all()


def test_nan_and_infinity():
    V = 5000
    x = torch.randn(4, V, generator=torch.Generator().manual_seed(42))
    x[0, 100] = math.nan
    x[1, 4999] = math.inf
    x[2] = math.nan
    got = call(x.to(DEV), torch.zeros(4, dtype=torch.int64, device=DEV), top_k=3)
    for t in (got.logprobs, got.entropy, got.top_logprobs):
        assert torch.isnan(t[:3]).all() and torch.isfinite(t[3]).all()
    assert ((got.top_ids >= 0) & (got.top_ids < V)).all()
    want = torch.where(torch.isnan(x[0]), -math.inf, x[0]).topk(3).indices
    assert torch.equal(got.top_ids[0].cpu(), want) and int(got.top_ids[1, 0]) == 4999
    assert got.top_ids[2].tolist() == [0, 1, 2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks_over_most_of_a_long_row(dtype):
    """Rows long enough to be several blocks' work, of which some see -inf, the lowest value, or NaN alone."""
    V, low = 400003, torch.finfo(dtype).min
    x = 2.0 * torch.randn(6, V, generator=torch.Generator().manual_seed(46))
    x[0, :V // 2 + 7] = -math.inf
    x[1, 9:] = -math.inf
    x[2, 100:] = low
    x[3] = -math.inf
    x[4] = low
    x[5, V - 1] = math.nan
    x = x.to(dtype).to(DEV)
    tokens = torch.tensor([V - 1, 3, 50, 5, V // 2, 1], device=DEV)
    for k in (0, 32):
        got = call(x, tokens, top_k=k)
        check(type(got)(*[t[:5] for t in got]), x[:5], tokens[:5], k, 1.0)
        assert torch.isnan(got.logprobs[5]) and torch.isnan(got.entropy[5]) and torch.isnan(got.top_logprobs[5]).all()
    assert torch.equal(got.top_ids[5], torch.where(torch.isnan(x[5]), -math.inf, x[5]).float().sort(stable=True, descending=True).indices[:32])
    assert error_word() == 0


def test_ids_outside_the_vocabulary():
    x = torch.randn(3, 100, device=DEV)
    got = call(x, torch.tensor([-1, 100, 5], device=DEV))
    assert got.logprobs[:2].tolist() == [-math.inf] * 2 and math.isfinite(float(got.logprobs[2]))
    assert error_word() == 4


def test_shapes_streams_graphs_and_repeats():
    g = torch.Generator().manual_seed(43)
    x = (2.0 * torch.randn(3, 5, 3003, generator=g)).to(torch.bfloat16).to(DEV)
    tokens = torch.randint(0, 3003, (3, 5), generator=g).to(DEV)
    a = call(x, tokens, top_k=4)
    assert a.logprobs.shape == (3, 5) and a.top_ids.shape == (3, 5, 4)
    check(type(a)(*[t.flatten(0, 1) for t in a]), x.flatten(0, 1), tokens.flatten(), 4, 1.0)
    one = call(x[1, 2], tokens[1, 2], top_k=4)
    assert one.logprobs.shape == () and torch.equal(one.top_ids, a.top_ids[1, 2])
    strided = call(x.transpose(0, 1)[:, :, 1:], (tokens.T - 1).clamp(min=0).contiguous(), top_k=2)
    check(type(a)(*[t.flatten(0, 1) for t in strided]), x.transpose(0, 1)[:, :, 1:].reshape(15, 3002),
          (tokens.T - 1).clamp(min=0).flatten(), 2, 1.0)
    empty = call(x[:0], tokens[:0], top_k=3)
    assert empty.top_logprobs.shape == (0, 5, 3)
    row = (2.0 * torch.randn(1, 100003, generator=g)).to(DEV)
    t = torch.tensor([77], device=DEV)
    runs = [call(row, t, top_k=9) for _ in range(3)]
    assert all(torch.equal(p, q) for r in runs[1:] for p, q in zip(runs[0], r))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(row, t, top_k=9)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(runs[0], other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call(row, t, top_k=9)
    row.copy_(2.0 * torch.randn(1, 100003, generator=g))
    graph.replay()
    check(held, row, t, 9, 1.0)


def test_rows_past_32_bit_offsets():
    V, stride = 500, 2_200_000_000
    pool = torch.empty(stride + V, dtype=torch.bfloat16, device=DEV)
    x = pool.as_strided((2, V), (stride, 1))
    x.copy_(torch.randn(2, V, generator=torch.Generator().manual_seed(44)))
    t = torch.tensor([3, 4], device=DEV)
    check(call(x, t, top_k=5), x.contiguous(), t, 5, 1.0)


def test_refusals():
    x, t = torch.randn(2, 50, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    for a, k in (((x.half(), t), {}), ((x.cpu(), t), {}), ((x, t.int()), {}), ((x, t[:1]), {}), ((x, t.cpu()), {}),
                 ((x, t), dict(top_k=33)), ((x, t), dict(top_k=-1)), ((x[:, :3], t), dict(top_k=4)), ((x, t), dict(temperature=0.0)),
                 ((x, t), dict(temperature=math.nan)), ((x, t), dict(temperature=math.inf)), ((x[:, ::2], t), {}),
                 ((x.clone().requires_grad_(), t), {}), ((x[:, :0], t), {})):
        with pytest.raises((ValueError, RuntimeError)):
            call(*a, **k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [9, 603])  # a cluster to a row, a block to a row
@pytest.mark.parametrize("T", [1.0, 0.7, 0.01])
def test_large_logits(dtype, rows, T):
    """Logits whose products with log2(e) / T are rounded by more than the exponentials' range (masks of -1e10 or -1e30 all
    over a row, single large ones), and ones about 2^24, where the kernel changes how it forms differences."""
    V, g = 3001, torch.Generator().manual_seed(48)
    x = 2.0 * torch.randn(rows, V, generator=g)
    border = round(2.0 ** 24 * T / math.log2(math.e))
    x[0] = -1e10
    x[1] *= 1e10
    x[2] = -7e29
    x[2, 50:60] = -6.9e29
    x[3, 77] = 1e12
    x[4] = border + torch.randint(-4, 5, (V,), generator=g)
    x[5] = -border + torch.randint(-4, 5, (V,), generator=g)
    x[6] = -1e9
    x[6, 3::7] = -1e9 + 64
    x[7] = -3.3e30
    x[7, :1500] = -1e4
    x = x.to(dtype).to(DEV)
    tokens = torch.randint(0, V, (rows,), generator=g).to(DEV)
    for k in (0, 5):
        got = call(x, tokens, top_k=k, temperature=T)
        check(type(got)(*[t[:9] for t in got]), x[:9], tokens[:9], k, T)
    assert error_word() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [3, 600])  # a cluster to a row, a block to a row
@pytest.mark.parametrize("T", [1.0, 1.3, 1.5, 0.6])
def test_tokens_of_the_lowest_value(dtype, rows, T):
    """A mask of the type's lowest value beside ordinary and beside huge logits, as the given token and among the
    alternatives: about -3.4e38 / T, which fp32 holds for a T of 1 and more; under 1 it is -inf."""
    V, low, n = 3001, torch.finfo(dtype).min, 7
    x = torch.full((rows, V), low)
    open_ids = [3, 700, 701, 1500, 2999, 3000]
    x[:, open_ids] = 3.0 * torch.randn(rows, 6, generator=torch.Generator().manual_seed(47))
    x[2, open_ids] *= 1e31  # the row's largest value times log2(e) is no ordinary number
    x = x.to(dtype)
    tokens = torch.full((rows,), 5)
    tokens[1] = 700
    x, tokens = x.to(DEV), tokens.to(DEV)
    got = call(x, tokens, top_k=n, temperature=T)
    check(type(got)(*[t[:4] for t in got]), x[:4], tokens[:4], n, T)
    ordinary = torch.arange(rows, device=DEV) != 2  # at T = 1 that row's masks are past fp32's range
    assert math.isinf(float(got.logprobs[0])) == (T < 1) and (torch.isinf(got.top_logprobs[ordinary, 6]) == (T < 1)).all()
    assert torch.isfinite(got.top_logprobs[:, :6]).all() and error_word() == 0


@pytest.mark.parametrize("rows", [1, 128, 700])
@pytest.mark.parametrize("T", [1.0, 0.7])
def test_signs_of_certain_tokens(rows, T):
    """One logit far above the rest, at values whose products with log2(e) / T round either way, and rows whose maximum
    comes a little after a thread's first values: no log probability above 0, no entropy below 0."""
    V = 5000
    top = (1.3 + 0.37 * torch.arange(rows)) % 40
    x = torch.full((rows, V), -80.0)
    at = torch.arange(rows) * 7 % V
    x[torch.arange(rows), at] = top
    x[rows // 2:, 0] = top[rows // 2:] - 16.5  # e^-16.5 = 7e-8 of it
    x, tokens = x.to(DEV), at.to(DEV)
    got = call(x, tokens, top_k=3, temperature=T)
    check(got, x, tokens, 3, T)
    for t in (got.logprobs, got.top_logprobs, -got.entropy):
        assert (t <= 0).all(), t.max().item()
