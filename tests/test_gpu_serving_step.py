"""A target's serving steps on a 4-bit cache, the operators together: prompts are
appended and attended to, tokens decoded one by one, a drafted block verified,
its rejected rows written over, and the emitted tokens scored.

The oracle repeats every step from the same inputs: rotation in fp32 (each
product and sum rounded, which the CPU repeats bit for bit), 4-bit rows by the
distance to every code, attention in 64 bits.  Outputs are held to the tolerance
of the attentions alone: (2^-11 + 2^-14) sum w |v| + (2^-8 + 2^-14) |out|.
"""

import pytest
import torch

from oracle import cache_ops as C
from oracle import serving_step as O
from oracle.accept import accept_greedy

pytestmark = pytest.mark.gpu

DEV = "cuda"
H, KH, D, PAGE, COLS, VOCAB = 8, 2, 128, 16, 12, 1003
FP8 = torch.float8_e4m3fn


class Target:
    """One attention layer over a paged 4-bit cache, on the GPU and as the oracle sees it."""

    def __init__(self, requests, seed):
        self.g = torch.Generator().manual_seed(seed)
        pages = requests * COLS
        self.table = torch.randperm(pages, generator=self.g).int().view(requests, COLS)
        self.codes = torch.zeros(2, pages, KH, PAGE, D // 2, dtype=torch.uint8)
        self.factors = torch.zeros(2, pages, KH, PAGE, D // 16, dtype=torch.uint8)
        self.lengths = torch.zeros(requests, dtype=torch.int32)
        angle = torch.arange(COLS * PAGE, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        self.rope = torch.stack([angle.cos(), angle.sin()], -1).float()
        self.dev = dict(codes=self.codes.to(DEV), factors=self.factors.to(DEV), table=self.table.to(DEV), rope=self.rope.to(DEV),
                        lengths=self.lengths.to(DEV))

    def caches(self):
        c, f = self.dev["codes"], self.dev["factors"].view(FP8)
        return c[0], c[1], f[0], f[1]

    def grow(self, rows):
        self.lengths += torch.tensor(rows, dtype=torch.int32)
        self.dev["lengths"].copy_(self.lengths)

    def draw(self, tokens):
        return torch.randn(tokens, H + 2 * KH, D, generator=self.g).to(torch.bfloat16)

    def step(self, qkv, rows):
        """Appends rows[r] tokens to every request and attends: the GPU's outputs, and the oracle's with their scale."""
        from flashmap_b200 import cache_ops
        self.grow(rows)
        kc, vc, kf, vf = self.caches()
        d = qkv.to(DEV)
        one = all(n == 1 for n in rows)
        cu = torch.tensor([0] + rows).cumsum(0).int()
        q = cache_ops.append_paged_context(d[:, H: H + KH], d[:, H + KH:], kc, vc, self.dev["lengths"], self.dev["table"],
                                           cu_seqlens_q=None if one else cu.to(DEV), query=d[:, :H], rope=self.dev["rope"],
                                           k_scales=kf, v_scales=vf)
        longest = int(self.lengths.max())
        if one:
            out = cache_ops.paged_decode_attention_fp4(q, kc, vc, kf, vf, self.dev["lengths"], self.dev["table"], longest, D ** -0.5)
        else:
            out = cache_ops.paged_window_attention_fp4(q, kc, vc, kf, vf, cu.to(DEV), self.dev["lengths"], self.dev["table"],
                                                       max(rows), longest, D ** -0.5)
        return out, self.oracle(qkv, rows, cu)

    def oracle(self, qkv, rows, cu):
        queries = torch.zeros(qkv.shape[0], H, D, dtype=torch.bfloat16)
        for r, n in enumerate(rows):
            at = torch.arange(int(self.lengths[r]) - n, int(self.lengths[r]))
            x = qkv[cu[r]: cu[r + 1]].float()
            page, tok = self.table[r, at // PAGE].long(), at % PAGE
            queries[cu[r]: cu[r + 1]] = O.rotate(x[:, :H], self.rope[at], False).to(torch.bfloat16)
            for i, y in enumerate((O.rotate(x[:, H: H + KH], self.rope[at], False), x[:, H + KH:])):
                codes, factors = O.quantise4(y)
                self.codes[i][page, :, tok], self.factors[i][page, :, tok] = codes, factors.view(torch.uint8)
        k, v = (O.values4(self.codes[i], self.factors[i].view(FP8)) for i in (0, 1))
        want, mag, _ = C.window_attention(queries, k, v, cu, self.lengths.tolist(), self.table, D ** -0.5)
        return want, mag


def close(got, want, mag):
    err = (got.double().cpu() - want).abs()
    assert (err <= (2.0 ** -11 + 2.0 ** -14) * mag + (2.0 ** -8 + 2.0 ** -14) * want.abs() + 1e-30).all()


def scored(logits, tokens):
    from flashmap_b200 import ops
    got = ops.token_logprobs(logits, tokens, top_k=4, temperature=0.8)
    lp, ent, ids, top = O.token_logprobs(logits.flatten(0, -2).cpu(), tokens.flatten().cpu().tolist(), 4, 0.8)
    assert torch.equal(got.top_ids.flatten(0, -2).cpu(), ids)
    for a, b in ((got.logprobs.flatten(), lp), (got.entropy.flatten(), ent), (got.top_logprobs.flatten(0, -2), top)):
        assert torch.allclose(a.double().cpu(), b, rtol=1e-5, atol=3e-5)
    return got


def test_prompt_decode_verify_score():
    from flashmap_b200 import cache_ops, ops
    t = Target(3, 61)
    head = (torch.randn(H * D, VOCAB, generator=t.g) / (H * D) ** 0.5 * 4).to(torch.bfloat16).to(DEV)
    prompts = [70, 5, 33]
    out, (want, mag) = t.step(t.draw(sum(prompts)), prompts)
    close(out, want, mag)
    for _ in range(3):
        out, (want, mag) = t.step(t.draw(3), [1, 1, 1])
        close(out, want, mag)
        logits = out.flatten(1) @ head
        scored(logits, logits.argmax(-1))
    # a drafted block: K tokens and the one before them, in one call
    K = 4
    out, (want, mag) = t.step(t.draw(3 * (K + 1)), [K + 1] * 3)
    close(out, want, mag)
    logits = (out.flatten(1) @ head).view(3, K + 1, VOCAB).contiguous()
    draft = logits.argmax(-1)[:, :K].contiguous()
    draft[0, 2] = (draft[0, 2] + 1) % VOCAB  # request 0 keeps two of its tokens, request 1 none
    draft[1, 0] = (draft[1, 0] + 1) % VOCAB
    accepted, bonus = ops.accept_greedy(logits, draft)
    ref, ref_bonus = accept_greedy(logits.cpu(), draft.cpu())
    assert accepted.tolist() == ref.tolist() == [2, 0, K] and bonus.tolist() == ref_bonus.tolist()
    emitted = torch.cat([draft, bonus[:, None]], 1)
    emitted[torch.arange(3, device=DEV), accepted] = bonus
    scored(logits, emitted)
    # the rejected rows leave the context, and the next tokens are written over them
    t.grow([int(n) - K for n in accepted])
    out, (want, mag) = t.step(t.draw(3), [1, 1, 1])
    close(out, want, mag)
    cache_ops.check_device_errors()


def test_captured_steps_of_a_padded_batch():
    """A decoding step captured once, with an idle request, and replayed beside a second graph of another size."""
    from flashmap_b200 import cache_ops, ops
    t = Target(4, 62)
    t.step(t.draw(20 + 37 + 9), [20, 37, 0, 9])
    head = (torch.randn(H * D, VOCAB, generator=t.g) / (H * D) ** 0.5 * 4).to(torch.bfloat16).to(DEV)
    kc, vc, kf, vf = t.caches()

    def capture(n):
        held = dict(qkv=torch.zeros(n, H + 2 * KH, D, dtype=torch.bfloat16, device=DEV), tokens=torch.zeros(n, dtype=torch.int64, device=DEV))

        def step():
            x = held["qkv"]
            q = cache_ops.append_paged_context(x[:, H: H + KH], x[:, H + KH:], kc, vc, t.dev["lengths"][:n], t.dev["table"][:n],
                                               query=x[:, :H], rope=t.dev["rope"], k_scales=kf, v_scales=vf)
            held["out"] = cache_ops.paged_decode_attention_fp4(q, kc, vc, kf, vf, t.dev["lengths"][:n], t.dev["table"][:n],
                                                               COLS * PAGE, D ** -0.5)
            held["scores"] = ops.token_logprobs(held["out"].flatten(1) @ head, held["tokens"], top_k=3)

        kept = t.dev["lengths"].clone()
        t.dev["lengths"].zero_()  # warmed up on requests that hold nothing: nothing is written
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        t.dev["lengths"].copy_(kept)
        return graph, held

    graphs = {n: capture(n) for n in (4, 2)}
    for n in (4, 2, 4):
        graph, held = graphs[n]
        rows = [1, 1, 0, 1][:n] + [0] * (4 - n)  # request 2 is idle
        t.grow(rows)
        x = t.draw(n)
        held["qkv"].copy_(x)
        held["tokens"].copy_(torch.randint(0, VOCAB, (n,), generator=t.g))
        graph.replay()
        live = [r for r in range(n) if rows[r]]
        want, mag = t.oracle(x[live], rows, torch.tensor([0] + rows).cumsum(0))
        close(held["out"][live], want, mag)
        if n == 4:
            assert float(held["out"][2].abs().max()) == 0.0
        lp, ent, ids, top = O.token_logprobs((held["out"].flatten(1) @ head).cpu(), held["tokens"].cpu().tolist(), 3, 1.0)
        s = held["scores"]
        assert torch.equal(s.top_ids.cpu(), ids) and torch.allclose(s.logprobs.double().cpu(), lp, rtol=1e-5, atol=3e-5)
    assert torch.equal(t.dev["codes"].cpu(), t.codes) and torch.equal(t.dev["factors"].cpu(), t.factors)
    cache_ops.check_device_errors()
