"""Appending, 4-bit caches and token log probabilities without a GPU: the
oracle's own properties and the C entries' refusals, which come before any CUDA
call."""

import ctypes
import math

import torch

from flashmap_b200 import _lib
from oracle import serving_step as O

INVALID, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE = 1, 2, 3, 7, 8


def _cache(**kw):
    c = _lib.PagedCache(k=1 << 20, v=1 << 21, dtype=_lib.FM_DT_E2M1, k_page_stride=4096, k_head_stride=2048,
                        k_token_stride=64, v_page_stride=4096, v_head_stride=2048, v_token_stride=64, page_size=16,
                        num_pages=8, page_table=1 << 22, page_table_stride=4, page_table_cols=4, lengths=1 << 23,
                        max_length=64, requests=2, kv_heads=2, head_dim=128, descales=None)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _scales(**kw):
    s = _lib.BlockScales(k=1 << 24, v=1 << 25, k_page_stride=512, k_head_stride=256, k_token_stride=8, v_page_stride=512,
                         v_head_stride=256, v_token_stride=8)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _append(**kw):
    a = _lib.Append(key=1 << 26, value=1 << 27, k_token_stride=256, k_head_stride=128, v_token_stride=256, v_head_stride=128,
                    query=1 << 28, q_token_stride=512, q_head_stride=128, heads=4, out=1 << 29, out_token_stride=512,
                    out_head_stride=128, tokens=2, rope=1 << 30, rope_rows=64, rotary_dim=128)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _status(cache, scales, args):
    lib = _lib.load()
    st = lib.fm_paged_append(ctypes.byref(cache), None if scales is None else ctypes.byref(scales), ctypes.byref(args), None)
    return st, lib.fm_last_error().decode()


def test_append_refusals():
    for cache, scales, args, want in (
            (_cache(dtype=_lib.FM_DT_F32), _scales(), _append(), INVALID),
            (_cache(k=None), _scales(), _append(), INVALID),
            (_cache(head_dim=96), _scales(), _append(), UNSUPPORTED),
            (_cache(k_token_stride=72), _scales(), _append(), ALIGN),
            (_cache(), None, _append(), INVALID),
            (_cache(), _scales(k=None), _append(), INVALID),
            (_cache(), _scales(v_token_stride=4), _append(), ALIGN),
            (_cache(), _scales(k=(1 << 24) + 4), _append(), ALIGN),
            (_cache(), _scales(), _append(tokens=3), SHAPE),
            (_cache(), _scales(), _append(tokens=-1), SHAPE),
            (_cache(), _scales(), _append(heads=0), SHAPE),
            (_cache(), _scales(), _append(rotary_dim=24), SHAPE),
            (_cache(), _scales(), _append(rotary_dim=144), SHAPE),
            (_cache(), _scales(), _append(rotary_dim=0), SHAPE),
            (_cache(), _scales(), _append(rope=None), INVALID),
            (_cache(), _scales(), _append(positions=1 << 31, positions_dtype=7), INVALID),
            (_cache(), _scales(), _append(key=None), INVALID),
            (_cache(), _scales(), _append(out=None), INVALID),
            (_cache(), _scales(), _append(key=(1 << 26) + 8), ALIGN),
            (_cache(), _scales(), _append(q_head_stride=132), ALIGN),
            (_cache(dtype=_lib.FM_DT_BF16, descales=1 << 31), None, _append(), INVALID)):
        st, msg = _status(cache, scales, args)
        assert st == want and "paged_append" in msg, (st, want, msg)
    # nothing to do
    assert _status(_cache(requests=0), _scales(), _append(tokens=0))[0] == 0
    assert _status(_cache(), _scales(), _append(tokens=0, cu_seqlens_q=1 << 31))[0] == 0


def test_logprobs_refusals():
    lib = _lib.load()

    def status(dtype=_lib.FM_DT_BF16, stride=100, tokens=1 << 21, rows=2, V=100, T=1.0, k=3, logits=1 << 20, ids=1 << 22, ws=1 << 23,
               size=1 << 30):
        return lib.fm_token_logprobs(logits, dtype, stride, tokens, rows, V, T, k, 1 << 24, 1 << 25, ids, 1 << 26, ws, size, None,
                                     None)

    for kw, want in ((dict(dtype=_lib.FM_DT_E4M3), SHAPE), (dict(rows=-1), SHAPE), (dict(V=0), SHAPE), (dict(k=33, V=100), SHAPE),
                     (dict(V=2), SHAPE), (dict(k=-1), SHAPE), (dict(V=1 << 31), SHAPE), (dict(T=0.0), INVALID),
                     (dict(T=4e-39), INVALID), (dict(T=math.nan), INVALID), (dict(T=math.inf), INVALID), (dict(logits=None), INVALID),
                     (dict(tokens=None), INVALID), (dict(ids=None), INVALID), (dict(logits=(1 << 20) + 1), ALIGN),
                     (dict(V=151936, rows=1000, ws=None), WORKSPACE), (dict(V=151936, rows=1000, size=8), WORKSPACE),
                     (dict(V=151936, rows=1000, ws=(1 << 23) + 8), ALIGN)):
        assert status(**kw) == want, kw
    assert status(rows=0) == 0
    assert lib.fm_token_logprobs_workspace_size(0, 100, 0, 0) == 0
    assert lib.fm_token_logprobs_workspace_size(1000, 151936, 0, 5) > 0
    assert lib.fm_token_logprobs_workspace_size(1, 151936, 0, 5) == 0 == lib.fm_token_logprobs_workspace_size(1000, 151936, 0, 0)


def test_four_bit_rows():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(50, 128, generator=g)
    codes, factors = O.quantise4(x)
    assert codes.shape == (50, 64) and factors.shape == (50, 8)
    back = O.values4(codes, factors)
    again = O.quantise4(back)  # what 4 bits hold comes back, unless the factor was rounded up past its largest value
    top = back.unflatten(-1, (-1, 16)).abs().amax(-1) == 6 * factors.double()
    assert torch.equal(again[1].double()[top], factors.double()[top])
    # the nearest code, on a grid of every tie
    ties = torch.tensor([6.0] + [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0] + [0.2, 0.3, 0.7, 1.3, 2.4, 3.6, 4.9, 5.1])
    c, f = O.quantise4(ties[None])
    assert float(f) == 1.0
    assert O.values4(c, f)[0].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, .5, .5, 1.5, 2, 4, 4, 6]


def test_rotation_is_one():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 3, 64, generator=g, dtype=torch.float64)
    angle = torch.rand(4, 16, generator=g, dtype=torch.float64)
    cs = torch.stack([angle.cos(), angle.sin()], -1)
    for inter in (False, True):
        y = O.rotate(x, cs, inter)
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1)) and torch.equal(y[..., 32:], x[..., 32:])
        back = O.rotate(y, cs * torch.tensor([1.0, -1.0]), inter)
        assert torch.allclose(back, x)


def test_token_logprobs_oracle():
    x = torch.tensor([[0.0, 1.0, 1.0, -math.inf], [-math.inf] * 4])
    lp, ent, ids, top = O.token_logprobs(x, [3, 0], 3, 0.5)
    p = torch.softmax(x[0].double() * 2, 0)
    assert lp[0] == -math.inf and torch.allclose(ent[0], -(p[:3] * p[:3].log()).sum()) and float(ent[1]) == 0.0
    assert ids.tolist() == [[1, 2, 0], [0, 1, 2]] and torch.allclose(top[0], p[[1, 2, 0]].log())
