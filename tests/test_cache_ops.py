"""The paged-cache operators without a GPU: the oracle's own properties and the
C entries' refusals, which come before any CUDA call."""

import ctypes
import math

import torch

from flashmap_b200 import _lib
from oracle import cache_ops as O


def _cache(**kw):
    c = _lib.PagedCache(k=1 << 20, v=1 << 21, dtype=_lib.FM_DT_BF16, k_page_stride=4096, k_head_stride=2048,
                        k_token_stride=128, v_page_stride=4096, v_head_stride=2048, v_token_stride=128, page_size=16,
                        num_pages=8, page_table=1 << 22, page_table_stride=4, page_table_cols=4, lengths=1 << 23,
                        max_length=64, requests=2, kv_heads=2, head_dim=128, descales=None)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _decode(**kw):
    a = _lib.DecodeAttn(q=1 << 24, q_request_stride=512, q_head_stride=128, heads=4, softmax_scale=0.1, window=0, sinks=0,
                        weight_sums=None, out=1 << 25, out_request_stride=512, out_head_stride=128)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _window(**kw):
    a = _lib.WindowAttn(q=1 << 24, q_token_stride=512, q_head_stride=128, rows=2, heads=4, cu_seqlens_q=1 << 26, max_q=1,
                        softmax_scale=0.1, window=0, sinks=0, out=1 << 25, out_token_stride=512, out_head_stride=128)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _evict(**kw):
    a = _lib.Evict(weight_sums=1 << 24, sums_request_stride=128, sums_head_stride=64, budget=32, sinks=4, recent=8,
                   out_page_table=None, kept=1 << 25, lengths=1 << 26, out_sums=1 << 27)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _status(name, cache, args):
    lib = _lib.load()
    return getattr(lib, name)(ctypes.byref(cache), ctypes.byref(args), None), lib.fm_last_error().decode()


INVALID, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE = 1, 2, 3, 7, 8


def test_cache_refusals():
    for name, args in (("fm_paged_decode_attn", _decode()), ("fm_paged_window_attn", _window()),
                       ("fm_paged_evict", _evict())):
        for kw, want in ((dict(k=None), INVALID), (dict(page_table=None), INVALID), (dict(lengths=None), INVALID),
                         (dict(dtype=_lib.FM_DT_F32), INVALID), (dict(head_dim=96), UNSUPPORTED),
                         (dict(kv_heads=0), SHAPE), (dict(page_size=0), SHAPE), (dict(max_length=-1), SHAPE),
                         (dict(requests=-1), SHAPE), (dict(k=(1 << 20) + 8), ALIGN), (dict(v_token_stride=132), ALIGN),
                         (dict(k_page_stride=4100), ALIGN)):
            st, msg = _status(name, _cache(**kw), args)
            assert st == want, (name, kw, st, msg)
        assert getattr(_lib.load(), name)(None, ctypes.byref(args), None) == INVALID
        assert getattr(_lib.load(), name)(ctypes.byref(_cache()), None, None) == INVALID
        # nothing to do is no error
        assert _status(name, _cache(requests=0), args)[0] == 0


def test_argument_refusals():
    for kw, want in ((dict(heads=3), SHAPE), (dict(heads=0), SHAPE), (dict(window=-1), SHAPE), (dict(sinks=-1), SHAPE),
                     (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(q_head_stride=127), ALIGN),
                     (dict(out=(1 << 25) + 4), ALIGN), (dict(weight_sums=1 << 28), WORKSPACE)):
        st, msg = _status("fm_paged_decode_attn", _cache(), _decode(**kw))
        assert st == want, (kw, st, msg)
    for kw, want in ((dict(heads=3), SHAPE), (dict(rows=-1), SHAPE), (dict(rows=1 << 40), SHAPE), (dict(window=-1), SHAPE),
                     (dict(cu_seqlens_q=None), INVALID), (dict(q=(1 << 24) + 8), ALIGN), (dict(out_head_stride=132), ALIGN)):
        st, msg = _status("fm_paged_window_attn", _cache(), _window(**kw))
        assert st == want, (kw, st, msg)
    # contexts long enough to be cut need room for the parts
    st, msg = _status("fm_paged_window_attn", _cache(max_length=4096, page_table_cols=256), _window())
    assert st == WORKSPACE, (st, msg)
    for kw, want in ((dict(budget=0), SHAPE), (dict(sinks=30, recent=3), SHAPE), (dict(recent=-1), SHAPE),
                     (dict(weight_sums=None), INVALID), (dict(kept=None), INVALID), (dict(lengths=1 << 23), INVALID),
                     (dict(out_page_table=1 << 22, out_page_table_cols=4), INVALID),
                     (dict(out_page_table=1 << 28, out_page_table_cols=1), SHAPE), ({}, WORKSPACE)):
        st, msg = _status("fm_paged_evict", _cache(), _evict(**kw))
        assert st == want, (kw, st, msg)


def test_packed_arguments_have_the_structures_layout():
    from flashmap_b200 import cache_ops as C
    for packed, fields in ((C._CACHE, _lib.PagedCache), (C._DECODE, _lib.DecodeAttn), (C._WINDOW, _lib.WindowAttn),
                           (C._EVICT, _lib.Evict)):
        assert packed.size == ctypes.sizeof(fields)
        values = [0.5 if t is ctypes.c_float else 3 + i for i, (_, t) in enumerate(fields._fields_)]
        assert packed.pack(*values) == bytes(fields(*values))


def test_workspace_sizes():
    lib = _lib.load()
    size = lib.fm_paged_decode_attn_workspace_size
    assert size(1, 32, 8, 128, 200, 0, 0, 0) == 0  # one chunk: nothing to join
    assert size(1, 32, 8, 128, 40000, 0, 0, 0) > 0
    assert size(1, 32, 8, 128, 40000, 128, 4, 0) == 0  # a window that is one chunk
    assert size(1, 32, 8, 128, 200, 0, 0, 1) >= 32 * 200 * 4  # the scores that become weights
    assert size(1, 3, 2, 128, 200, 0, 0, 0) == 0 and size(0, 4, 2, 128, 200, 0, 0, 0) == 0
    assert lib.fm_paged_evict_workspace_size(3, 4, 100) == 3 * 4 * 100 * 8


def _pool(g, n, page, KH, D):
    pages = -(-n // page)
    table = torch.randperm(pages, generator=g).view(1, pages)
    return torch.randn(pages, KH, page, D, generator=g), table


def test_oracle_window_of_one_row_is_decode():
    g = torch.Generator().manual_seed(1)
    k, table = _pool(g, 50, 8, 2, 16)
    v = torch.randn(k.shape, generator=g)
    q = torch.randn(1, 6, 16, generator=g)
    a, _, sums = O.decode_attention(q, k, v, [50], table, 0.25, window=20, sinks=3)
    b, _, _ = O.window_attention(q, k, v, [0, 1], [50], table, 0.25, window=20, sinks=3)
    assert torch.equal(a, b)
    assert torch.allclose(sums[0].sum(-1), torch.full((2,), 3.0, dtype=torch.float64))
    assert float(sums[0][:, 3:30].abs().sum()) == 0.0  # between the first tokens and the window


def test_oracle_matches_dense_attention():
    g = torch.Generator().manual_seed(2)
    k, table = _pool(g, 40, 8, 1, 16)
    v = torch.randn(k.shape, generator=g)
    q = torch.randn(40, 2, 16, generator=g)
    out, _, _ = O.window_attention(q, k, v, [0, 40], [40], table, 0.25)
    rows = k[table[0]].transpose(1, 2).reshape(40, 1, 16).double(), v[table[0]].transpose(1, 2).reshape(40, 1, 16).double()
    s = torch.einsum("qhd,kd->hqk", q.double(), rows[0][:, 0]) * 0.25
    s = s + torch.full((40, 40), -math.inf, dtype=torch.float64).triu(1)
    want = torch.einsum("hqk,kd->qhd", s.softmax(-1), rows[1][:, 0])
    assert torch.allclose(out, want, atol=1e-12)


def test_oracle_evict_rules():
    sums = torch.tensor([[[5.0, 1.0, 3.0, 3.0, math.nan, 3.0, 0.0, 9.0]]])
    assert O.evict(sums, [8], 8, 0, 0) == [[list(range(8))]]
    assert O.evict(sums, [8], 4, 0, 0) == [[[0, 2, 3, 7]]]  # ties go to the lowest position
    assert O.evict(sums, [8], 4, 2, 1) == [[[0, 1, 2, 7]]]
    assert O.evict(sums, [7], 6, 1, 1) == [[[0, 1, 2, 3, 5, 6]]]  # what is no number goes first
    assert O.evict(sums, [8], 3, 1, 2) == [[[0, 6, 7]]]


def test_strides_of_dimensions_of_one_do_not_matter():
    """A tensor may give a dimension of size 1 any stride, and nothing steps by it."""
    for kw in (dict(num_pages=1, k_page_stride=4101, v_page_stride=3), dict(kv_heads=1, k_head_stride=7, v_head_stride=1),
               dict(page_size=1, k_token_stride=5, v_token_stride=9)):
        st, msg = _status("fm_paged_evict", _cache(**kw), _evict())
        assert st == WORKSPACE, (kw, st, msg)  # the check that comes after the alignment
    st, msg = _status("fm_paged_decode_attn", _cache(requests=1), _decode(q_request_stride=3, weight_sums=1 << 28))
    assert st == WORKSPACE, (st, msg)
    st, msg = _status("fm_paged_decode_attn", _cache(kv_heads=1), _decode(heads=1, q_head_stride=3, weight_sums=1 << 28))
    assert st == WORKSPACE, (st, msg)
    long = _cache(max_length=4096, page_table_cols=256)
    st, msg = _status("fm_paged_window_attn", long, _window(rows=1, q_token_stride=5))
    assert st == WORKSPACE, (st, msg)
    long.kv_heads = 1
    st, msg = _status("fm_paged_window_attn", long, _window(heads=1, q_head_stride=5))
    assert st == WORKSPACE, (st, msg)


def test_caches_that_hold_nothing():
    """Empty tensors have no address: no pages, no table columns, no positions are no error."""
    for kw in (dict(num_pages=0, k=None, v=None), dict(page_table_cols=0, page_table=None), dict(max_length=0, k=None),
               dict(max_length=0, page_table_cols=0, page_table=None, num_pages=0, k=None, v=None)):
        st, msg = _status("fm_paged_evict", _cache(**kw), _evict())
        assert st == WORKSPACE, (kw, st, msg)  # the check that comes after the addresses
    st, msg = _status("fm_paged_evict", _cache(max_length=0), _evict(weight_sums=None))
    assert st == WORKSPACE, (st, msg)
    assert _status("fm_paged_evict", _cache(num_pages=0, lengths=None), _evict())[0] == INVALID
    assert _status("fm_paged_evict", _cache(), _evict(weight_sums=None))[0] == INVALID


def test_workspace_sizes_are_kept_by_device(monkeypatch):
    """The chunk kernel's workspace goes by the device's number of SMs."""
    from flashmap_b200 import cache_ops as C
    device = [0]

    class Library:
        def fm_paged_window_attn_workspace_size(self, *sizes):
            return sum(sizes) * (1 + device[0])

    monkeypatch.setattr(C._lib, "load", lambda: Library())
    C._workspace_size.cache_clear()
    got = []
    for device[0] in (0, 1, 0):
        got.append(C._workspace_size("fm_paged_window_attn_workspace_size", device[0], 3, 4))
    C._workspace_size.cache_clear()
    assert got == [7, 14, 7]


def test_attentions_are_registered_with_a_fake():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from flashmap_b200 import cache_ops  # noqa: F401
    with FakeTensorMode():
        k = torch.empty(4, 2, 16, 64, dtype=torch.bfloat16)
        q, L = torch.empty(3, 4, 64, dtype=torch.bfloat16), torch.empty(3, dtype=torch.int32)
        t, cu = torch.empty(3, 2, dtype=torch.int32), torch.empty(4, dtype=torch.int32)
        a = torch.ops.flashmap_b200.paged_decode_attention(q, k, k, L, t, 20, 0.1, 0, 0, None, torch.empty(3, 2, 20))
        b = torch.ops.flashmap_b200.paged_window_attention(q, k, k, cu, L, t, 1, 20, 0.1, 5, 1, None)
        for x in (a, b):
            assert x.shape == q.shape and x.dtype == q.dtype and x.is_contiguous()
