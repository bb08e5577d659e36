"""Operators on a paged key/value cache that a target model decodes with:

* ``paged_decode_attention``: attention of one new token per request, split
  over the cache's length and joined, which can also gather each position's
  attention weight;
* ``paged_window_attention``: causal attention of chunks of query rows (a
  prompt, a drafted block to verify) with a sliding window and first tokens
  that stay visible;
* ``evict_paged_context``: cuts contexts to a budget of positions, those that
  gathered the most attention weight among them;
* ``append_paged_context``: writes new tokens' keys and values, rotated on the
  way, and rotates their queries;
* ``paged_decode_attention_fp4`` and ``paged_window_attention_fp4``: the two
  attentions on a cache held in 4 bits.

The cache is given by two views ``k_cache`` and ``v_cache (pages, kv_heads,
page_size, head_dim)``, bf16 or e4m3, whose rows are contiguous and 16-byte
aligned; the other strides are free.  For vLLM's joint cache they are
``kv_cache[..., :head_dim]`` and ``kv_cache[..., head_dim:]``; for a pool of
rows ``(slots, kv_heads, head_dim)`` they are ``pool.unsqueeze(2)``, a page
size of 1.  Token i of request r is token ``i % page_size`` of page
``block_table[r, i // page_size]``.  An e4m3 cache takes ``descales (2,
requests, kv_heads)``, the factors of keys and values.

A 4-bit cache is ``k_cache`` and ``v_cache (pages, kv_heads, page_size, head_dim
/ 2)`` uint8, e2m1 codes of 0, .5, 1, 1.5, 2, 3, 4, 6 and a sign bit, value 2 i in
the low half of byte i, with ``k_scales`` and ``v_scales (pages, kv_heads,
page_size, head_dim / 16)`` e4m3, the factor of each 16 values (rows of factors
aligned to their 4 or 8 bytes): 0.5625 bytes a value.  ``append_paged_context``
writes it, and f16 holds its values exactly.

Query head h reads kv head ``h // (heads / kv_heads)``.  Scores, softmax sums
and outputs are held in fp32; the softmax numerators are rounded to bf16 (to
f16 for an e4m3 or 4-bit cache, 2^11 or more of a row's largest) for the product with
the values, and the output to bf16.
A row that sees no position is zero.  A position that no row of a request may
see is never read.  Each call checks its arguments (``OpArgumentError``; the
alignment of addresses and strides and the limits of sizes are the library's to
check, ``FlashMapError``), records lengths, bounds and page ids out of range
for ``check_device_errors``, runs on the current stream without a host
synchronisation, and can be captured in a CUDA graph.  The two attentions are
registered operators (``flashmap_b200::paged_decode_attention[_fp4]``,
``::paged_window_attention[_fp4]``) to ``torch.compile``, which breaks a graph at the
other calls; they have no gradient, and asking for one raises.  There is no fallback.
"""

from __future__ import annotations

import functools
import struct
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .serving_ops import OpArgumentError, _err, _need

__all__ = ["OpArgumentError", "paged_decode_attention", "paged_window_attention", "evict_paged_context",
           "append_paged_context", "paged_decode_attention_fp4", "paged_window_attention_fp4", "check_device_errors"]

_FP8 = torch.float8_e4m3fn

# fm_paged_cache, fm_decode_attn, fm_window_attn and fm_evict as the C entries
# read them (native sizes and alignment): packing one takes a fifth of the time
# that filling a ctypes.Structure of these fields does.
_CACHE = struct.Struct("@PPiqqqqqqqqPqqPqqqqP")
_DECODE = struct.Struct("@PqqqfqqPqqPqqPNP")
_WINDOW = struct.Struct("@PqqqqPqfqqPqqPNP")
_EVICT = struct.Struct("@PqqqqqPqqPPPPNP")
_SCALES = struct.Struct("@PPqqqqqq")
_APPEND = struct.Struct("@PPqqqqPqqqPqqqPPiPqqiP")


class _Cache(NamedTuple):
    """A checked cache: its packed fm_paged_cache and the sizes that calls go by."""
    packed: bytes
    device: torch.device
    requests: int
    kv_heads: int
    page_size: int
    head_dim: int
    max_length: int


class _Cache4(NamedTuple):
    """A checked 4-bit cache: ``_Cache`` and its factors' packed fm_block_scales."""
    packed: bytes
    scales: bytes
    device: torch.device
    requests: int
    kv_heads: int
    page_size: int
    head_dim: int
    max_length: int


def _on(t: torch.Tensor, name: str, device) -> None:
    if t.device != device:
        raise OpArgumentError(f"{name} must be on {device}, got {t.device}")


def _refuse_cache(k_cache, v_cache, lengths, block_table, descales, max_len: int) -> None:
    """Raises for the argument that ``_cache`` could not take."""
    _need(k_cache.is_cuda, "k_cache must be a CUDA tensor")
    dev = k_cache.device
    _need(dev.index == torch.cuda.current_device(), f"the cache is on {dev}, which is not the current device")
    _on(v_cache, "v_cache", dev)
    _on(lengths, "the lengths", dev)
    _on(block_table, "block_table", dev)
    _need(k_cache.dtype in (torch.bfloat16, _FP8), f"the cache must be bf16 or e4m3, got {k_cache.dtype}")
    _need(v_cache.dtype == k_cache.dtype, "k_cache and v_cache must share a dtype")
    _need(k_cache.dim() == 4 and v_cache.shape == k_cache.shape,
          "k_cache and v_cache must both be (pages, kv_heads, page_size, head_dim)")
    _need(k_cache.shape[3] in (64, 128), f"head_dim must be 64 or 128, got {k_cache.shape[3]}")
    _need(k_cache.shape[1] > 0 and k_cache.shape[2] > 0, "the cache needs a kv head and a token to a page")
    _need(k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "cache rows must be contiguous")
    _need(lengths.dtype == torch.int32 and lengths.dim() == 1 and lengths.is_contiguous(),
          "the lengths must be contiguous int32 (requests,)")
    _need(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == lengths.shape[0],
          "block_table must be int32 (requests, pages)")
    _need(block_table.shape[1] <= 1 or block_table.stride(1) == 1, "block_table rows must be contiguous")
    _need(max_len >= 0, "the largest length must not be negative")
    if k_cache.dtype == torch.bfloat16:
        _need(descales is None, "descales go with an e4m3 cache")
    elif descales is not None:
        _on(descales, "descales", dev)
        _need(descales.dtype == torch.float32 and descales.is_contiguous()
              and descales.shape == (2, lengths.shape[0], k_cache.shape[1]),
              "descales must be contiguous float32 (2, requests, kv_heads)")


def _cache(k_cache, v_cache, lengths, block_table, descales, max_len: int) -> _Cache:
    # one condition on the way through; which part of it failed is found out only then
    dev, dtype = k_cache.device, k_cache.dtype
    shape, ks, vs, ts, table = k_cache.shape, k_cache.stride(), v_cache.stride(), block_table.stride(), block_table.shape
    if not (dev.type == "cuda" and dev.index == torch._C._cuda_getDevice() and v_cache.device == dev
            and lengths.device == dev and block_table.device == dev and v_cache.dtype == dtype
            and (dtype == torch.bfloat16 and descales is None or dtype == _FP8)
            and len(shape) == 4 and v_cache.shape == shape and shape[3] in (64, 128) and shape[1] > 0 and shape[2] > 0
            and ks[3] == 1 and vs[3] == 1 and lengths.dtype == torch.int32 and block_table.dtype == torch.int32
            and lengths.dim() == 1 and lengths.is_contiguous() and len(table) == 2 and table[0] == lengths.shape[0]
            and (table[1] <= 1 or ts[1] == 1) and max_len >= 0
            and (descales is None or descales.device == dev and descales.dtype == torch.float32
                 and descales.is_contiguous() and descales.shape == (2, table[0], shape[1]))):
        _refuse_cache(k_cache, v_cache, lengths, block_table, descales, max_len)
        raise OpArgumentError("the cache's tensors do not go together")
    return _Cache(_CACHE.pack(k_cache.data_ptr(), v_cache.data_ptr(),
                              _lib.FM_DT_BF16 if dtype == torch.bfloat16 else _lib.FM_DT_E4M3,
                              ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], shape[2], shape[0], block_table.data_ptr(),
                              ts[0], table[1], lengths.data_ptr(), max_len, table[0], shape[1], shape[3],
                              0 if descales is None else descales.data_ptr()),
                  dev, table[0], shape[1], shape[2], shape[3], max_len)


def _refuse_cache4(k_cache, v_cache, k_scales, v_scales, lengths, block_table, descales, max_len: int) -> None:
    """Raises for the argument that ``_cache4`` could not take."""
    _need(k_cache.is_cuda, "k_cache must be a CUDA tensor")
    dev = k_cache.device
    _need(dev.index == torch.cuda.current_device(), f"the cache is on {dev}, which is not the current device")
    _need(k_scales is not None and v_scales is not None, "a 4-bit cache needs k_scales and v_scales")
    for t, name in ((v_cache, "v_cache"), (k_scales, "k_scales"), (v_scales, "v_scales"), (lengths, "the lengths"),
                    (block_table, "block_table")):
        _on(t, name, dev)
    _need(k_cache.dtype == torch.uint8 and v_cache.dtype == torch.uint8, f"a 4-bit cache is uint8, got {k_cache.dtype}")
    _need(k_cache.dim() == 4 and v_cache.shape == k_cache.shape,
          "k_cache and v_cache must both be (pages, kv_heads, page_size, head_dim / 2)")
    _need(k_cache.shape[3] in (32, 64), f"head_dim must be 64 or 128, got {2 * k_cache.shape[3]}")
    _need(k_cache.shape[1] > 0 and k_cache.shape[2] > 0, "the cache needs a kv head and a token to a page")
    _need(k_scales.dtype == _FP8 and v_scales.dtype == _FP8, f"k_scales and v_scales must be e4m3, got {k_scales.dtype}")
    rows = (*k_cache.shape[:3], k_cache.shape[3] // 8)
    _need(k_scales.shape == rows and v_scales.shape == rows,
          "k_scales and v_scales must both be (pages, kv_heads, page_size, head_dim / 16)")
    _need(k_cache.stride(3) == 1 and v_cache.stride(3) == 1 and k_scales.stride(3) == 1 and v_scales.stride(3) == 1,
          "cache rows must be contiguous")
    _need(lengths.dtype == torch.int32 and lengths.dim() == 1 and lengths.is_contiguous(),
          "the lengths must be contiguous int32 (requests,)")
    _need(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == lengths.shape[0],
          "block_table must be int32 (requests, pages)")
    _need(block_table.shape[1] <= 1 or block_table.stride(1) == 1, "block_table rows must be contiguous")
    _need(max_len >= 0, "the largest length must not be negative")
    if descales is not None:
        _on(descales, "descales", dev)
        _need(descales.dtype == torch.float32 and descales.is_contiguous()
              and descales.shape == (2, lengths.shape[0], k_cache.shape[1]),
              "descales must be contiguous float32 (2, requests, kv_heads)")


def _cache4(k_cache, v_cache, k_scales, v_scales, lengths, block_table, descales, max_len: int) -> _Cache4:
    dev, u8 = k_cache.device, torch.uint8
    if k_scales is None or v_scales is None:
        _refuse_cache4(k_cache, v_cache, k_scales, v_scales, lengths, block_table, descales, max_len)
    shape, ks, vs, ts, table = k_cache.shape, k_cache.stride(), v_cache.stride(), block_table.stride(), block_table.shape
    fk, fv = k_scales.stride(), v_scales.stride()
    if not (dev.type == "cuda" and dev.index == torch._C._cuda_getDevice() and v_cache.device == dev
            and k_scales.device == dev and v_scales.device == dev and lengths.device == dev and block_table.device == dev
            and k_cache.dtype == u8 and v_cache.dtype == u8 and k_scales.dtype == _FP8 and v_scales.dtype == _FP8
            and len(shape) == 4 and v_cache.shape == shape and shape[3] in (32, 64) and shape[1] > 0 and shape[2] > 0
            and k_scales.shape == (shape[0], shape[1], shape[2], shape[3] // 8) and v_scales.shape == k_scales.shape
            and ks[3] == 1 and vs[3] == 1 and fk[3] == 1 and fv[3] == 1
            and lengths.dtype == torch.int32 and block_table.dtype == torch.int32
            and lengths.dim() == 1 and lengths.is_contiguous() and len(table) == 2 and table[0] == lengths.shape[0]
            and (table[1] <= 1 or ts[1] == 1) and max_len >= 0
            and (descales is None or descales.device == dev and descales.dtype == torch.float32
                 and descales.is_contiguous() and descales.shape == (2, table[0], shape[1]))):
        _refuse_cache4(k_cache, v_cache, k_scales, v_scales, lengths, block_table, descales, max_len)
        raise OpArgumentError("the cache's tensors do not go together")
    return _Cache4(_CACHE.pack(k_cache.data_ptr(), v_cache.data_ptr(), _lib.FM_DT_E2M1, ks[0], ks[1], ks[2],
                               vs[0], vs[1], vs[2], shape[2], shape[0], block_table.data_ptr(), ts[0], table[1],
                               lengths.data_ptr(), max_len, table[0], shape[1], 2 * shape[3],
                               0 if descales is None else descales.data_ptr()),
                   _SCALES.pack(k_scales.data_ptr(), v_scales.data_ptr(), fk[0], fk[1], fk[2], fv[0], fv[1], fv[2]),
                   dev, table[0], shape[1], shape[2], 2 * shape[3], max_len)


def _query(query, cache: _Cache, device) -> torch.Tensor:
    shape, stride = query.shape, query.stride()
    if not (query.device == device and query.dtype == torch.bfloat16 and len(shape) == 3
            and shape[2] == cache.head_dim and shape[1] > 0 and shape[1] % cache.kv_heads == 0):
        _on(query, "query", device)
        _need(query.dtype == torch.bfloat16 and query.dim() == 3, "query must be bf16 (rows, heads, head_dim)")
        _need(shape[2] == cache.head_dim, f"query has rows of {shape[2]}, the cache of {cache.head_dim}")
        raise OpArgumentError(f"{shape[1]} query heads are no multiple of {cache.kv_heads} kv heads")
    if stride[2] != 1 or stride[0] % 8 or stride[1] % 8 or query.data_ptr() % 16:
        query = query.contiguous()
        if query.data_ptr() % 16:  # a contiguous view that starts between two 16-byte lines
            query = query.clone()
    return query


def _visibility(window: int, sinks: int) -> None:
    _need(window >= 0 and sinks >= 0, "window and sinks must not be negative")


def _sums(weight_sums, cache: _Cache, device, least: int) -> None:
    _on(weight_sums, "weight_sums", device)
    _need(weight_sums.dtype is torch.float32 and weight_sums.dim() == 3
          and weight_sums.shape[0] == cache.requests and weight_sums.shape[1] == cache.kv_heads,
          "weight_sums must be float32 (requests, kv_heads, positions)")
    if not (weight_sums.shape[2] >= least):
        raise OpArgumentError(f"weight_sums has {weight_sums.shape[2]} positions, {least} are needed")
    _need(weight_sums.shape[2] <= 1 or weight_sums.stride(2) == 1, "weight_sums rows must be contiguous")


def _apart(sums) -> bool:
    """Whether no two of the rows share memory, for strides that do not show it at a glance."""
    reach = sums.shape[2]
    for stride, size in sorted((sums.stride(d), sums.shape[d]) for d in (0, 1) if sums.shape[d] > 1):
        if stride < reach:
            return False
        reach += stride * (size - 1)
    return True


_ERR_WORDS: dict = {}  # device index -> address of its error word, which lives as long as the process


def _err_word(device) -> int:
    err = _ERR_WORDS.get(device.index)
    if err is None:
        err = _ERR_WORDS[device.index] = _err(device).data_ptr()
    return err


def check_device_errors(device=None) -> None:
    """Raises ``FlashMapError`` for what kernels of this process have recorded
    on `device` (the current one by default) since the last check, an index out
    of range or a wait that ran out, and clears it.  Waits for the device's
    current stream; the calls themselves wait for nothing and go on past both."""
    word = _err(torch.device("cuda") if device is None else device)
    code = int(word.item())
    if code:
        word.zero_()
        raise _lib.FlashMapError(f"a FlashMap kernel reported device error {code} (index or wait)")


@functools.lru_cache(maxsize=1024)
def _workspace_size(name: str, device: int, *sizes: int) -> int:
    # the index of the current device is part of the key: a size may go by its number of SMs
    return getattr(_lib.load(), name)(*sizes)


def _launch(name: str, cache: _Cache, args: bytes) -> None:
    status = getattr(_lib.load(), name)(cache.packed, args, torch._C._cuda_getCurrentRawStream(cache.device.index))
    if status:
        _lib.check(status, name)


def _decode(query, k_cache, v_cache, seqused_k, block_table, max_seqlen_k, softmax_scale, window, sinks, descales,
            weight_sums) -> torch.Tensor:
    cache = _cache(k_cache, v_cache, seqused_k, block_table, descales, int(max_seqlen_k))
    dev = k_cache.device
    query = _query(query, cache, dev)
    shape = query.shape
    if shape[0] != cache.requests or window < 0 or sinks < 0:
        _need(shape[0] == cache.requests, "one query row per request")
        _visibility(window, sinks)
    out = query.new_empty(shape)
    sums, s0, s1 = 0, 0, 0
    if weight_sums is not None:
        _sums(weight_sums, cache, dev, cache.max_length)
        sums, s0, s1 = weight_sums.data_ptr(), weight_sums.stride(0), weight_sums.stride(1)
        inner, outer, n = (s1, s0, cache.kv_heads) if s1 <= s0 else (s0, s1, cache.requests)
        if inner < weight_sums.shape[2] or outer < inner * (n - 1) + weight_sums.shape[2]:  # a dimension of size 1 may have any stride
            _need(_apart(weight_sums), "rows of weight_sums must not share memory")
    if cache.requests == 0:
        return out
    heads, qs = shape[1], query.stride()
    need = _workspace_size("fm_paged_decode_attn_workspace_size", dev.index, cache.requests, heads, cache.kv_heads,
                           cache.head_dim, cache.max_length, window, sinks, int(weight_sums is not None))
    ws = seqused_k.new_empty(need // 4) if need else None  # sizes are multiples of 8
    _launch("fm_paged_decode_attn", cache,
            _DECODE.pack(query.data_ptr(), qs[0], qs[1], heads, softmax_scale, window, sinks, sums, s0, s1,
                         out.data_ptr(), heads * cache.head_dim, cache.head_dim, ws.data_ptr() if need else 0, need,
                         _err_word(dev)))
    return out


def _window(query, k_cache, v_cache, cu_seqlens_q, seqused_k, block_table, max_seqlen_q, max_seqlen_k, softmax_scale,
            window, sinks, descales) -> torch.Tensor:
    cache = _cache(k_cache, v_cache, seqused_k, block_table, descales, int(max_seqlen_k))
    dev = k_cache.device
    query = _query(query, cache, dev)
    _on(cu_seqlens_q, "cu_seqlens_q", dev)
    _need(cu_seqlens_q.dtype is torch.int32 and cu_seqlens_q.shape == (cache.requests + 1,)
          and cu_seqlens_q.is_contiguous(), "cu_seqlens_q must be contiguous int32 (requests + 1,)")
    _need(max_seqlen_q >= 0, "max_seqlen_q must not be negative")
    _visibility(window, sinks)
    out = query.new_empty(query.shape)
    tokens, heads = query.shape[0], query.shape[1]
    if cache.requests == 0 or tokens == 0:
        return out
    qs, os = query.stride(), out.stride()
    need = _workspace_size("fm_paged_window_attn_workspace_size", dev.index, cache.requests, tokens, heads, cache.kv_heads,
                           cache.head_dim, int(max_seqlen_q), cache.max_length, window, sinks)
    ws = seqused_k.new_empty(need // 4) if need else None  # sizes are multiples of 8
    _launch("fm_paged_window_attn", cache,
            _WINDOW.pack(query.data_ptr(), qs[0], qs[1], tokens, heads, cu_seqlens_q.data_ptr(), int(max_seqlen_q),
                         softmax_scale, window, sinks, out.data_ptr(), os[0], os[1], ws.data_ptr() if need else 0, need,
                         _err_word(dev)))
    return out


def _launch4(name: str, cache: _Cache4, args: bytes) -> None:
    status = getattr(_lib.load(), name)(cache.packed, cache.scales, args,
                                        torch._C._cuda_getCurrentRawStream(cache.device.index))
    if status:
        _lib.check(status, name)


def _decode4(query, k_cache, v_cache, k_scales, v_scales, seqused_k, block_table, max_seqlen_k, softmax_scale, window,
             sinks, descales) -> torch.Tensor:
    cache = _cache4(k_cache, v_cache, k_scales, v_scales, seqused_k, block_table, descales, int(max_seqlen_k))
    dev = cache.device
    query = _query(query, cache, dev)
    shape = query.shape
    if shape[0] != cache.requests or window < 0 or sinks < 0:
        _need(shape[0] == cache.requests, "one query row per request")
        _visibility(window, sinks)
    out = query.new_empty(shape)
    if cache.requests == 0:
        return out
    heads, qs = shape[1], query.stride()
    need = _workspace_size("fm_paged_decode_attn_fp4_workspace_size", dev.index, cache.requests, heads, cache.kv_heads,
                           cache.head_dim, cache.max_length, window, sinks)
    ws = seqused_k.new_empty(need // 4) if need else None  # sizes are multiples of 8
    _launch4("fm_paged_decode_attn_fp4", cache,
             _DECODE.pack(query.data_ptr(), qs[0], qs[1], heads, softmax_scale, window, sinks, 0, 0, 0, out.data_ptr(),
                          heads * cache.head_dim, cache.head_dim, ws.data_ptr() if need else 0, need, _err_word(dev)))
    return out


def _window4(query, k_cache, v_cache, k_scales, v_scales, cu_seqlens_q, seqused_k, block_table, max_seqlen_q,
             max_seqlen_k, softmax_scale, window, sinks, descales) -> torch.Tensor:
    cache = _cache4(k_cache, v_cache, k_scales, v_scales, seqused_k, block_table, descales, int(max_seqlen_k))
    dev = cache.device
    query = _query(query, cache, dev)
    _on(cu_seqlens_q, "cu_seqlens_q", dev)
    _need(cu_seqlens_q.dtype is torch.int32 and cu_seqlens_q.shape == (cache.requests + 1,)
          and cu_seqlens_q.is_contiguous(), "cu_seqlens_q must be contiguous int32 (requests + 1,)")
    _need(max_seqlen_q >= 0, "max_seqlen_q must not be negative")
    _visibility(window, sinks)
    out = query.new_empty(query.shape)
    tokens, heads = query.shape[0], query.shape[1]
    if cache.requests == 0 or tokens == 0:
        return out
    qs, os = query.stride(), out.stride()
    need = _workspace_size("fm_paged_window_attn_workspace_size", dev.index, cache.requests, tokens, heads, cache.kv_heads,
                           cache.head_dim, int(max_seqlen_q), cache.max_length, window, sinks)
    ws = seqused_k.new_empty(need // 4) if need else None  # sizes are multiples of 8
    _launch4("fm_paged_window_attn_fp4", cache,
             _WINDOW.pack(query.data_ptr(), qs[0], qs[1], tokens, heads, cu_seqlens_q.data_ptr(), int(max_seqlen_q),
                          softmax_scale, window, sinks, out.data_ptr(), os[0], os[1], ws.data_ptr() if need else 0, need,
                          _err_word(dev)))
    return out


@torch.library.custom_op("flashmap_b200::paged_decode_attention", mutates_args=("weight_sums",))
def _decode_op(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, seqused_k: torch.Tensor,
               block_table: torch.Tensor, max_seqlen_k: int, softmax_scale: float, window: int, sinks: int,
               descales: Optional[torch.Tensor], weight_sums: Optional[torch.Tensor]) -> torch.Tensor:
    return _decode(query, k_cache, v_cache, seqused_k, block_table, max_seqlen_k, softmax_scale, window, sinks, descales,
                   weight_sums)


@_decode_op.register_fake
def _(query, k_cache, v_cache, seqused_k, block_table, max_seqlen_k, softmax_scale, window, sinks, descales, weight_sums):
    return query.new_empty(query.shape)


@torch.library.custom_op("flashmap_b200::paged_window_attention", mutates_args=())
def _window_op(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cu_seqlens_q: torch.Tensor,
               seqused_k: torch.Tensor, block_table: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int,
               softmax_scale: float, window: int, sinks: int, descales: Optional[torch.Tensor]) -> torch.Tensor:
    return _window(query, k_cache, v_cache, cu_seqlens_q, seqused_k, block_table, max_seqlen_q, max_seqlen_k,
                   softmax_scale, window, sinks, descales)


@_window_op.register_fake
def _(query, k_cache, v_cache, cu_seqlens_q, seqused_k, block_table, max_seqlen_q, max_seqlen_k, softmax_scale, window,
      sinks, descales):
    return query.new_empty(query.shape)


@torch.library.custom_op("flashmap_b200::paged_decode_attention_fp4", mutates_args=())
def _decode4_op(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scales: torch.Tensor,
                v_scales: torch.Tensor, seqused_k: torch.Tensor, block_table: torch.Tensor, max_seqlen_k: int,
                softmax_scale: float, window: int, sinks: int, descales: Optional[torch.Tensor]) -> torch.Tensor:
    return _decode4(query, k_cache, v_cache, k_scales, v_scales, seqused_k, block_table, max_seqlen_k, softmax_scale,
                    window, sinks, descales)


@_decode4_op.register_fake
def _(query, k_cache, v_cache, k_scales, v_scales, seqused_k, block_table, max_seqlen_k, softmax_scale, window, sinks,
      descales):
    return query.new_empty(query.shape)


@torch.library.custom_op("flashmap_b200::paged_window_attention_fp4", mutates_args=())
def _window4_op(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scales: torch.Tensor,
                v_scales: torch.Tensor, cu_seqlens_q: torch.Tensor, seqused_k: torch.Tensor, block_table: torch.Tensor,
                max_seqlen_q: int, max_seqlen_k: int, softmax_scale: float, window: int, sinks: int,
                descales: Optional[torch.Tensor]) -> torch.Tensor:
    return _window4(query, k_cache, v_cache, k_scales, v_scales, cu_seqlens_q, seqused_k, block_table, max_seqlen_q,
                    max_seqlen_k, softmax_scale, window, sinks, descales)


@_window4_op.register_fake
def _(query, k_cache, v_cache, k_scales, v_scales, cu_seqlens_q, seqused_k, block_table, max_seqlen_q, max_seqlen_k,
      softmax_scale, window, sinks, descales):
    return query.new_empty(query.shape)


# A call goes through its registered operator where it is traced, and where a
# gradient would be asked of it (which that operator refuses).  Else it goes
# straight to the kernels: the operator's dispatch costs as much host time as
# the rest of a short call.
_tracing = torch.compiler.is_compiling


def paged_decode_attention(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           seqused_k: torch.Tensor, block_table: torch.Tensor, max_seqlen_k: int,
                           softmax_scale: float, *, window: int = 0, sinks: int = 0,
                           descales: Optional[torch.Tensor] = None,
                           weight_sums: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per request, ``query (requests, heads,
    head_dim)`` bf16, at position ``seqused_k - 1`` of its context (its own key
    and value are in the cache already); ``(requests, heads, head_dim)`` bf16.

    It sees every position, or with ``window > 0`` the last ``window`` and the
    first ``sinks``.  ``weight_sums (requests, kv_heads, >= max_seqlen_k)`` fp32
    is added to in place: position j of a kv head gathers the attention weights
    of its query heads, which ``evict_paged_context`` goes by; no two of its rows
    may share memory.  A request has at most ``max_seqlen_k`` positions."""
    call = _decode
    if _tracing() or (query.requires_grad or k_cache.requires_grad or v_cache.requires_grad) and torch.is_grad_enabled():
        call = _decode_op
    return call(query, k_cache, v_cache, seqused_k, block_table, max_seqlen_k, softmax_scale, window, sinks, descales,
                weight_sums)


def paged_window_attention(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           cu_seqlens_q: torch.Tensor, seqused_k: torch.Tensor, block_table: torch.Tensor,
                           max_seqlen_q: int, max_seqlen_k: int, softmax_scale: float, *, window: int = 0,
                           sinks: int = 0, descales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of chunks of query rows: rows ``cu_seqlens_q[r] ..
    cu_seqlens_q[r + 1]`` of ``query (tokens, heads, head_dim)`` bf16 are the
    last positions of request r's ``seqused_k[r]`` (their own keys and values
    are in the cache already); ``(tokens, heads, head_dim)`` bf16.

    The row at position p sees the positions j <= p; with ``window > 0`` of
    those only p - j < ``window`` or j < ``sinks``.  A request has at most
    ``max_seqlen_q`` rows and ``max_seqlen_k`` positions.  Values that some rows
    of a chunk see and others do not must be finite.  Rows that ``cu_seqlens_q``
    gives to no request are not written."""
    call = _window
    if _tracing() or (query.requires_grad or k_cache.requires_grad or v_cache.requires_grad) and torch.is_grad_enabled():
        call = _window_op
    return call(query, k_cache, v_cache, cu_seqlens_q, seqused_k, block_table, max_seqlen_q, max_seqlen_k, softmax_scale,
                window, sinks, descales)


def paged_decode_attention_fp4(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                               k_scales: torch.Tensor, v_scales: torch.Tensor, seqused_k: torch.Tensor,
                               block_table: torch.Tensor, max_seqlen_k: int, softmax_scale: float, *, window: int = 0,
                               sinks: int = 0, descales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_decode_attention`` on a 4-bit cache: ``k_cache`` and ``v_cache (pages, kv_heads, page_size, head_dim / 2)``
    uint8 with ``k_scales`` and ``v_scales (pages, kv_heads, page_size, head_dim / 16)`` e4m3, as
    ``append_paged_context`` writes them; ``descales (2, requests, kv_heads)`` go on top.  It gathers no weights."""
    call = _decode4
    if _tracing() or query.requires_grad and torch.is_grad_enabled():
        call = _decode4_op
    return call(query, k_cache, v_cache, k_scales, v_scales, seqused_k, block_table, max_seqlen_k, softmax_scale, window,
                sinks, descales)


def paged_window_attention_fp4(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                               k_scales: torch.Tensor, v_scales: torch.Tensor, cu_seqlens_q: torch.Tensor,
                               seqused_k: torch.Tensor, block_table: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int,
                               softmax_scale: float, *, window: int = 0, sinks: int = 0,
                               descales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_window_attention`` on a 4-bit cache, given as to ``paged_decode_attention_fp4``."""
    call = _window4
    if _tracing() or query.requires_grad and torch.is_grad_enabled():
        call = _window4_op
    return call(query, k_cache, v_cache, k_scales, v_scales, cu_seqlens_q, seqused_k, block_table, max_seqlen_q,
                max_seqlen_k, softmax_scale, window, sinks, descales)


def evict_paged_context(k_cache: torch.Tensor, v_cache: torch.Tensor, seqused_k: torch.Tensor,
                        block_table: torch.Tensor, weight_sums: torch.Tensor, budget: int, *, sinks: int = 0,
                        recent: int = 0, out_block_table: Optional[torch.Tensor] = None
                        ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cuts every context to ``budget`` positions, for each kv head its own: the
    first ``sinks``, the last ``recent`` and, of those between, the ones with
    the largest ``weight_sums (requests, kv_heads, positions)`` (the lowest
    position among equal sums; a sum that is no number ranks last).  A context
    within the budget stays whole.

    The kept rows move, in order of position, to the request's first slots: in
    place (the pages after them are free then; no other request may share the
    pages), or with ``out_block_table (requests, pages)`` to its pages of the
    same pool, which must be none that ``block_table`` names (pages shared
    between requests keep their rows).
    Keys move as they are, rotated at their old positions.

    Returns ``kept (requests, kv_heads, budget)`` int32, the kept positions and
    then -1; the new lengths ``(requests,)`` int32; and the kept positions' sums
    ``(requests, kv_heads, budget)``, then 0, to go on gathering in."""
    _need(weight_sums.dim() == 3, "weight_sums must be float32 (requests, kv_heads, positions)")
    cache = _cache(k_cache, v_cache, seqused_k, block_table, None, weight_sums.shape[2])
    dev = k_cache.device
    _sums(weight_sums, cache, dev, 0)
    _need(budget >= 1, "the budget must be positive")
    _need(sinks >= 0 and recent >= 0 and sinks + recent <= budget, "sinks + recent must lie within the budget")
    kept = seqused_k.new_empty((cache.requests, cache.kv_heads, budget))
    lengths = seqused_k.new_empty(cache.requests)
    sums = weight_sums.new_empty((cache.requests, cache.kv_heads, budget))
    to, to_stride, to_cols = 0, 0, 0
    if out_block_table is not None:
        _on(out_block_table, "out_block_table", dev)
        _need(out_block_table.dtype is torch.int32 and out_block_table.dim() == 2
              and out_block_table.shape[0] == cache.requests, "out_block_table must be int32 (requests, pages)")
        _need(out_block_table.shape[1] <= 1 or out_block_table.stride(1) == 1, "out_block_table rows must be contiguous")
        _need(out_block_table.shape[1] * cache.page_size >= budget, "out_block_table does not cover the budget")
        to, to_stride, to_cols = out_block_table.data_ptr(), out_block_table.stride(0), out_block_table.shape[1]
    if cache.requests:
        need = _workspace_size("fm_paged_evict_workspace_size", dev.index, cache.requests, cache.kv_heads, budget)
        ws = seqused_k.new_empty(need // 4)
        _launch("fm_paged_evict", cache,
                _EVICT.pack(weight_sums.data_ptr(), weight_sums.stride(0), weight_sums.stride(1), budget, sinks, recent,
                            to, to_stride, to_cols, kept.data_ptr(), lengths.data_ptr(), sums.data_ptr(), ws.data_ptr(),
                            need, _err_word(dev)))
    return kept, lengths, sums


def _rows(x, name: str, shape, device):
    """``x`` of ``shape (tokens, heads, head_dim)``, bf16, and its token and head stride, with rows that the kernels can
    read 16 bytes at a time."""
    if not (x.shape == shape and x.dtype == torch.bfloat16 and x.device == device):
        _on(x, name, device)
        raise OpArgumentError(f"{name} must be bf16 {tuple(shape)}, got {x.dtype} {tuple(x.shape)}")
    s0, s1, s2 = x.stride()
    if s2 != 1 or s0 % 8 or s1 % 8 or x.data_ptr() % 16:
        x = x.contiguous()
        if x.data_ptr() % 16:  # a contiguous view that starts between two 16-byte lines
            x = x.clone()
        s0, s1, s2 = x.stride()
    return x, s0, s1


def append_paged_context(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         seqused_k: torch.Tensor, block_table: torch.Tensor, *,
                         cu_seqlens_q: Optional[torch.Tensor] = None, query: Optional[torch.Tensor] = None,
                         rope: Optional[torch.Tensor] = None, interleaved: bool = False,
                         positions: Optional[torch.Tensor] = None, k_scales: Optional[torch.Tensor] = None,
                         v_scales: Optional[torch.Tensor] = None,
                         descales: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes new tokens' ``key`` and ``value (tokens, kv_heads, head_dim)`` bf16 into the cache, in place: rows
    ``cu_seqlens_q[r] .. cu_seqlens_q[r + 1]`` become the last positions of request r's ``seqused_k[r]``, which
    counts them already; without ``cu_seqlens_q`` every request has one new token.

    ``rope (positions, rotary_dim / 2, 2)`` fp32, the cosines and sines of ``serving_ops.rope_table``, rotates keys
    and ``query (tokens, heads, head_dim)`` bf16 on the way: the pairs (i, i + rotary_dim / 2) of the first
    ``rotary_dim`` values (a multiple of 16), or (2 i, 2 i + 1) when ``interleaved``.  A token stands at
    ``positions (tokens,)`` int32 or int64, or where those are not given at its place in the cache (a context that was
    cut holds fewer positions than its text); rows that are not rotated stand nowhere else than in the cache.  Returns the rotated queries ``(tokens, heads, head_dim)``, or None.

    A bf16 cache takes the rotated values rounded; an e4m3 cache rounded and cut to +-448; a 4-bit cache (uint8, with
    ``k_scales`` and ``v_scales``) as e2m1 codes with one e4m3 factor for 16 values, their largest magnitude / 6.  The
    last two divide by ``descales`` first.

    A row without a place (a request of length 0, more rows than positions) writes nothing and its query comes back
    zero; so does, recorded for ``check_device_errors``, one whose request is longer than its table or whose position
    lies outside ``rope``.  A bad page id is recorded and not written to.  Rows that ``cu_seqlens_q`` gives to no request
    are not touched.  No two requests may append to the same page's slot."""
    table, pool = block_table.shape, k_cache.shape
    most = min(table[1] * pool[2], 0x7ffffff0) if len(table) == 2 and len(pool) == 4 else 0
    scales = None
    if k_cache.dtype == torch.uint8:
        cache = _cache4(k_cache, v_cache, k_scales, v_scales, seqused_k, block_table, descales, most)
        scales = cache.scales
    else:
        if k_scales is not None or v_scales is not None:
            raise OpArgumentError("k_scales and v_scales go with a 4-bit cache")
        cache = _cache(k_cache, v_cache, seqused_k, block_table, descales, most)
    dev, requests, kv_heads, head_dim = cache.device, cache.requests, cache.kv_heads, cache.head_dim
    if (key.requires_grad or value.requires_grad or query is not None and query.requires_grad) and torch.is_grad_enabled():
        raise OpArgumentError("append_paged_context has no gradient: detach the rows")
    tokens = key.shape[0] if key.dim() == 3 else -1
    shape = (tokens, kv_heads, head_dim)
    key, k0, k1 = _rows(key, "key", shape, dev)
    value, v0, v1 = _rows(value, "value", shape, dev)
    cu = 0
    if cu_seqlens_q is not None:
        _on(cu_seqlens_q, "cu_seqlens_q", dev)
        _need(cu_seqlens_q.dtype is torch.int32 and cu_seqlens_q.shape == (requests + 1,) and cu_seqlens_q.is_contiguous(),
              "cu_seqlens_q must be contiguous int32 (requests + 1,)")
        cu = cu_seqlens_q.data_ptr()
    elif tokens != requests:
        raise OpArgumentError("one new token per request without cu_seqlens_q")
    angles, rows, rotary = 0, 0, 0
    if rope is not None:
        turns = rope.shape
        if not (rope.device == dev and rope.dtype is torch.float32 and len(turns) == 3 and turns[2] == 2
                and rope.is_contiguous() and turns[1] >= 8 and turns[1] % 8 == 0 and 2 * turns[1] <= head_dim):
            _on(rope, "rope", dev)
            _need(rope.dtype is torch.float32 and rope.dim() == 3 and turns[2] == 2 and rope.is_contiguous(),
                  "rope must be contiguous float32 (positions, rotary_dim / 2, 2)")
            raise OpArgumentError(f"rotary_dim must be a multiple of 16 up to head_dim, got {2 * turns[1]}")
        angles, rows, rotary = rope.data_ptr(), turns[0], 2 * turns[1]
        if angles % 16:
            rope = rope.clone()
            angles = rope.data_ptr()
    at, at_dtype = 0, _lib.FM_DT_I32
    if positions is not None:
        _on(positions, "positions", dev)
        _need(positions.dtype in (torch.int32, torch.int64) and positions.shape == (tokens,)
              and positions.is_contiguous(), "positions must be contiguous int32 or int64 (tokens,)")
        at, at_dtype = positions.data_ptr(), _lib.FM_DT_I32 if positions.dtype == torch.int32 else _lib.FM_DT_I64
    out, q, q0, q1, heads, to, o0, o1 = None, 0, 0, 0, 0, 0, 0, 0
    if query is not None:
        heads = query.shape[1] if query.dim() == 3 else 0
        if rope is None or heads <= 0 or heads % kv_heads:
            _need(rope is not None, "queries are taken to be rotated: they go with a rope table")
            raise OpArgumentError(f"{heads} query heads are no multiple of {kv_heads} kv heads")
        query, q0, q1 = _rows(query, "query", (tokens, heads, head_dim), dev)
        out = query.new_empty((tokens, heads, head_dim))
        q, to, o0, o1 = query.data_ptr(), out.data_ptr(), heads * head_dim, head_dim
    if requests and tokens:
        status = _lib.load().fm_paged_append(
            cache.packed, scales,
            _APPEND.pack(key.data_ptr(), value.data_ptr(), k0, k1, v0, v1, q, q0, q1, heads, to, o0, o1, tokens, cu, at,
                         at_dtype, angles, rows, rotary, interleaved, _err_word(dev)),
            torch._C._cuda_getCurrentRawStream(dev.index))
        if status:
            _lib.check(status, "fm_paged_append")
    return out
