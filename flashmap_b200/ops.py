"""Torch-tensor wrappers of the C-ABI operators (CUDA tensors in, CUDA tensors out).

Each wrapper checks dtypes/contiguity like the reference's torch.library ops
(``assert``s in flashmap/vllm/kernels.py:51, 112) but raises ``ValueError``
instead, runs on the current CUDA stream, and returns new tensors.
"""

from __future__ import annotations

import ctypes
import functools
import math
import threading
from typing import NamedTuple

import torch

from . import _lib

STORE, GELU, SWIGLU, RESID, F32 = (_lib.FM_EPI_STORE, _lib.FM_EPI_GELU, _lib.FM_EPI_SWIGLU, _lib.FM_EPI_RESID,
                                   _lib.FM_EPI_F32)


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


_ERR_WORDS: dict = {}
_ERR_LOCK = threading.Lock()


class _Int32:
    """One int32 of device memory, as torch takes it over."""

    def __init__(self, address: int):
        self.__cuda_array_interface__ = {"shape": (1,), "typestr": "<i4", "data": (address, False), "version": 2}


def _new_error_word(device) -> torch.Tensor:
    if device.type != "cuda":
        return torch.zeros(1, dtype=torch.int32, device=device)
    at = ctypes.c_void_p()
    with torch.cuda.device(device):
        _lib.call("fm_error_word", ctypes.byref(at))
        return torch.as_tensor(_Int32(at.value))


def error_word(device) -> torch.Tensor:
    """The device's error word (int32, zero until a kernel records an index or
    timeout code; the first code sticks): the library's own memory, so that the
    first call may come from any thread and while a graph is captured, and no
    call launches a fill kernel for it."""
    key = torch.device(device)
    if key.index is None:
        key = torch.device(key.type, torch.cuda.current_device())
    w = _ERR_WORDS.get(key)
    if w is None:
        with _ERR_LOCK, torch.inference_mode(False):  # the word outlives the mode that it is first asked for in
            w = _ERR_WORDS.get(key)
            if w is None:
                w = _ERR_WORDS[key] = _new_error_word(key)
    return w


_ERR_ADDRESSES: dict = {}  # device index -> address of its error word, which lives as long as the process


def _error_address(device) -> int:
    at = _ERR_ADDRESSES.get(device.index)
    if at is None:
        at = _ERR_ADDRESSES[device.index] = error_word(device).data_ptr()
    return at


def _logits_dtype(t) -> int:
    if not t.is_cuda or not t.is_contiguous() or t.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"logits must be a contiguous CUDA bf16 or fp32 tensor, got {t.dtype} on {t.device}")
    return 0 if t.dtype == torch.bfloat16 else 1


def _need(t, dtype, name):
    if t is None:
        return
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA {dtype} tensor, got {t.dtype} on {t.device}")


def gemm(W: torch.Tensor, X: torch.Tensor, epilogue: int = STORE, bias=None, gate=None, out=None,
         err: torch.Tensor | None = None) -> torch.Tensor:
    """``out = epilogue(X @ W.T)`` on the tcgen05 GEMM (``fm_gemm_bf16``)."""
    _need(W, torch.bfloat16, "W")
    _need(X, torch.bfloat16, "X")
    _need(bias, torch.bfloat16, "bias")
    _need(gate, torch.bfloat16, "gate")
    M, K = W.shape
    N = X.shape[0]
    if X.shape[1] != K:
        raise ValueError(f"X has {X.shape[1]} columns, W has {K}")
    width = M // 2 if epilogue == SWIGLU else M
    if out is None:
        if epilogue == RESID:
            raise ValueError("the residual epilogue updates `out` in place")
        out = torch.empty(N, width, device=W.device, dtype=torch.float32 if epilogue == F32 else torch.bfloat16)
    ws_bytes = _lib.load().fm_gemm_workspace_size(M, N, K)
    ws = torch.zeros(ws_bytes, dtype=torch.uint8, device=W.device)
    _lib.call("fm_gemm_bf16", _p(W), _p(X), _p(out), M, N, K, out.shape[1], _p(bias), _p(gate), epilogue, _p(ws),
              ws_bytes, _p(err), _stream())
    return out


def rmsnorm(x, w, eps):
    _need(x, torch.bfloat16, "x")
    _need(w, torch.bfloat16, "w")
    y = torch.empty_like(x)
    cols = x.shape[-1]
    _lib.call("fm_rmsnorm", _p(x), _p(w), _p(y), x.numel() // cols, cols, float(eps), _stream())
    return y


def adaln(x, mod, eps):
    """``mod`` is the (scale | shift | gate) row of 3*D values."""
    _need(x, torch.bfloat16, "x")
    _need(mod, torch.bfloat16, "mod")
    y = torch.empty_like(x)
    cols = x.shape[-1]
    _lib.call("fm_adaln", _p(x), _p(mod), _p(y), x.numel() // cols, cols, float(eps), _stream())
    return y


def rope_inv_freq(head_dim: int, theta: float) -> torch.Tensor:
    """``1 / theta^(2i/hd)`` in fp32, the reference's expression (modeling_flashmap.py:56)
    evaluated on the host, so that every angle is bit-identical to the reference's."""
    return 1.0 / theta ** (torch.arange(0, head_dim, 2).float() / head_dim)


def rope_table(max_pos: int, head_dim: int, theta: float, device="cuda"):
    cs = torch.empty(max_pos, head_dim // 2, device=device, dtype=torch.float32)
    sn = torch.empty_like(cs)
    inv = rope_inv_freq(head_dim, theta).to(device)
    _lib.call("fm_rope_table", _p(cs), _p(sn), max_pos, head_dim, _p(inv), _stream())
    return cs, sn


def philox_normal(shape, seed: int, offset: int, device="cuda"):
    out = torch.empty(shape, device=device, dtype=torch.bfloat16)
    _lib.call("fm_philox_normal", _p(out), out.numel(), int(seed), int(offset), _stream())
    return out


def block_self_attn(qkv, batch: int, block: int, heads: int, head_dim: int):
    _need(qkv, torch.bfloat16, "qkv")
    out = torch.empty(batch * block, heads * head_dim, device=qkv.device, dtype=torch.bfloat16)
    _lib.call("fm_block_self_attn", _p(qkv), _p(out), batch, block, heads, head_dim, _stream())
    return out


def cross_attn(q, cache_kv, lengths, layer: int, nsplit: int = 0, err=None):
    """``cache_kv`` (L, 2, Bc, H, T, hd); ``lengths`` int32 (B,): keys 0..lengths[b]."""
    _need(q, torch.bfloat16, "q")
    _need(cache_kv, torch.bfloat16, "cache")
    _need(lengths, torch.int32, "lengths")
    L, _, Bc, H, Tc, hd = cache_kv.shape
    B = lengths.shape[0]
    if nsplit <= 0:
        nsplit = max(1, min((148 + B * H - 1) // (B * H), (Tc + 63) // 64))
    out = torch.empty(B * 16, H * hd, device=q.device, dtype=torch.bfloat16)
    wsb = _lib.load().fm_cross_attn_workspace_size(B, H, hd, nsplit)
    ws = torch.zeros(wsb, dtype=torch.uint8, device=q.device)
    _lib.call("fm_cross_attn", _p(q), _p(cache_kv), _p(out), _p(lengths), B, H, hd, L, layer, Bc, Tc, nsplit, _p(ws),
              wsb, _p(err), _stream())
    return out


def row_stats(logits, temperature: float):
    dt = _logits_dtype(logits)
    V = logits.shape[-1]
    rows = logits.numel() // V
    stats = torch.empty(rows, 2, device=logits.device, dtype=torch.float32)
    am = torch.empty(rows, device=logits.device, dtype=torch.int64)
    _lib.call("fm_row_stats", _p(logits), dt, rows, V, float(temperature), _p(stats), _p(am), _stream())
    return stats, am


def softmax_rows(logits, temperature: float):
    dt = _logits_dtype(logits)
    V = logits.shape[-1]
    probs = torch.empty(logits.shape, device=logits.device, dtype=torch.float32)
    _lib.call("fm_softmax_rows", _p(logits), dt, logits.numel() // V, V, float(temperature), _p(probs), _stream())
    return probs


def sample_rows(logits, probs, temperature: float, seed: int, offset: int):
    """Draft tokens (B, K) from logits (B, K, V): argmax at T <= 0, else drawn from probs."""
    B, K, V = logits.shape
    dt = _logits_dtype(logits)
    tokens = torch.empty(B, K, device=logits.device, dtype=torch.int64)
    _lib.call("fm_sample_rows", _p(logits), dt, _p(probs), B, K, V, float(temperature), int(seed), int(offset),
              _p(tokens), _stream())
    return tokens


def accept_greedy(target_logits, draft):
    dt = _logits_dtype(target_logits)
    _need(draft, torch.int64, "draft")
    B, K1, V = target_logits.shape
    acc = torch.empty(B, device=draft.device, dtype=torch.int64)
    bonus = torch.empty_like(acc)
    wsb = _lib.load().fm_accept_workspace_size(B, K1 - 1)
    ws = torch.empty(wsb, dtype=torch.uint8, device=draft.device)
    _lib.call("fm_accept_greedy", _p(target_logits), dt, _p(draft), B, K1 - 1, V, _p(acc), _p(bonus), _p(ws), wsb,
              _stream())
    return acc, bonus


def accept_rejection(target_logits, draft, q, temperature: float, seed: int, offset: int):
    dt = _logits_dtype(target_logits)
    _need(draft, torch.int64, "draft")
    _need(q, torch.float32, "q")
    B, K1, V = target_logits.shape
    acc = torch.empty(B, device=draft.device, dtype=torch.int64)
    bonus = torch.empty_like(acc)
    wsb = _lib.load().fm_accept_workspace_size(B, K1 - 1)
    ws = torch.empty(wsb, dtype=torch.uint8, device=draft.device)
    _lib.call("fm_accept_rejection", _p(target_logits), dt, _p(draft), _p(q), B, K1 - 1, V, float(temperature),
              int(seed), int(offset), _p(acc), _p(bonus), _p(ws), wsb, _stream())
    return acc, bonus


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` says of each row: fp32 ``logprobs`` and ``entropy`` (rows...), int64 ``top_ids`` and fp32
    ``top_logprobs`` (rows..., top_k)."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


@functools.lru_cache(maxsize=1024)
def _logprobs_workspace(device: int, rows: int, V: int, dtype: int, top_k: int) -> int:
    # the index of the current device is part of the key: the size goes by its number of SMs
    return _lib.load().fm_token_logprobs_workspace_size(rows, V, dtype, top_k)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0, temperature: float = 1.0) -> TokenLogprobs:
    """Log probabilities of ``tokens (...)`` int64 under ``softmax(logits / temperature)`` of ``logits (..., V)`` bf16 or
    fp32, the softmax's entropy (in nats) and the ``top_k`` (at most 32) likeliest ids with theirs, equal logits by the
    lowest id; in one pass over the logits and without writing probabilities (``fm_token_logprobs``).

    A row's values are contiguous, rows may lie further apart (a vocabulary padded in memory); more than one leading
    dimension is flattened, with a copy where its strides do not allow a view.  An id outside the vocabulary has
    log probability -inf and is recorded for ``cache_ops.check_device_errors``.  A row of -inf alone has -inf and entropy 0,
    one with a NaN or +inf NaN throughout; a finite logit's is finite where fp32 holds it (a mask of the type's lowest value:
    about -3.4e38 / temperature).  None is above 0, and no entropy below.  Runs on the current stream without a host
    synchronisation and can be captured in a CUDA graph; it is no registered operator, so ``torch.compile`` breaks a graph
    here, and there is no gradient."""
    if not logits.is_cuda or logits.dtype not in (torch.bfloat16, torch.float32) or logits.dim() < 1:
        raise ValueError(f"logits must be a CUDA bf16 or fp32 tensor, got {logits.dtype} on {logits.device}")
    dev, shape = logits.device, logits.shape[:-1]
    if dev.index != torch._C._cuda_getDevice():
        raise ValueError(f"the logits are on {dev}, which is not the current device")
    if tokens.device != dev or tokens.dtype != torch.int64 or tokens.shape != shape or not tokens.is_contiguous():
        raise ValueError(f"tokens must be contiguous int64 {tuple(shape)} on {dev}, "
                         f"got {tokens.dtype} {tuple(tokens.shape)} on {tokens.device}")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("token_logprobs has no gradient: detach the logits")
    V = logits.shape[-1]
    if not 0 <= top_k <= min(V, _lib.FM_TOKEN_LOGPROBS_MAX_TOP):
        raise ValueError(f"top_k must lie in 0 .. {min(V, _lib.FM_TOKEN_LOGPROBS_MAX_TOP)}, got {top_k}")
    if not 0.0 < temperature < math.inf:
        raise ValueError(f"the temperature must be positive, got {temperature}")
    if V > 1 and logits.stride()[-1] != 1:
        raise ValueError("a row of logits must be contiguous")
    if len(shape) != 1:
        logits = logits.reshape(-1, V)
    rows = logits.shape[0]
    f32 = torch.float32
    logprobs = logits.new_empty(shape, dtype=f32)
    entropy = torch.empty_like(logprobs)
    ids = tokens.new_empty(shape + (top_k,))
    top = logits.new_empty(shape + (top_k,), dtype=f32)
    if rows:
        dt = 0 if logits.dtype == torch.bfloat16 else 1
        need = _logprobs_workspace(dev.index, rows, V, dt, top_k)
        ws = tokens.new_empty(need // 8) if need else None  # sizes are multiples of 16
        status = _lib.load().fm_token_logprobs(
            logits.data_ptr(), dt, logits.stride()[0], tokens.data_ptr(), rows, V, temperature, top_k, logprobs.data_ptr(),
            entropy.data_ptr(), ids.data_ptr(), top.data_ptr(), ws.data_ptr() if need else None, need, _error_address(dev),
            torch._C._cuda_getCurrentRawStream(dev.index))
        if status:
            _lib.check(status, "fm_token_logprobs")
    return TokenLogprobs(logprobs, entropy, ids, top)


def transpose(x):
    _need(x, torch.bfloat16, "x")
    R, C = x.shape
    out = torch.empty(C, R, device=x.device, dtype=x.dtype)
    _lib.call("fm_transpose_bf16", _p(x), _p(out), R, C, _stream())
    return out


def time_freqs(dim: int) -> torch.Tensor:
    """``exp(-ln(10000) i / half)`` in fp32, the reference's expression (modeling_flashmap.py:94)."""
    half = dim // 2
    return torch.exp(-math.log(10000.0) * torch.arange(half).float() / half)


def time_sinusoid(dim: int, s: float, t: float, scale: float, device="cuda"):
    """Rows 0 and 1: sinusoidal features of ``s`` and ``t`` (bf16)."""
    out = torch.empty(2, dim, device=device, dtype=torch.bfloat16)
    freqs = time_freqs(dim).to(device)
    _lib.call("fm_time_sinusoid", _p(out), dim, float(s), float(t), float(scale), _p(freqs), _stream())
    return out


def silu(x):
    _need(x, torch.bfloat16, "x")
    y = torch.empty_like(x)
    _lib.call("fm_silu", _p(x), _p(y), x.numel(), _stream())
    return y


def add(a, b):
    _need(a, torch.bfloat16, "a")
    _need(b, torch.bfloat16, "b")
    y = torch.empty_like(a)
    _lib.call("fm_add", _p(a), _p(b), _p(y), a.numel(), _stream())
    return y


def attention_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)
