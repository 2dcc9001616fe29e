"""Python mirror of the paged-cache operators and the sampler (ie_paged_attention,
ie_qk_norm_rope_paged and ie_sample in include/infengine_b200.h).

A serving step over a paged cache: qk_norm_rope_paged puts the new tokens' keys
and values into their pages and returns the rotated queries, paged_attention
attends the cached rows, sample picks the next ids. The sequences of a call are
described by the same three device arrays throughout: q_start [B + 1] (the rows
each sequence owns), kv_len [B] (its cached rows, new ones included) and
page_table [B, max_pages], all int32.
"""
from __future__ import annotations

import ctypes

import torch

from . import IE_DTYPE_BF16, IE_DTYPE_F16, _check, lib

_DTYPES = {torch.float16: IE_DTYPE_F16, torch.bfloat16: IE_DTYPE_BF16}
_current_device = torch.cuda.current_device


class _Cache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("num_pages", ctypes.c_int),
                ("page_size", ctypes.c_int), ("n_kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64), ("row_stride", ctypes.c_int64)]


_calls = None


def _bind():
    """(paged_attention, qk_norm_rope_paged, sample, workspace bytes) of the library."""
    global _calls
    if _calls is None:
        L = lib()
        vp, i32, i64, f32, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
        L.ie_paged_attention_workspace_size.restype = sz
        L.ie_paged_attention_workspace_size.argtypes = []
        L.ie_paged_attention.argtypes = [i32, i32, i32, i32, i32, vp, i64, i64, vp, vp, i64, i32, vp, vp, i32, i32,
                                         f32, vp, i64, vp, sz, vp]
        L.ie_qk_norm_rope_paged.argtypes = [i32, i32, i32, i32, vp, i64, i64, vp, i64, i64, vp, i64, i64, vp, vp, f32,
                                            vp, vp, i32, vp, vp, i64, i32, vp, vp, vp, i64, i64, vp]
        L.ie_sample.argtypes = [i32, i32, i32, vp, i64, vp, vp, vp, vp, vp, vp, vp, vp]
        for name in ("ie_paged_attention", "ie_qk_norm_rope_paged", "ie_sample"):
            getattr(L, name).restype = i32
        _calls = (L.ie_paged_attention, L.ie_qk_norm_rope_paged, L.ie_sample,
                  int(L.ie_paged_attention_workspace_size()))
    return _calls


class PagedCache:
    """One layer's cache: k and v [num_pages, n_kv_heads, page_size, head_dim],
    fp16 or bf16, of the same shape and strides (a permuted view of a
    [num_pages, page_size, n_kv_heads, head_dim] pool will do). The tensors
    stay the caller's; the object keeps them alive."""

    def __init__(self, k, v):
        if not (k.is_cuda and v.is_cuda and k.device == v.device):
            raise ValueError("infengine_b200 operates on CUDA tensors of one device only")
        if k.dtype not in _DTYPES or v.dtype != k.dtype:
            raise TypeError(f"unsupported dtypes {k.dtype}, {v.dtype} (float16 or bfloat16, the same for both)")
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("k and v are [num_pages, n_kv_heads, page_size, head_dim] tensors of equal strides, "
                             "rows contiguous")
        self.k, self.v, self.dtype = k, v, k.dtype
        self.num_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.device_index = k.get_device()
        self.desc = _Cache(k.data_ptr(), v.data_ptr(), self.num_pages, self.page_size, self.n_kv_heads, self.head_dim,
                           k.stride(0), k.stride(1), k.stride(2))
        self._ref = ctypes.addressof(self.desc)


def _on_device(dev, *tensors):
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError("infengine_b200 operates on CUDA tensors of one device only")


def _ints(**tensors):
    for name, t in tensors.items():
        if t.dtype is not torch.int32 or t.stride(-1) != 1:
            raise TypeError(f"{name} must be an int32 tensor, contiguous along its last dimension")


def _raw_stream(dev, stream):
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(dev)
    return stream if isinstance(stream, int) else stream.cuda_stream


def _batch(cache, page_table, q_start, kv_len):
    """B, with the checks of a call's three int arrays."""
    _ints(page_table=page_table, q_start=q_start, kv_len=kv_len)
    B = kv_len.shape[0]
    if page_table.dim() != 2 or page_table.shape[0] != B or q_start.shape != (B + 1,) or kv_len.dim() != 1:
        raise ValueError("page_table [B, max_pages], q_start [B + 1] and kv_len [B] disagree about B")
    _on_device(cache.device_index, page_table, q_start, kv_len)
    return B


def paged_attention_workspace_bytes() -> int:
    """ie_paged_attention_workspace_size."""
    return _bind()[3]


def paged_attention_workspace(device="cuda"):
    """A workspace for paged_attention, its counters zeroed."""
    ws = torch.empty(paged_attention_workspace_bytes(), dtype=torch.uint8, device=device)
    ws[:65536].zero_()
    return ws


def paged_attention(q, cache, page_table, q_start, kv_len, out, max_q, window=0, sinks=0, scale=None, workspace=None,
                    stream=None):
    """ie_paged_attention: q [T, n_q_heads, head_dim] (rows of a head
    contiguous, any row and head strides), out [T, n_q_heads * head_dim].
    max_q: most new tokens of one sequence. scale: head_dim ** -0.5 by
    default. workspace: paged_attention_workspace(); one is allocated for the
    call when None, which a captured graph then owns."""
    dev = cache.device_index
    if dev != _current_device():
        with torch.cuda.device(dev):
            return paged_attention(q, cache, page_table, q_start, kv_len, out, max_q, window, sinks, scale, workspace,
                                   stream)
    B = _batch(cache, page_table, q_start, kv_len)
    if q.dtype is not cache.dtype or out.dtype is not cache.dtype:
        raise TypeError(f"q, out and the cache differ in dtype ({q.dtype}, {out.dtype}, {cache.dtype})")
    T, heads, dim = q.shape
    if dim != cache.head_dim or q.stride(2) != 1 or out.shape != (T, heads * dim) or out.stride(1) != 1:
        raise ValueError("q is [T, n_q_heads, head_dim] and out [T, n_q_heads * head_dim], rows contiguous")
    raw = _raw_stream(dev, stream)
    if workspace is None:
        workspace = paged_attention_workspace(q.device)
        if stream is not None and raw != torch._C._cuda_getCurrentRawStream(dev):
            workspace.record_stream(torch.cuda.ExternalStream(raw, device=dev))
    _on_device(dev, q, out, workspace)
    s = _bind()[0](_DTYPES[cache.dtype], B, T, max_q, heads, q.data_ptr(), q.stride(0), q.stride(1), cache._ref,
                   page_table.data_ptr(), page_table.stride(0), page_table.shape[1], q_start.data_ptr(),
                   kv_len.data_ptr(), window, sinks, dim ** -0.5 if scale is None else scale, out.data_ptr(),
                   out.stride(0), workspace.data_ptr(), workspace.numel() * workspace.element_size(), raw)
    if s:
        _check(s, "ie_paged_attention")


def qk_norm_rope_paged(q, k, v, q_weight, k_weight, rope_cos, rope_sin, cache, page_table, q_start, kv_len, q_out,
                       eps=1e-5, stream=None):
    """ie_qk_norm_rope_paged: q [T, n_q_heads, head_dim], k and v
    [T, n_kv_heads, head_dim] (views of one projection's output will do),
    weights [head_dim] or None, rope tables fp32 [rows, head_dim / 2] or None,
    q_out like q (q itself to work in place)."""
    dev = cache.device_index
    if dev != _current_device():
        with torch.cuda.device(dev):
            return qk_norm_rope_paged(q, k, v, q_weight, k_weight, rope_cos, rope_sin, cache, page_table, q_start,
                                      kv_len, q_out, eps, stream)
    B = _batch(cache, page_table, q_start, kv_len)
    T, heads, dim = q.shape
    want = (T, cache.n_kv_heads, cache.head_dim)
    if dim != cache.head_dim or k.shape != want or v.shape != want or q_out.shape != q.shape:
        raise ValueError("q and q_out are [T, n_q_heads, head_dim], k and v [T, n_kv_heads, head_dim]")
    for t in (q, k, v, q_out, q_weight, k_weight):
        if t is not None and (t.dtype is not cache.dtype or t.stride(-1) != 1):
            raise TypeError("q, k, v, q_out and the weights have the cache's dtype, rows contiguous")
    for t in (q_weight, k_weight):
        if t is not None and t.shape != (dim,):
            raise ValueError("a weight is [head_dim]")
    if (rope_cos is None) != (rope_sin is None):
        raise ValueError("rope_cos and rope_sin come together")
    for t in (rope_cos, rope_sin):
        if t is not None and (t.dtype is not torch.float32 or not t.is_contiguous() or t.dim() != 2 or
                              t.shape[1] != dim // 2 or t.shape != rope_cos.shape):
            raise ValueError("the rope tables are contiguous fp32 [rows, head_dim / 2]")
    _on_device(dev, q, k, v, q_out, q_weight, k_weight, rope_cos, rope_sin)
    s = _bind()[1](_DTYPES[cache.dtype], B, T, heads, q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(),
                   k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                   None if q_weight is None else q_weight.data_ptr(),
                   None if k_weight is None else k_weight.data_ptr(), eps,
                   None if rope_cos is None else rope_cos.data_ptr(),
                   None if rope_sin is None else rope_sin.data_ptr(), 0 if rope_cos is None else rope_cos.shape[0],
                   cache._ref, page_table.data_ptr(), page_table.stride(0), page_table.shape[1], q_start.data_ptr(),
                   kv_len.data_ptr(), q_out.data_ptr(), q_out.stride(0), q_out.stride(1), _raw_stream(dev, stream))
    if s:
        _check(s, "ie_qk_norm_rope_paged")


def sample(logits, u, idx_out, temperature=None, top_k=None, top_p=None, min_p=None, logprob_out=None, stream=None):
    """ie_sample: logits [M, V] (fp16 or bf16, any row stride), u [M] fp32 in
    [0, 1), idx_out [M] int32; temperature, top_p, min_p [M] fp32 and top_k [M]
    int32, or None; logprob_out [M] fp32 or None."""
    dev = logits.get_device()
    if dev < 0:
        raise ValueError("infengine_b200 operates on CUDA tensors of one device only")
    if dev != _current_device():
        with torch.cuda.device(dev):
            return sample(logits, u, idx_out, temperature, top_k, top_p, min_p, logprob_out, stream)
    if logits.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {logits.dtype} (float16 or bfloat16)")
    M, V = logits.shape
    if V > 1 and logits.stride(1) != 1:
        raise ValueError("a row of logits is contiguous")
    ptrs = []
    for t, kind in ((temperature, torch.float32), (top_k, torch.int32), (top_p, torch.float32),
                    (min_p, torch.float32), (u, torch.float32), (idx_out, torch.int32), (logprob_out, torch.float32)):
        if t is None:
            ptrs.append(None)
            continue
        if t.dtype is not kind or t.shape != (M,) or not t.is_contiguous():
            raise TypeError(f"a parameter, u or an output is not a contiguous [{M}] tensor of {kind}")
        if t.get_device() != dev:
            raise ValueError("infengine_b200 operates on CUDA tensors of one device only")
        ptrs.append(t.data_ptr())
    s = _bind()[2](_DTYPES[logits.dtype], M, V, logits.data_ptr(), logits.stride(0) if M > 1 else V, *ptrs,
                   _raw_stream(dev, stream))
    if s:
        _check(s, "ie_sample")
