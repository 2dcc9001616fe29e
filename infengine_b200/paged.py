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
            raise ValueError(_ONE_DEVICE)
        if k.dtype not in _DTYPES or v.dtype != k.dtype:
            raise TypeError(f"unsupported dtypes {k.dtype}, {v.dtype} (float16 or bfloat16, the same for both)")
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("k and v are [num_pages, n_kv_heads, page_size, head_dim] tensors of equal strides, "
                             "rows contiguous")
        self.k, self.v, self.dtype, self.code = k, v, k.dtype, _DTYPES[k.dtype]
        self.num_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.device_index = k.get_device()
        self.desc = _Cache(k.data_ptr(), v.data_ptr(), self.num_pages, self.page_size, self.n_kv_heads, self.head_dim,
                           k.stride(0), k.stride(1), k.stride(2))
        self._ref = ctypes.addressof(self.desc)


_ONE_DEVICE = "infengine_b200 operates on CUDA tensors of one device only"
_INTS = "page_table, q_start and kv_len are int32 tensors, contiguous along their last dimension"
_get_device = torch._C._cuda_getDevice
_get_stream = torch._C._cuda_getCurrentRawStream
_i32, _f32 = torch.int32, torch.float32


def _raw_stream(dev, stream):
    if stream is None:
        return _get_stream(dev)
    return stream if isinstance(stream, int) else stream.cuda_stream


def _batch(dev, page_table, q_start, kv_len):
    """(B, row stride of the table, its width), with the checks of a call's three int arrays."""
    if page_table.dtype is not _i32 or q_start.dtype is not _i32 or kv_len.dtype is not _i32:
        raise TypeError(_INTS)
    B, wide = page_table.shape
    ld, one = page_table.stride()
    if q_start.shape != (B + 1,) or kv_len.shape != (B,):
        raise ValueError("page_table [B, max_pages], q_start [B + 1] and kv_len [B] disagree about B")
    if (one != 1 and wide > 1) or not (q_start.is_contiguous() and kv_len.is_contiguous()):
        raise TypeError(_INTS)
    if not page_table.get_device() == q_start.get_device() == kv_len.get_device() == dev:
        raise ValueError(_ONE_DEVICE)
    return B, ld if B > 1 else wide, wide


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
    dev, dt = cache.device_index, cache.dtype
    if dev != _get_device():
        with torch.cuda.device(dev):
            return paged_attention(q, cache, page_table, q_start, kv_len, out, max_q, window, sinks, scale, workspace,
                                   stream)
    B, ld_table, wide = _batch(dev, page_table, q_start, kv_len)
    if q.dtype is not dt or out.dtype is not dt:
        raise TypeError(f"q, out and the cache differ in dtype ({q.dtype}, {out.dtype}, {dt})")
    T, heads, dim = q.shape
    ldq, hs, one = q.stride()
    ldo, one_o = out.stride()
    if dim != cache.head_dim or one != 1 or out.shape != (T, heads * dim) or one_o != 1:
        raise ValueError("q is [T, n_q_heads, head_dim] and out [T, n_q_heads * head_dim], rows contiguous")
    raw = _raw_stream(dev, stream)
    if workspace is None:
        workspace = paged_attention_workspace(q.device)
        if stream is not None and raw != _get_stream(dev):
            other = torch.cuda.ExternalStream(raw, device=dev)
            other.wait_stream(torch.cuda.current_stream(dev))
            workspace.record_stream(other)
    if not q.get_device() == out.get_device() == workspace.get_device() == dev:
        raise ValueError(_ONE_DEVICE)
    if not workspace.is_contiguous():
        raise ValueError("workspace is not contiguous")
    s = (_calls or _bind())[0](
        cache.code, B, T, max_q, heads, q.data_ptr(), ldq, hs, cache._ref, page_table.data_ptr(), ld_table, wide,
        q_start.data_ptr(), kv_len.data_ptr(), window, sinks, dim ** -0.5 if scale is None else scale, out.data_ptr(),
        ldo if T > 1 else heads * dim, workspace.data_ptr(), workspace.nbytes, raw)
    if s:
        _check(s, "ie_paged_attention")


def qk_norm_rope_paged(q, k, v, q_weight, k_weight, rope_cos, rope_sin, cache, page_table, q_start, kv_len, q_out,
                       eps=1e-5, stream=None):
    """ie_qk_norm_rope_paged: q [T, n_q_heads, head_dim], k and v
    [T, n_kv_heads, head_dim] (views of one projection's output will do),
    weights [head_dim] or None, rope tables fp32 [rows, head_dim / 2] or None,
    q_out like q (q itself to work in place)."""
    dev, dt = cache.device_index, cache.dtype
    if dev != _get_device():
        with torch.cuda.device(dev):
            return qk_norm_rope_paged(q, k, v, q_weight, k_weight, rope_cos, rope_sin, cache, page_table, q_start,
                                      kv_len, q_out, eps, stream)
    B, ld_table, wide = _batch(dev, page_table, q_start, kv_len)
    shape = q.shape
    T, heads, dim = shape
    kv_shape = k.shape
    if (dim != cache.head_dim or q_out.shape != shape or v.shape != kv_shape or
            kv_shape != (T, cache.n_kv_heads, dim)):
        raise ValueError("q and q_out are [T, n_q_heads, head_dim], k and v [T, n_kv_heads, head_dim]")
    (lq, hq, q1), (lk, hk, k1), (lv, hv, v1), (lo, ho, o1) = q.stride(), k.stride(), v.stride(), q_out.stride()
    if not (q.dtype is dt and k.dtype is dt and v.dtype is dt and q_out.dtype is dt) or q1 * k1 * v1 * o1 != 1:
        raise TypeError("q, k, v and q_out have the cache's dtype, rows contiguous")
    if not q.get_device() == k.get_device() == v.get_device() == q_out.get_device() == dev:
        raise ValueError(_ONE_DEVICE)
    wq = wk = cos = sin = None
    rows = 0
    if q_weight is not None:
        wq = _weight(q_weight, dt, dim, dev)
    if k_weight is not None:
        wk = _weight(k_weight, dt, dim, dev)
    if rope_cos is not None or rope_sin is not None:
        if rope_cos is None or rope_sin is None:
            raise ValueError("rope_cos and rope_sin come together")
        rows = rope_cos.shape[0]
        if (rope_cos.dtype is not _f32 or rope_sin.dtype is not _f32 or rope_cos.shape != (rows, dim // 2) or
                rope_sin.shape != (rows, dim // 2) or not (rope_cos.is_contiguous() and rope_sin.is_contiguous())):
            raise ValueError("the rope tables are contiguous fp32 [rows, head_dim / 2]")
        if not rope_cos.get_device() == rope_sin.get_device() == dev:
            raise ValueError(_ONE_DEVICE)
        cos, sin = rope_cos.data_ptr(), rope_sin.data_ptr()
    s = (_calls or _bind())[1](
        cache.code, B, T, heads, q.data_ptr(), lq, hq, k.data_ptr(), lk, hk, v.data_ptr(), lv, hv, wq, wk, eps, cos,
        sin, rows, cache._ref, page_table.data_ptr(), ld_table, wide, q_start.data_ptr(), kv_len.data_ptr(),
        q_out.data_ptr(), lo, ho, _raw_stream(dev, stream))
    if s:
        _check(s, "ie_qk_norm_rope_paged")


def _weight(w, dt, dim, dev):
    if w.dtype is not dt or w.shape != (dim,) or not w.is_contiguous():
        raise TypeError("a weight is a contiguous [head_dim] tensor of the cache's dtype")
    if w.get_device() != dev:
        raise ValueError(_ONE_DEVICE)
    return w.data_ptr()


def sample(logits, u, idx_out, temperature=None, top_k=None, top_p=None, min_p=None, logprob_out=None, stream=None):
    """ie_sample: logits [M, V] (fp16 or bf16, any row stride), u [M] fp32 in
    [0, 1), idx_out [M] int32; temperature, top_p, min_p [M] fp32 and top_k [M]
    int32, or None; logprob_out [M] fp32 or None."""
    dev = logits.get_device()
    if dev < 0:
        raise ValueError(_ONE_DEVICE)
    if dev != _get_device():
        with torch.cuda.device(dev):
            return sample(logits, u, idx_out, temperature, top_k, top_p, min_p, logprob_out, stream)
    if logits.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {logits.dtype} (float16 or bfloat16)")
    M, V = logits.shape
    if V > 1 and logits.stride(1) != 1:
        raise ValueError("a row of logits is contiguous")
    def ptr(t, kind):
        if t is None:
            return None
        if t.dtype is not kind or t.shape != (M,) or not t.is_contiguous():
            raise TypeError(f"a parameter, u or an output is not a contiguous [{M}] tensor of {kind}")
        if t.get_device() != dev:
            raise ValueError(_ONE_DEVICE)
        return t.data_ptr()

    s = (_calls or _bind())[2](
        _DTYPES[logits.dtype], M, V, logits.data_ptr(), logits.stride(0) if M > 1 else V, ptr(temperature, _f32),
        ptr(top_k, _i32), ptr(top_p, _f32), ptr(min_p, _f32), ptr(u, _f32), ptr(idx_out, _i32),
        ptr(logprob_out, _f32), _raw_stream(dev, stream))
    if s:
        _check(s, "ie_sample")
