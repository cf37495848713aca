"""The kernel facade and the token-by-token serving operators
(include/esm_b200.h, sections 1 and 3) over torch CUDA tensors.

Each function mirrors one esm::kernels function of the reference
(include/esm_cpp/kernels.h) with device tensors instead of host pointers.
PyTorch provides device memory and the stream; every computation runs in
libesm_b200.so.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import threading

import numpy as np

from . import _lib

_ctx = {}


def context(device: int = 0):
    """A per-device esmcu_context bound to torch's current stream (so the ops
    are stream-ordered with the torch work around them)."""
    if device not in _ctx:
        h = C.c_void_p()
        _lib.call("esmcu_open", device, C.byref(h))
        _ctx[device] = h
    h = _ctx[device]
    _lib.call("esmcu_set_stream", h, _lib.torch_stream_handle(device))
    return h


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _dev(t):
    return t.device.index or 0


def set_math_mode(mode: str, device: int = 0) -> None:
    """esmcu_set_math_mode on the facade's context of `device`: "default"
    (tensor-core / fused kernels) or "avx512" (LayerNorm, GELU and attention
    reproduce the reference's default x86 kernels bit for bit)."""
    _lib.call("esmcu_set_math_mode", context(device), _lib.MATH_MODES[mode])


def synchronize(device: int = 0):
    _lib.call("esmcu_synchronize", context(device))
    if device in _serving_ctx:
        with _serving(device) as ctx:
            _lib.call("esmcu_synchronize", ctx)


def linear(A, W, bias=None):
    """kernels::Linear: A [M,K] f32, W [N,K] f32 -> [M,N]."""
    import torch

    M, K = A.shape
    N = W.shape[0]
    out = torch.empty((M, N), dtype=torch.float32, device=A.device)
    _lib.call("esmcu_linear", context(_dev(A)), _p(A), _p(W), _p(bias), _p(out), M, N, K)
    return out


def linear_int8(A, Wq, w_scales, bias=None, act_quant: int = _lib.ACT_PER_TENSOR):
    """kernels::LinearInt8 (W8A8): A [M,K] f32, Wq [N,K] int8, w_scales [N]."""
    import torch

    M, K = A.shape
    N = Wq.shape[0]
    out = torch.empty((M, N), dtype=torch.float32, device=A.device)
    _lib.call("esmcu_linear_int8", context(_dev(A)), _p(A), _p(Wq), _p(w_scales), _p(bias),
              _p(out), M, N, K, act_quant)
    return out


def quantize_activations(A, act_quant: int = _lib.ACT_PER_TENSOR):
    """-> (q int8 [M, ldq], scales f32 [1] or [M]); ldq = K rounded up to 16."""
    import torch

    M, K = A.shape
    ldq = (K + 15) // 16 * 16
    q = torch.empty((M, ldq), dtype=torch.int8, device=A.device)
    s = torch.empty((M if act_quant == _lib.ACT_PER_TOKEN else 1,), dtype=torch.float32, device=A.device)
    _lib.call("esmcu_quantize_activations", context(_dev(A)), _p(A), M, K, _p(q), ldq, _p(s), act_quant)
    return q, s


def quantize_weights(W):
    """quant::Quantize on the device: W [N, K] float32 -> (q int8 [N, K],
    scales float32 [N]), bit-identical to prep.quantize_weight."""
    import torch

    W = W.contiguous()
    N, K = W.shape
    q = torch.empty((N, K), dtype=torch.int8, device=W.device)
    s = torch.empty((N,), dtype=torch.float32, device=W.device)
    _lib.call("esmcu_quantize_weights", context(_dev(W)), _p(W), N, K, _p(q), _p(s))
    return q, s


def gemm_int8_s32(q, Wq):
    """int32 acc [M,N] = q [M,K] . Wq [N,K]^T on the tensor cores."""
    import torch

    M, K = q.shape
    N = Wq.shape[0]
    acc = torch.empty((M, N), dtype=torch.int32, device=q.device)
    _lib.call("esmcu_gemm_int8_s32", context(_dev(q)), _p(q), q.stride(0), _p(Wq), Wq.stride(0),
              _p(acc), M, N, K)
    return acc


def layernorm(x, gamma, beta, eps: float = 1e-5):
    import torch

    rows, d = x.shape
    out = torch.empty_like(x)
    _lib.call("esmcu_layernorm", context(_dev(x)), _p(x), _p(gamma), _p(beta), float(eps), _p(out), rows, d)
    return out


def gelu(x):
    import torch

    out = torch.empty_like(x)
    _lib.call("esmcu_gelu", context(_dev(x)), _p(x), _p(out), x.numel())
    return out


def residual_add_inplace(y, x):
    _lib.call("esmcu_residual_add_inplace", context(_dev(y)), _p(y), _p(x), y.numel())
    return y


def scale_inplace(x, s: float):
    _lib.call("esmcu_scale_inplace", context(_dev(x)), _p(x), x.numel(), float(s))
    return x


def rope_build_tables(seq_len: int, head_dim: int):
    """kernels::RopeBuildTables on the host -> (cos, sin) numpy [L, dh]."""
    c = np.zeros((seq_len, head_dim), np.float32)
    s = np.zeros((seq_len, head_dim), np.float32)
    _lib.call("esmcu_rope_build_tables", seq_len, head_dim, c.ctypes.data, s.ctypes.data)
    return c, s


def rope_apply_varlen(x, cos_t, sin_t, cu_seqlens, num_heads: int, head_dim: int):
    B = cu_seqlens.numel() - 1
    _lib.call("esmcu_rope_apply_varlen", context(_dev(x)), _p(x), _p(cos_t), _p(sin_t),
              _p(cu_seqlens), B, num_heads, head_dim)
    return x


def attention_varlen(q, k, v, cu_seqlens, num_heads: int, head_dim: int):
    import torch

    out = torch.empty_like(q)
    B = cu_seqlens.numel() - 1
    _lib.call("esmcu_attention_varlen", context(_dev(q)), _p(q), _p(k), _p(v), _p(cu_seqlens), B,
              num_heads, head_dim, _p(out))
    return out


# ------------------------------------------------- token-by-token serving
# The serving operators share one context per device, apart from the facade's,
# and bind the caller's stream and enqueue under a lock: threads on streams of
# their own can call them at once.
_serving_ctx = {}
_serving_lock = threading.Lock()


@contextlib.contextmanager
def _serving(device: int):
    import torch

    with torch.cuda.device(device), _serving_lock:
        if device not in _serving_ctx:
            h = C.c_void_p()
            _lib.call("esmcu_open", device, C.byref(h))
            _serving_ctx[device] = h
        h = _serving_ctx[device]
        _lib.call("esmcu_set_stream", h, _lib.torch_stream_handle(device))
        yield h


def _dtype(t, name: str) -> int:
    import torch

    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    return code


def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _on(device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def _rows(t, name: str, dtype=None) -> None:
    """t has contiguous last-dimension elements, of `dtype` where given."""
    _need(dtype is None or t.dtype == dtype, f"{name} must be {dtype}, not {t.dtype}")
    _need(t.shape[-1] <= 1 or t.stride(-1) == 1, f"{name}: the last dimension must be contiguous")


def linear_w4(x, wq, scales, zeros=None, bias=None, group_size: int = 128):
    """A Linear with 4-bit weights and group scales, for few rows:
    out[m, n] = sum_k x[m, k] * (q[n, k] - z[n, k // group_size])
    * scales[n, k // group_size] + bias[n], of x's type.

    x [M, K] float32, float16 or bfloat16; wq uint8 [N, ceil(K / 2)], column 2j
    in the low four bits of byte j; scales [N, ceil(K / group_size)] of any of
    the three types; zeros uint8 of the same shape with values 0 to 15 (None: 8
    everywhere); bias float32 [N]; group_size 32, 64 or 128
    (prep.quantize_weight_w4 makes wq and scales).  Sums are float32, rounded
    once.  Rows of wq that start on 16-byte boundaries are read fastest."""
    import torch

    _need(x.dim() == 2 and wq.dim() == 2 and scales.dim() == 2, "x, wq and scales must be matrices")
    _need(x.is_cuda, "x must be a CUDA tensor")
    M, K = x.shape
    N = wq.shape[0]
    _need(group_size in (32, 64, 128), "group_size must be 32, 64 or 128")
    _need(wq.shape[1] == (K + 1) // 2, f"wq must be [N, {(K + 1) // 2}] for K = {K}")
    groups = -(-K // group_size)
    _need(tuple(scales.shape) == (N, groups), f"scales must be [{N}, {groups}]")
    _rows(x, "x")
    _rows(wq, "wq", torch.uint8)
    _rows(scales, "scales")
    if zeros is not None:
        _need(zeros.shape == scales.shape, "zeros must have the shape of scales")
        _rows(zeros, "zeros", torch.uint8)
    if bias is not None:
        _need(tuple(bias.shape) == (N,), f"bias must be [{N}]")
        _rows(bias, "bias", torch.float32)
    _on(x.device, wq=wq, scales=scales, zeros=zeros, bias=bias)
    code = _dtype(x, "x")
    out = torch.empty((M, N), dtype=x.dtype, device=x.device)
    with _serving(_dev(x)) as ctx:
        _lib.call("esmcu_linear_w4", ctx, _p(x), _stride(x, 0), code, _p(wq), _stride(wq, 0),
                  _p(scales), _dtype(scales, "scales"), _stride(scales, 0), _p(zeros),
                  0 if zeros is None else _stride(zeros, 0), group_size, _p(bias), _p(out), N, M, N, K)
    return out


def _stride(t, dim: int) -> int:
    """The stride of a dimension; of one with a single entry, which torch may
    give any stride, the dense one."""
    if t.shape[dim] > 1:
        return t.stride(dim)
    n = 1
    for size in t.shape[dim + 1:]:
        n *= size
    return n


def _paged(k_cache, v_cache, page_table):
    import torch

    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape,
          "k_cache and v_cache must be [pages, page_size, kv_heads, head_dim], of one shape")
    _need(k_cache.is_cuda, "k_cache must be a CUDA tensor")
    _need(page_table.dim() == 2, "page_table must be [sequences, max_pages]")
    _rows(k_cache, "k_cache")
    _rows(v_cache, "v_cache", k_cache.dtype)
    _rows(page_table, "page_table", torch.int32)
    _on(k_cache.device, v_cache=v_cache, page_table=page_table)
    pages, page_size, heads, dh = k_cache.shape
    return _lib.PagedKV(
        k_cache.data_ptr(), v_cache.data_ptr(), _dtype(k_cache, "k_cache"), pages, page_size, heads, dh,
        _stride(k_cache, 0), _stride(k_cache, 1), _stride(k_cache, 2),
        _stride(v_cache, 0), _stride(v_cache, 1), _stride(v_cache, 2),
        page_table.data_ptr(), _stride(page_table, 0), page_table.shape[1])


def kv_append_paged(k, v, k_cache, v_cache, page_table, cu_seqlens, cache_lens, q=None, cos=None,
                    sin=None):
    """Appends packed new tokens to a paged K/V cache, RoPE applied on the way;
    returns the rotated queries (None without q).

    k, v [T, kv_heads, dh] and q [T, q_heads, dh] in the cache's type, or
    float32 to be rounded to it (views into a joint qkv row are fine); k_cache
    and v_cache [pages, page_size, kv_heads, dh], any strides with contiguous
    heads' elements, written in place; page_table int32 [B, max_pages];
    cu_seqlens int32 [B + 1]; cache_lens int32 [B], the tokens already cached
    (not advanced).  Token t of sequence b goes to position
    cache_lens[b] + t - cu_seqlens[b].  cos and sin float32 [positions, rot]
    rotate the first rot (<= dh) elements of every q and k head by the row of
    the token's position, as rope_build_tables lays them out; None: no
    rotation.  Rows behind cu_seqlens[B] are left out (their q rows hold
    nothing).  A position or page id outside the cache or the tables is
    skipped and reported by synchronize()."""
    import torch

    cache = _paged(k_cache, v_cache, page_table)
    dev = k_cache.device
    _need(k.dim() == 3 and k.shape == v.shape and tuple(k.shape[1:]) == tuple(k_cache.shape[2:]),
          "k and v must be [T, kv_heads, head_dim] with the cache's heads")
    _need(k.dtype in (k_cache.dtype, torch.float32), "k must have the cache's type or be float32")
    _need(v.dtype == k.dtype, "v must have k's type")
    B = cache_lens.numel()
    _need(cache_lens.dim() == 1 and cu_seqlens.dim() == 1 and cu_seqlens.numel() == B + 1,
          "cu_seqlens must be [B + 1] for cache_lens [B]")
    _need(page_table.shape[0] >= B, "page_table has fewer rows than cache_lens")
    _rows(k, "k")
    _rows(v, "v")
    _rows(cu_seqlens, "cu_seqlens", torch.int32)
    _rows(cache_lens, "cache_lens", torch.int32)
    T, _, dh = k.shape
    out, heads = None, 0
    if q is not None:
        _need(q.dim() == 3 and q.shape[0] == T and q.shape[2] == dh and q.dtype == k.dtype,
              "q must be [T, q_heads, head_dim] of k's type")
        _rows(q, "q")
        heads = q.shape[1]
        out = torch.empty((T, heads, dh), dtype=k_cache.dtype, device=dev)
    rot = rows = 0
    _need((cos is None) == (sin is None), "cos and sin go together")
    if cos is not None:
        _need(cos.dim() == 2 and cos.shape == sin.shape, "cos and sin must be [positions, rot]")
        _need(cos.is_contiguous() and sin.is_contiguous(), "cos and sin must be contiguous")
        _rows(cos, "cos", torch.float32)
        _rows(sin, "sin", torch.float32)
        rows, rot = cos.shape
    _on(dev, k=k, v=v, q=q, cos=cos, sin=sin, cu_seqlens=cu_seqlens, cache_lens=cache_lens)
    with _serving(_dev(k_cache)) as ctx:
        _lib.call("esmcu_kv_append_paged", ctx, C.byref(cache), _p(q) if heads else None,
                  _stride(q, 0) if heads else 0, _stride(q, 1) if heads else 0, heads, _p(k),
                  _stride(k, 0), _stride(k, 1), _p(v), _stride(v, 0), _stride(v, 1), _dtype(k, "k"),
                  _p(cos), _p(sin), rows, rot, _p(cu_seqlens), _p(cache_lens), B, T,
                  _p(out) if heads else None)
    return out


def attention_decode_paged(q, k_cache, v_cache, page_table, seq_lens, scale: float = 1.0,
                           window: int = 0, return_lse: bool = False):
    """Attention of one new token per sequence over a paged K/V cache:
    out[b, h] = sum_t softmax_t(scale * q[b, h] . k[t, h']) v[t, h'] over the
    seq_lens[b] cached keys (the last `window` of them when window > 0),
    h' = h // (q_heads // kv_heads).

    q [B, q_heads, dh] of the cache's type (pre-scaled for scale = 1, as for
    attention_varlen); caches and page_table as for kv_append_paged, dh a
    multiple of 8 up to 256 and rows on 16-byte boundaries; seq_lens int32 [B],
    on the device, the new token's own key included.  Returns out [B, q_heads,
    dh], and with return_lse also float32 log(sum_t exp(scale * q . k))
    [B, q_heads].  A sequence of length 0 gives zeros and -inf.  A length or
    page id outside the cache is skipped and reported by synchronize()."""
    import torch

    cache = _paged(k_cache, v_cache, page_table)
    dev = k_cache.device
    _need(q.dim() == 3 and q.shape[2] == k_cache.shape[3], "q must be [B, q_heads, head_dim]")
    _rows(q, "q", k_cache.dtype)
    B, heads, dh = q.shape
    _need(tuple(seq_lens.shape) == (B,), f"seq_lens must be [{B}]")
    _rows(seq_lens, "seq_lens", torch.int32)
    _need(page_table.shape[0] >= B, "page_table has fewer rows than q")
    _on(dev, q=q, seq_lens=seq_lens)
    out = torch.empty((B, heads, dh), dtype=q.dtype, device=dev)
    lse = torch.empty((B, heads), dtype=torch.float32, device=dev) if return_lse else None
    with _serving(_dev(k_cache)) as ctx:
        n = C.c_size_t()
        _lib.call("esmcu_attention_decode_paged_workspace", ctx, C.byref(cache), heads, C.byref(n))
        work = torch.empty((n.value,), dtype=torch.uint8, device=dev)
        _lib.call("esmcu_attention_decode_paged", ctx, C.byref(cache), _p(q), _stride(q, 0),
                  _stride(q, 1), heads, _p(seq_lens), B, float(scale), int(window), _p(out), _p(lse),
                  _p(work), n.value)
    return (out, lse) if return_lse else out


def plan_batches(lengths, imbalance_threshold: float = 1.2, max_batch_size: int = 256):
    """PlanBatches on the host -> list of index groups."""
    lens = np.ascontiguousarray(lengths, np.int32)
    n = lens.shape[0]
    order = np.zeros(max(n, 1), np.int32)
    sizes = np.zeros(max(n, 1), np.int32)
    g = _lib.lib().esmcu_plan_batches(lens.ctypes.data, n, float(imbalance_threshold),
                                      int(max_batch_size), order.ctypes.data, sizes.ctypes.data)
    if g < 0:
        _lib.check(1, "esmcu_plan_batches")
    out, pos = [], 0
    for i in range(g):
        out.append(order[pos:pos + sizes[i]].tolist())
        pos += sizes[i]
    return out


def batch_view_check(T: int, n_masks: int, cu_seqlens, batch_size: int) -> None:
    cu = np.ascontiguousarray(cu_seqlens, np.int32)
    _lib.call("esmcu_batch_view_check", T, n_masks, cu.ctypes.data, cu.shape[0], batch_size)
