"""The token-by-token serving operators (include/esm_b200.h, section 3) over
torch CUDA tensors, reached as ops.linear_w4, ops.kv_append_paged and
ops.attention_decode_paged: a 4-bit Linear for few rows, the append to a paged
K/V cache with RoPE on the way, and the attention of one new token over it.

A decoding step makes many of these calls, each a few microseconds of device
time, so the wrappers keep their own host time low: one pass over the shapes
and strides, the argument blocks of the C ABI packed with one struct call each,
the stream bound only when it changes, a workspace per stream.
"""
from __future__ import annotations

import ctypes as C
import struct
import threading

import torch

from . import _lib

_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # esmcu_dtype
_I32, _U8, _F32 = torch.int32, torch.uint8, torch.float32


# The raw handle of torch's current stream, and the current device; the public
# ways (a Stream object per call) take a microsecond more.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_workspace_bytes: dict[tuple, int] = {}  # functions of the shapes alone
_w4_workspace_bytes: dict[tuple, int] = {}

# One esmcu_context per device, apart from the facade's, and the stream that it
# is bound to.  Calls bind the caller's stream and enqueue under the lock:
# threads on streams of their own can call at once.
_lock = threading.Lock()
_contexts: dict[int, list] = {}  # device -> [handle, stream]


def _open(device: int) -> list:
    """The device's context (lock held, the device current)."""
    h = C.c_void_p()
    _lib.call("esmcu_open", device, C.byref(h))
    ctx = _contexts[device] = [h, None]
    return ctx


def _enqueue(device: int, f, *args) -> None:
    """f(context, *args) on torch's current stream of `device`."""
    if _current_device() != device:
        with torch.cuda.device(device):
            return _enqueue(device, f, *args)
    stream = _raw_stream(device)
    with _lock:
        ctx = _contexts.get(device) or _open(device)
        if stream != ctx[1]:
            _lib.call("esmcu_set_stream", ctx[0], stream if stream else 1)  # 1: cudaStreamLegacy
            ctx[1] = stream
        rc = f(ctx[0], *args)
    if rc != 0:
        _lib.check(rc, f.__name__)


# Workspaces of eager calls, one per device and stream, grown on demand: calls on
# a stream follow one another.  A call that is captured gets memory of its own
# (of the graph's pool), so that graphs share none.
_workspaces: dict[tuple, torch.Tensor] = {}
_capturing = torch._C._cuda_isCurrentStreamCapturing


def _workspace(t, device: int, nbytes: int) -> torch.Tensor:
    if _current_device() != device:
        with torch.cuda.device(device):
            return _workspace(t, device, nbytes)
    if _capturing():
        return t.new_empty((nbytes,), dtype=_U8)
    key = (device, _raw_stream(device))
    w = _workspaces.get(key)
    if w is None or w.numel() < nbytes:
        w = _workspaces[key] = t.new_empty((nbytes,), dtype=_U8)
    return w


def synchronize(device: int = 0) -> None:
    """Waits for torch's current stream and raises on what the device found
    wrong; ops.synchronize calls it."""
    if device in _contexts:
        # The waiting is done without the lock.
        torch.cuda.current_stream(device).synchronize()
        _enqueue(device, _lib.lib().esmcu_synchronize)


def _wrong(msg: str):
    raise ValueError(msg)


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
    dev = x.get_device()
    xs, ws, ss = x.shape, wq.shape, scales.shape
    if len(xs) != 2 or len(ws) != 2 or len(ss) != 2:
        _wrong("x, wq and scales must be matrices")
    if dev < 0:
        _wrong("x must be a CUDA tensor")
    M, K = xs
    N, half = ws
    code, scode = _CODE.get(x.dtype), _CODE.get(scales.dtype)
    if code is None or scode is None:
        _wrong("x and scales must be float32, float16 or bfloat16")
    if group_size not in (32, 64, 128):
        _wrong("group_size must be 32, 64 or 128")
    groups = (K + group_size - 1) // group_size
    if half != (K + 1) // 2 or wq.dtype != _U8:
        _wrong(f"wq must be uint8 [N, {(K + 1) // 2}] for K = {K}")
    if ss[0] != N or ss[1] != groups:
        _wrong(f"scales must be [{N}, {groups}]")
    if wq.get_device() != dev or scales.get_device() != dev:
        _wrong("wq and scales must be on x's device")
    ldx, cx = x.stride()
    ldw, cw = wq.stride()
    lds, cs = scales.stride()
    if (cx != 1 and K > 1) or (cw != 1 and half > 1) or (cs != 1 and groups > 1):
        _wrong("x, wq and scales must be contiguous in their last dimension")
    z = ldz = b = 0
    if zeros is not None:
        if zeros.shape != ss or zeros.dtype != _U8 or zeros.get_device() != dev:
            _wrong("zeros must be uint8, of the shape and on the device of scales")
        ldz, cz = zeros.stride()
        if cz != 1 and groups > 1:
            _wrong("zeros must be contiguous in its last dimension")
        z = zeros.data_ptr()
        if N <= 1:
            ldz = groups
    if bias is not None:
        if bias.shape != (N,) or bias.dtype != _F32 or bias.get_device() != dev or not bias.is_contiguous():
            _wrong(f"bias must be contiguous float32 [{N}] on x's device")
        b = bias.data_ptr()
    if M <= 1:  # torch may give a dimension of one entry any stride
        ldx = K
    if N <= 1:
        ldw, lds = half, groups
    nbytes = _w4_workspace_bytes.get((code, M, K, group_size))
    if nbytes is None:
        n = C.c_size_t()
        _lib.call("esmcu_linear_w4_workspace", code, M, K, group_size, C.byref(n))
        if len(_w4_workspace_bytes) >= 4096:
            _w4_workspace_bytes.clear()
        nbytes = _w4_workspace_bytes[code, M, K, group_size] = n.value
    out = x.new_empty((M, N))
    work = _workspace(x, dev, nbytes) if nbytes else None
    _enqueue(dev, _lib.lib().esmcu_linear_w4,
             _pack_linear(x.data_ptr(), ldx, wq.data_ptr(), ldw, scales.data_ptr(), lds, z, ldz, b, out.data_ptr(), N,
                          0 if work is None else work.data_ptr(), nbytes, code, scode, group_size, M, N, K))
    return out


_pack_linear = struct.Struct("@PqPqPqPqPPqPNiiiiii").pack  # esmcu_linear_w4_args
_pack_append = struct.Struct("@PPPqqqqqqPPPPPiiiiii").pack  # esmcu_kv_append_args
_pack_decode = struct.Struct("@PqqPPPPNiiif").pack  # esmcu_attention_decode_args
_pack_cache = struct.Struct("@PPiiiiiqqqqqqPqi4x").pack  # esmcu_paged_kv


def _paged(k_cache, v_cache, page_table, sequences: int):
    """(device, shape, esmcu_paged_kv as bytes) of a cache."""
    dev = k_cache.get_device()
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype != k_cache.dtype:
        _wrong("k_cache and v_cache must be [pages, page_size, kv_heads, head_dim], of one shape and type")
    if dev < 0:
        _wrong("k_cache must be a CUDA tensor")
    code = _CODE.get(k_cache.dtype)
    if code is None:
        _wrong("the cache must be float32, float16 or bfloat16")
    ts = page_table.shape
    if len(ts) != 2 or page_table.dtype != _I32 or ts[0] < sequences:
        _wrong(f"page_table must be int32 [sequences, max_pages] for at least {sequences} sequences")
    if v_cache.get_device() != dev or page_table.get_device() != dev:
        _wrong("k_cache, v_cache and page_table must be on one device")
    pages, size, heads, dh = shape
    kp, ks, kh, kc = k_cache.stride()
    vp, vs, vh, vc = v_cache.stride()
    tp, tc = page_table.stride()
    if ((kc != 1 or vc != 1) and dh > 1) or (tc != 1 and ts[1] > 1):
        _wrong("k_cache, v_cache and page_table must be contiguous in their last dimension")
    if pages <= 1:  # torch may give a dimension of one entry any stride
        kp = vp = 0
    if size == 1:
        ks = vs = 0
    if heads == 1:
        kh = vh = 0
    return dev, shape, _pack_cache(k_cache.data_ptr(), v_cache.data_ptr(), code, pages, size, heads, dh, kp, ks, kh,
                                   vp, vs, vh, page_table.data_ptr(), tp, ts[1])


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
    if cache_lens.dim() != 1:
        _wrong("cache_lens must be [B]")
    B = cache_lens.shape[0]
    dev, shape, cache = _paged(k_cache, v_cache, page_table, B)
    heads, dh = shape[2], shape[3]
    ksh, dt = k.shape, k.dtype
    if len(ksh) != 3 or ksh[1] != heads or ksh[2] != dh or v.shape != ksh:
        _wrong("k and v must be [T, kv_heads, head_dim] with the cache's heads")
    if (dt != k_cache.dtype and dt != _F32) or v.dtype != dt:
        _wrong("k and v must have the cache's type or be float32, both the same")
    if (cu_seqlens.shape != (B + 1,) or cu_seqlens.dtype != _I32 or cache_lens.dtype != _I32
            or not cu_seqlens.is_contiguous() or not cache_lens.is_contiguous()):
        _wrong("cu_seqlens [B + 1] and cache_lens [B] must be contiguous int32")
    if (k.get_device() != dev or v.get_device() != dev or cu_seqlens.get_device() != dev
            or cache_lens.get_device() != dev):
        _wrong("k, v, cu_seqlens and cache_lens must be on the cache's device")
    T = ksh[0]
    kt, kh, kc = k.stride()
    vt, vh, vc = v.stride()
    if (kc != 1 or vc != 1) and dh > 1:
        _wrong("k and v must be contiguous in their last dimension")
    if T <= 1:
        kt = vt = 0
    if heads == 1:
        kh = vh = 0
    out = None
    qp = op = nq = qt = qh = 0
    if q is not None:
        qs = q.shape
        if len(qs) != 3 or qs[0] != T or qs[2] != dh or q.dtype != dt or q.get_device() != dev:
            _wrong("q must be [T, q_heads, head_dim] of k's type, on the cache's device")
        nq = qs[1]
        qt, qh, qc = q.stride()
        if qc != 1 and dh > 1:
            _wrong("q must be contiguous in its last dimension")
        if T <= 1:
            qt = 0
        if nq <= 1:
            qh = 0
        out = k_cache.new_empty((T, nq, dh))
        if nq:
            qp, op = q.data_ptr(), out.data_ptr()
    cp = sp = rows = rot = 0
    if cos is not None or sin is not None:
        if cos is None or sin is None or cos.dim() != 2 or sin.shape != cos.shape:
            _wrong("cos and sin must both be [positions, rot]")
        if (cos.dtype != _F32 or sin.dtype != _F32 or not cos.is_contiguous() or not sin.is_contiguous()
                or cos.get_device() != dev or sin.get_device() != dev):
            _wrong("cos and sin must be contiguous float32 on the cache's device")
        rows, rot = cos.shape
        cp, sp = cos.data_ptr(), sin.data_ptr()
    if T and B:
        _enqueue(dev, _lib.lib().esmcu_kv_append_paged, cache,
                 _pack_append(qp, k.data_ptr(), v.data_ptr(), qt, qh, kt, kh, vt, vh, cp, sp, cu_seqlens.data_ptr(),
                              cache_lens.data_ptr(), op, _CODE[dt], nq, rows, rot, B, T))
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
    qs = q.shape
    if len(qs) != 3:
        _wrong("q must be [B, q_heads, head_dim]")
    B, nq, dh = qs
    dev, shape, cache = _paged(k_cache, v_cache, page_table, B)
    if dh != shape[3] or q.dtype != k_cache.dtype:
        _wrong("q must have the cache's head_dim and type")
    if seq_lens.shape != (B,) or seq_lens.dtype != _I32 or not seq_lens.is_contiguous():
        _wrong(f"seq_lens must be contiguous int32 [{B}]")
    if q.get_device() != dev or seq_lens.get_device() != dev:
        _wrong("q and seq_lens must be on the cache's device")
    qt, qh, qc = q.stride()
    if qc != 1 and dh > 1:
        _wrong("q must be contiguous in its last dimension")
    if B <= 1:
        qt = 0
    if nq <= 1:
        qh = 0
    window = min(int(window), 0x7FFFFFFF)
    key = (dev, q.dtype, nq, shape[2], dh)
    nbytes = _workspace_bytes.get(key)
    if nbytes is None:
        n = C.c_size_t()
        _enqueue(dev, _lib.lib().esmcu_attention_decode_paged_workspace, cache, nq, C.byref(n))
        nbytes = _workspace_bytes[key] = n.value
    out = q.new_empty(qs)
    lse, lp = None, 0
    if return_lse:
        lse = q.new_empty((B, nq), dtype=_F32)
        lp = lse.data_ptr()
    _enqueue(dev, _lib.lib().esmcu_attention_decode_paged, cache,
             _pack_decode(q.data_ptr(), qt, qh, seq_lens.data_ptr(), out.data_ptr(), lp,
                          _workspace(q, dev, nbytes).data_ptr(), nbytes, nq, B, window, scale))
    return (out, lse) if return_lse else out
