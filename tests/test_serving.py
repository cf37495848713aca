"""The token-by-token serving operators without a GPU: refusals of the C ABI
(arguments are checked before the context), the index arithmetic of the paged
cache (esm-cpp_b200/csrc/paged.h, compiled for the host) against a plain
restatement, and the 4-bit weight packing."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
INVALID = 1
SOME = 4096  # a non-null pointer that a refused call never follows


def _refused(name, *args, say=""):
    from esm_b200 import _lib

    rc = getattr(_lib.lib(), name)(*args)
    assert rc == INVALID, f"{name} returned {rc}"
    msg = _lib.lib().esmcu_last_error().decode()
    assert say in msg, msg


def _w4(**over):
    from esm_b200 import _lib

    a = dict(x=SOME, ldx=256, dtype=0, wq=SOME, ldw=128, scales=SOME, scales_dtype=0, lds=2, zeros=None,
             ldz=0, group=128, bias=None, out=SOME, ldo=64, M=2, N=64, K=256, workspace=SOME, workspace_bytes=1 << 24)
    a.update(over)
    return None, C.byref(_lib.LinearW4Args(**a))


LONG = dict(M=30, K=8192, ldx=8192, ldw=4096, lds=64)  # x's records need the workspace


@pytest.mark.parametrize("over,say", [
    (dict(), "null context"), (dict(M=-1), "negative"), (dict(N=-1), "negative"), (dict(K=-1), "negative"),
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(scales_dtype=7), "dtype"),
    (dict(group=16), "group"), (dict(group=96), "group"), (dict(group=0), "group"),
    (dict(ldx=255), "stride"), (dict(ldw=127), "stride"), (dict(lds=1), "stride"), (dict(ldo=63), "stride"),
    (dict(zeros=SOME, ldz=1), "stride"), (dict(K=257, ldx=257, ldw=128, lds=3), "stride"),
    (dict(x=None), "null"), (dict(wq=None), "null"), (dict(scales=None), "null"), (dict(out=None), "null"),
    (dict(K=131073, ldx=131073, ldw=65537, lds=1025), "131072"), (dict(LONG, workspace=None), "workspace"), (dict(LONG, workspace_bytes=64), "workspace"), (dict(LONG, workspace=SOME + 8), "workspace"),
])
def test_linear_w4_refusals(over, say):
    _refused("esmcu_linear_w4", *_w4(**over), say=say)


def _cache(**over):
    from esm_b200 import _lib

    a = dict(k=SOME, v=SOME, dtype=2, num_pages=4, page_size=16, num_kv_heads=2, head_dim=64,
             k_stride_page=2048, k_stride_slot=128, k_stride_head=64, v_stride_page=2048,
             v_stride_slot=128, v_stride_head=64, page_table=SOME, page_table_stride=2, max_pages=2)
    a.update(over)
    return _lib.PagedKV(**a)


BAD_CACHES = [
    (dict(dtype=3), "dtype"), (dict(page_size=0), "page_size"), (dict(num_pages=-1), "num_pages"),
    (dict(num_kv_heads=0), "num_kv_heads"), (dict(head_dim=0), "head_dim"), (dict(max_pages=-1), "max_pages"),
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(page_table=None), "null"),
    (dict(k_stride_slot=-1), "stride"), (dict(v_stride_page=-5), "stride"), (dict(page_table_stride=-1), "stride"),
    (dict(k_stride_page=0), "stride of 0"), (dict(v_stride_slot=0), "stride of 0"), (dict(k_stride_head=0), "stride of 0"),
]


def _append(cache, **over):
    from esm_b200 import _lib

    a = dict(q=SOME, q_stride_token=256, q_stride_head=64, num_q_heads=4, k=SOME, k_stride_token=128, k_stride_head=64,
             v=SOME, v_stride_token=128, v_stride_head=64, dtype=2, cos_t=SOME, sin_t=SOME, table_rows=32, rot_dim=64,
             cu_seqlens=SOME, cache_lens=SOME, B=2, T=3, q_out=SOME)
    a.update(over)
    return None, None if cache is None else C.byref(cache), C.byref(_lib.KvAppendArgs(**a))


@pytest.mark.parametrize("over,say", BAD_CACHES)
def test_append_refuses_bad_caches(over, say):
    _refused("esmcu_kv_append_paged", *_append(_cache(**over)), say=say)


@pytest.mark.parametrize("over,say", [
    (dict(), "null context"), (dict(B=-1), "negative"), (dict(T=-1), "negative"), (dict(num_q_heads=-1), "negative"),
    (dict(table_rows=-1), "negative"), (dict(dtype=1), "dtype"), (dict(rot_dim=63), "rot_dim"), (dict(rot_dim=66), "rot_dim"),
    (dict(rot_dim=-2), "rot_dim"), (dict(q_stride_token=-1), "stride"), (dict(v_stride_head=-1), "stride"), (dict(k=None), "null"),
    (dict(v=None), "null"), (dict(cu_seqlens=None), "null"), (dict(cache_lens=None), "null"), (dict(q=None), "q and q_out"),
    (dict(q_out=None), "q and q_out"), (dict(num_q_heads=0), "q and q_out"), (dict(cos_t=None), "null"), (dict(sin_t=None), "null"),
])
def test_append_refusals(over, say):
    _refused("esmcu_kv_append_paged", *_append(_cache(), **over), say=say)


def test_refuses_null_blocks():
    _refused("esmcu_kv_append_paged", *_append(None), say="cache is null")
    _refused("esmcu_kv_append_paged", None, C.byref(_cache()), None, say="args is null")
    _refused("esmcu_attention_decode_paged", *_decode(None), say="cache is null")
    _refused("esmcu_attention_decode_paged", None, C.byref(_cache()), None, say="args is null")
    _refused("esmcu_linear_w4", None, None, say="args is null")


def _decode(cache, **over):
    from esm_b200 import _lib

    a = dict(q=SOME, q_stride_seq=256, q_stride_head=64, num_q_heads=4, seq_lens=SOME, B=2, scale=0.125, window=0,
             out=SOME, lse=None, workspace=SOME, workspace_bytes=1 << 24)
    a.update(over)
    return None, None if cache is None else C.byref(cache), C.byref(_lib.AttentionDecodeArgs(**a))


@pytest.mark.parametrize("over,say", BAD_CACHES + [
    (dict(head_dim=60), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(k=SOME + 8), "16-byte"),
    (dict(v_stride_slot=132), "16-byte"), (dict(k_stride_head=68), "16-byte"), (dict(v_stride_page=2052), "16-byte"),
])
def test_decode_refuses_bad_caches(over, say):
    _refused("esmcu_attention_decode_paged", *_decode(_cache(**over)), say=say)
    n = C.c_size_t(7)
    _refused("esmcu_attention_decode_paged_workspace", None, C.byref(_cache(**over)), 4, C.byref(n), say=say)
    assert n.value == 0


@pytest.mark.parametrize("over,say", [
    (dict(), "null context"), (dict(num_q_heads=3), "num_q_heads"), (dict(num_q_heads=0), "num_q_heads"), (dict(B=-1), "negative"),
    (dict(window=-1), "window"), (dict(q_stride_seq=-1), "stride"), (dict(q=None), "null"), (dict(seq_lens=None), "null"),
    (dict(out=None), "null"), (dict(out=SOME + 8), "out must be 16-byte"),
])
def test_decode_refusals(over, say):
    _refused("esmcu_attention_decode_paged", *_decode(_cache(), **over), say=say)


def test_python_refusals():
    import torch

    from esm_b200 import ops

    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear_w4(x, torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 1))
    kc = torch.zeros(4, 16, 2, 64)
    table = torch.zeros(2, 2, dtype=torch.int32)
    lens = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attention_decode_paged(torch.zeros(2, 4, 64), kc, kc, table, lens)
    with pytest.raises(ValueError, match="one shape"):
        ops.kv_append_paged(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), kc, kc[:, :8], table,
                            torch.zeros(3, dtype=torch.int32), lens)


# --------------------------------------------------- index arithmetic (host)
SHIM = r"""
#include "paged.h"
extern "C" {
void append_place_c(const int* cu, int B, const int* lens, const int* table, long stride, int max_pages,
                    int page_size, int num_pages, int rows, int t, int* out) {
  const esmb200::Place p = esmb200::append_place(cu, B, lens, table, stride, max_pages, page_size, num_pages, rows, t);
  out[0] = p.page; out[1] = p.slot; out[2] = p.pos; out[3] = p.bad;
}
void key_range_c(int len, int max_pages, int page_size, int window, int* out) {
  const esmb200::KeyRange r = esmb200::key_range(len, max_pages, page_size, window);
  out[0] = r.first; out[1] = r.end; out[2] = r.bad;
}
int tiles_c(int first, int end) { return esmb200::tiles_of(esmb200::KeyRange{first, end, 0}); }
}
"""


@pytest.fixture(scope="module")
def paged(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", f"-I{ROOT / 'esm-cpp_b200' / 'csrc'}",
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    return C.CDLL(str(d / "shim.so"))


def test_append_places(paged):
    rng = np.random.default_rng(0)
    for _ in range(300):
        B = int(rng.integers(0, 6))
        new = rng.integers(0, 5, B)
        cu = (np.concatenate([[0], np.cumsum(new)]) + rng.integers(0, 3)).astype(np.int32)
        lens = rng.integers(-2, 30, B).astype(np.int32)
        page_size, max_pages, num_pages = int(rng.integers(1, 9)), int(rng.integers(0, 6)), int(rng.integers(1, 9))
        table = rng.integers(-1, num_pages + 1, (max(B, 1), max_pages + 1)).astype(np.int32)
        rows = int(rng.choice([-1, 0, 10, 100]))
        for t in range(int(cu[-1]) + 3):
            out = np.zeros(4, np.int32)
            paged.append_place_c(C.c_void_p(cu.ctypes.data), B, C.c_void_p(lens.ctypes.data),
                                 C.c_void_p(table.ctypes.data), C.c_long(max_pages + 1), max_pages, page_size,
                                 num_pages, rows, t, C.c_void_p(out.ctypes.data))
            owner = [b for b in range(B) if cu[b] <= t < cu[b + 1]]
            if not owner:
                assert out[0] == -1 and out[3] == 0
                continue
            b = owner[0]
            pos = int(lens[b]) + t - int(cu[b])
            ok = lens[b] >= 0 and pos // page_size < max_pages and (rows < 0 or pos < rows)
            ok = ok and 0 <= table[b, pos // page_size] < num_pages
            if ok:
                assert out.tolist() == [table[b, pos // page_size], pos % page_size, pos, 0]
            else:
                assert out[0] == -1 and out[3] == 1


def test_tiles(paged):
    top = 2**31 - 1
    for first, end in [(0, 0), (5, 5), (0, 1), (0, 16), (0, 17), (15, 16), (15, 17), (16, 32), (31, 33), (0, top),
                       (0, top - 14), (0, top - 15), (0, top - 16), (top - 17, top), (top - 1, top)]:
        assert paged.tiles_c(first, end) == len(range(first // 16 * 16, end, 16)) * (first < end), (first, end)


def test_append_place_survives_extreme_lengths(paged):
    cu, table = np.array([0, 4], np.int32), np.zeros((1, 4), np.int32)
    for n in (2**31 - 1, 2**31 - 3, -2**31):
        lens = np.array([n], np.int32)
        for t in range(4):
            out = np.zeros(4, np.int32)
            paged.append_place_c(C.c_void_p(cu.ctypes.data), 1, C.c_void_p(lens.ctypes.data),
                                 C.c_void_p(table.ctypes.data), C.c_long(4), 4, 16, 1, -1, t,
                                 C.c_void_p(out.ctypes.data))
            assert out[0] == -1 and out[3] == 1


@pytest.mark.parametrize("n,max_pages,page_size,window,want", [
    (0, 4, 16, 0, (0, 0, 0)), (64, 4, 16, 0, (0, 64, 0)), (65, 4, 16, 0, (0, 64, 1)), (-1, 4, 16, 0, (0, 0, 1)),
    (10, 4, 16, 3, (7, 10, 0)), (2, 4, 16, 3, (0, 2, 0)), (100, 4, 16, 3, (61, 64, 1)), (5, 0, 16, 0, (0, 0, 1)),
    (2**31 - 1, 2**31 - 1, 128, 0, (0, 2**31 - 1, 0)), (2**31 - 1, 2**20, 2048, 1, (2**31 - 2, 2**31 - 1, 0)),
])
def test_key_ranges(paged, n, max_pages, page_size, window, want):
    out = np.zeros(3, np.int32)
    paged.key_range_c(n, max_pages, page_size, window, C.c_void_p(out.ctypes.data))
    assert tuple(out) == want


# ------------------------------------------------------------ 4-bit packing
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (5, 64, 32), (7, 129, 64), (3, 257, 128), (4, 256, 128)])
def test_quantize_weight_w4(n, k, group):
    from esm_b200 import prep

    rng = np.random.default_rng(n * k)
    w = rng.standard_normal((n, k)).astype(np.float32)
    w[0, :min(k, group)] = 0.0  # an all-zero group
    packed, scale = prep.quantize_weight_w4(w, group)
    assert packed.shape == (n, (k + 1) // 2) and packed.dtype == np.uint8
    assert scale.shape == (n, -(-k // group)) and scale.dtype == np.float32 and scale[0, 0] == 0
    q = np.stack([packed & 15, packed >> 4], -1).reshape(n, -1)[:, :k].astype(int) - 8
    assert q.min() >= -7 and q.max() <= 7
    s = np.repeat(scale, group, axis=1)[:, :k].astype(np.float64)
    # half a step, and the float divisions' roundings (7 * 2^-23 of a step at most)
    assert np.all(np.abs(q * s - w) <= s * (0.5 + 2.0**-20))
    with pytest.raises(ValueError):
        prep.quantize_weight_w4(w, 48)


def test_linear_w4_workspace_of_most_rows():
    """Many rows run as equal passes of at most as many rows as one can take:
    64 of float16 at this K."""
    from esm_b200 import _lib

    def need(M):
        n = C.c_size_t()
        assert _lib.lib().esmcu_linear_w4_workspace(1, M, 4096, 128, C.byref(n)) == 0
        return n.value

    assert need(2**31 - 1) == need(64) > 0


@pytest.mark.parametrize("over", [dict(x=SOME + 2), dict(out=SOME + 2), dict(scales=SOME + 1, scales_dtype=1),
                                  dict(bias=SOME + 2), dict(dtype=2, x=SOME + 1)])
def test_linear_w4_refuses_split_elements(over):
    _refused("esmcu_linear_w4", *_w4(**over), say="boundary")


@pytest.mark.parametrize("over", [dict(q=SOME + 1), dict(k=SOME + 1), dict(v=SOME + 1), dict(q_out=SOME + 1),
                                  dict(cos_t=SOME + 2), dict(sin_t=SOME + 2), dict(cu_seqlens=SOME + 2),
                                  dict(cache_lens=SOME + 1)])
def test_append_refuses_split_elements(over):
    _refused("esmcu_kv_append_paged", *_append(_cache(), **over), say="boundary")


@pytest.mark.parametrize("over", [dict(k=SOME + 1), dict(v=SOME + 1), dict(page_table=SOME + 2)])
def test_caches_refuse_split_elements(over):
    _refused("esmcu_kv_append_paged", *_append(_cache(**over)), say="boundary")
    _refused("esmcu_attention_decode_paged", *_decode(_cache(**over)), say="boundary")


@pytest.mark.parametrize("over", [dict(q=SOME + 1), dict(seq_lens=SOME + 2), dict(lse=SOME + 2)])
def test_decode_refuses_split_elements(over):
    _refused("esmcu_attention_decode_paged", *_decode(_cache(), **over), say="boundary")


def test_build_goes_on_without_torch(tmp_path, monkeypatch):
    """The library needs no torch; only the binding is left out."""
    import importlib.util
    import sys

    spec = importlib.util.spec_from_file_location("esm_b200_build_no_torch", ROOT / "esm-cpp_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    monkeypatch.setattr(build, "OUT_EXT", tmp_path / "ext.so")
    monkeypatch.setitem(sys.modules, "torch", None)
    build._build_ext(True)
    assert not build.OUT_EXT.exists()


def test_binding_refuses_before_any_device():
    """Wrong tensors are a ValueError here too, where there is no GPU."""
    import torch

    from esm_b200 import ops

    x, wq, s = torch.zeros(2, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 1)
    kc, lens = torch.zeros(1, 16, 2, 64), torch.ones(1, dtype=torch.int32)
    for call in (lambda: ops.linear_w4(x, wq, s), lambda: ops.linear_w4(x[0], wq, s),
                 lambda: ops.kv_append_paged(kc[0], kc[0], kc, kc, lens[None], lens, lens),
                 lambda: ops.attention_decode_paged(kc[:, 0], kc, kc, lens[None], lens),
                 lambda: ops.attention_decode_paged(kc[0, 0], kc, kc, lens[None], lens)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.linear_w4(x, wq, None)
