"""The token-by-token serving operators (include/esm_b200.h, section 3) over
torch CUDA tensors, reached as ops.linear_w4, ops.kv_append_paged and
ops.attention_decode_paged: a 4-bit Linear for few rows, the append to a paged
K/V cache with RoPE on the way, and the attention of one new token over it.

The functions are those of the native binding (csrc/binding/serving_ext.cpp,
built by build.py), which calls the same C ABI through the addresses handed to
it here.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

try:
    from . import _serving_ext as _ext
except ImportError as e:
    raise ImportError(f"the serving operators' binding cannot be loaded ({e}): build it with "
                      "`python esm-cpp_b200/build.py`") from e

_ext.bind({name: C.cast(getattr(_lib.lib(), name), C.c_void_p).value
           for name in ("esmcu_open", "esmcu_set_stream", "esmcu_synchronize", "esmcu_linear_w4",
                        "esmcu_linear_w4_workspace", "esmcu_kv_append_paged", "esmcu_attention_decode_paged",
                        "esmcu_attention_decode_paged_workspace")}, _lib.check)

linear_w4 = _ext.linear_w4
kv_append_paged = _ext.kv_append_paged
attention_decode_paged = _ext.attention_decode_paged


def synchronize(device: int = 0) -> None:
    """Waits for torch's current stream and raises on what the device has found
    wrong since the last look, in calls on any of its streams; ops.synchronize
    calls it."""
    if torch.cuda.is_available():
        torch.cuda.current_stream(device).synchronize()
        _ext.synchronize(device)
