"""The serving operators' host side without a GPU, beyond test_serving: the status
word, builds without a binding, calls that want gradients, empty weights."""
import ctypes as C
import importlib.util
import subprocess
import sys
import types
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def _shim(tmp_path, text):
    (tmp_path / "shim.cpp").write_text(text)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", f"-I{ROOT / 'esm-cpp_b200' / 'csrc'}",
                    str(tmp_path / "shim.cpp"), "-o", str(tmp_path / "shim.so")], check=True)
    return C.CDLL(str(tmp_path / "shim.so"))


# ------------------------------------------------------------ status word
STATUS = r"""
#include "status.h"
using namespace esmb200;
// A look at a word that holds `first`, while kernels elsewhere set `between` behind
// the read and `after` behind the exchange; out: what was found, what is left.
extern "C" int look(uint32_t first, uint32_t between, uint32_t after, int read_rc, int take_rc, uint32_t* out) {
  uint32_t word = first;
  int takes = 0;
  const int rc = take_status(
      [&](uint32_t& w) { w = word; word |= between; return read_rc; },
      [&](uint32_t& w) { ++takes; w = word; word = 0; word |= after; return take_rc; }, out[0]);
  out[1] = word;
  out[2] = takes;
  return rc;
}
"""


def test_no_status_bit_is_lost(tmp_path):
    look = _shim(tmp_path, STATUS).look
    out = (C.c_uint32 * 3)()
    for first in range(4):
        for between in range(4):
            for after in range(4):
                assert look(first, between, after, 0, 0, out) == 0
                if first == 0:  # nothing found: nothing touched
                    assert list(out) == [0, between, 0]
                else:
                    assert list(out) == [first | between, after, 1]
    assert look(2, 0, 0, 7, 0, out) == 7 and list(out)[1:] == [2, 0]
    assert look(2, 0, 0, 0, 7, out) == 7


# --------------------------------------------------- numbers of a device
PER_DEVICE = r"""
#include "per_device.h"
static esmb200::PerDevice numbers;
static int asked = 0;
extern "C" int number(int device, int answer) {
  return numbers.get(device, [&] { ++asked; return answer; });
}
extern "C" int times() { return asked; }
"""


def test_a_number_is_asked_of_each_device(tmp_path):
    """Two devices of different sizes in one process keep their own answers."""
    lib = _shim(tmp_path, PER_DEVICE)
    assert [lib.number(0, 18), lib.number(1, 16), lib.number(0, 7), lib.number(1, 7)] == [18, 16, 18, 16]
    assert lib.times() == 2
    assert [lib.number(2, 0), lib.number(2, 5), lib.number(2, 6)] == [0, 5, 5]  # a device that could not say
    assert [lib.number(64, 3), lib.number(64, 4), lib.number(-1, 5)] == [3, 4, 5]  # no place: asked every time


# ------------------------------------------------------------------ builds
@pytest.fixture
def build(tmp_path, monkeypatch):
    """build.py with its outputs in tmp_path."""
    spec = importlib.util.spec_from_file_location("esm_b200_build_limits", ROOT / "esm-cpp_b200" / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    for name, file in (("OUT_SO", "lib.so"), ("OUT_EXT", "ext.so"), ("EXT_TORCH", "ext.torch")):
        monkeypatch.setattr(module, name, tmp_path / file)
    return module


def test_the_library_is_built_where_the_binding_fails(build, tmp_path, monkeypatch):
    (tmp_path / "empty.cpp").write_text("int nothing;\n")
    obj = tmp_path / "empty.o"
    subprocess.run([build.CXX, "-c", "-fPIC", str(tmp_path / "empty.cpp"), "-o", str(obj)], check=True)
    monkeypatch.setattr(build, "_compile", lambda *a: obj)
    monkeypatch.setattr(build, "REPO", tmp_path)

    def fails(force):
        raise RuntimeError("no c10")

    monkeypatch.setattr(build, "_build_ext", fails)
    monkeypatch.setattr(build, "_sources", lambda: ([obj], [], [obj]))
    with pytest.raises(RuntimeError, match="no c10"):
        build.build(verbose=False)
    assert build.OUT_SO.exists()


def test_a_torch_without_cuda_leaves_the_binding_out(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", types.SimpleNamespace(version=types.SimpleNamespace(cuda=None)))
    build._build_ext(True)
    assert not build.OUT_EXT.exists() and "without CUDA" in capsys.readouterr().out


def test_the_binding_is_built_again_for_another_torch(build, monkeypatch):
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        build.OUT_EXT.touch()
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build.subprocess, "run", run)
    for version, count in (("1.0", 1), ("1.0", 1), ("1.1", 2), ("1.1", 2)):
        monkeypatch.setattr(build, "_torch_version", lambda: version)
        build._build_ext(False)
        assert len(calls) == count, version


def test_build_entry_without_torch():
    code = "import sys; sys.modules['torch'] = None; import __graft_entry__; __graft_entry__.build(); print('built it')"
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=1200)
    assert r.returncode == 0 and "built it" in r.stdout, r.stderr[-2000:]


# --------------------------------------------------------------- gradients
def test_inputs_that_want_gradients_are_refused():
    """An output without its gradient would say nothing; with gradients off the
    calls come to their other checks (here: no CUDA tensor)."""
    import torch

    from esm_b200 import ops

    def w4(x=False, scales=False, bias=False):
        ops.linear_w4(torch.zeros(2, 64, requires_grad=x), torch.zeros(8, 32, dtype=torch.uint8),
                      torch.zeros(8, 1, requires_grad=scales), None, torch.zeros(8, requires_grad=bias))

    lens, table = torch.ones(1, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32)
    cu = torch.tensor([0, 2], dtype=torch.int32)

    def append(k=False, v=False, kc=False, vc=False, q=False, cos=False, sin=False):
        ops.kv_append_paged(torch.zeros(2, 2, 64, requires_grad=k), torch.zeros(2, 2, 64, requires_grad=v),
                            torch.zeros(4, 16, 2, 64, requires_grad=kc), torch.zeros(4, 16, 2, 64, requires_grad=vc),
                            table, cu, lens, torch.zeros(2, 4, 64, requires_grad=q),
                            torch.zeros(8, 64, requires_grad=cos), torch.zeros(8, 64, requires_grad=sin))

    def attend(q=False, kc=False, vc=False):
        ops.attention_decode_paged(torch.zeros(1, 4, 64, requires_grad=q), torch.zeros(4, 16, 2, 64, requires_grad=kc),
                                   torch.zeros(4, 16, 2, 64, requires_grad=vc), table, lens)

    for call, names in ((w4, ("x", "scales", "bias")), (append, ("k", "v", "kc", "vc", "q", "cos", "sin")),
                        (attend, ("q", "kc", "vc"))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
        for name in names:
            with pytest.raises(ValueError, match="gradient"):
                call(**{name: True})
            with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
                call(**{name: True})


# ------------------------------------------------------------ 4-bit packing
@pytest.mark.parametrize("n,k", [(0, 64), (0, 0), (3, 0), (0, 5)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_weight_w4_of_no_weights(n, k, group):
    import numpy as np

    from esm_b200 import prep

    packed, scales = prep.quantize_weight_w4(np.zeros((n, k), np.float32), group)
    assert packed.shape == (n, (k + 1) // 2) and scales.shape == (n, -(-k // group))
    assert packed.dtype == np.uint8 and scales.dtype == np.float32
