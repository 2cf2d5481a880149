"""Filtered sampling on the CPU: refusals of the Python entry and of the C ABI."""

from __future__ import annotations

import ctypes
import os
import subprocess

import pytest
import torch

from conftest import REPO
from flash_head import _lib
from flash_head.sampling import sample_logits


class FakeCuda(torch.Tensor):
    """A CPU tensor that says it lives on a GPU (argument checks only)."""

    is_cuda = property(lambda self: True)


def fake(t):
    return t.as_subclass(FakeCuda)


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        sample_logits(torch.zeros(1, 4), torch.zeros(1))


@pytest.mark.parametrize("kw,msg", [
    ({"temperature": -1.0}, "temperature"), ({"temperature": float("nan")}, "NaN"),
    ({"top_k": -3}, "top_k"), ({"top_p": 1.5}, "top_p"), ({"top_p": -0.1}, "top_p"),
    ({"min_p": 2.0}, "min_p"), ({"top_p": float("nan")}, "top_p"),
    ({"top_k": torch.zeros(3, dtype=torch.int32)}, "top_k"),
    ({"temperature": torch.zeros(2, 1)}, "temperature"),
    ({"ids": torch.zeros(8, dtype=torch.int64)}, "ids"),
    ({"ids": torch.zeros(7, dtype=torch.int32)}, "ids"),
    ({"out": torch.zeros(2, dtype=torch.int32)}, "out"),
    ({"out": torch.zeros(3, dtype=torch.int64)}, "out")])
def test_refused_arguments(kw, msg):
    x, u = fake(torch.zeros(2, 8)), torch.zeros(2, dtype=torch.float64)
    with pytest.raises(ValueError, match=msg):
        sample_logits(x, u, **kw)


def test_refused_tensors():
    u = torch.zeros(2, dtype=torch.float64)
    with pytest.raises(ValueError, match="logits"):
        sample_logits(fake(torch.zeros(2, 8, dtype=torch.float64)), u)
    with pytest.raises(ValueError, match="logits"):
        sample_logits(fake(torch.zeros(8)), u)
    with pytest.raises(ValueError, match="uniforms"):
        sample_logits(fake(torch.zeros(2, 8)), u[:1])
    with pytest.raises(ValueError, match="uniforms"):
        sample_logits(fake(torch.zeros(2, 8)), u.long())


@pytest.fixture(scope="module")
def lib():
    from importlib import util
    spec = util.spec_from_file_location("fh_build",
                                        os.path.join(REPO, "flash-head_b200", "build.py"))
    mod = util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.build()
    return _lib.load_library()


def test_refused_calls(lib):
    at, bad = 1 << 20, _lib.FH_ERR_INVALID_ARGUMENT
    d = _lib.SampleParams()
    d.uniforms, d.temperature_all, d.top_p_all = at, 1.0, 1.0
    ref = ctypes.byref(d)
    f = lib.fh_sample_logits
    assert f(None, _lib.FH_FP32, 0, 10, 10, ref, None, None, None) == _lib.FH_OK
    assert f(at, _lib.FH_FP32, -1, 10, 10, ref, at, None, None) == bad
    assert f(at, _lib.FH_FP32, 1, -1, 10, ref, at, None, None) == bad
    assert f(at, _lib.FH_FP32, 1, (1 << 28) + 1, 1 << 29, ref, at, None, None) == bad
    assert f(at, _lib.FH_FP8_E4M3, 1, 10, 10, ref, at, None, None) == bad
    assert f(at, _lib.FH_FP32, 1, 10, 9, ref, at, None, None) == bad
    assert "row_stride" in _lib.last_error()
    assert f(at, _lib.FH_FP32, 1, 10, 10, None, at, None, None) == bad
    assert f(None, _lib.FH_FP32, 1, 10, 10, ref, at, None, None) == bad
    assert f(at, _lib.FH_FP32, 1, 10, 10, ref, None, None, None) == bad
    assert f(at + 2, _lib.FH_FP32, 1, 10, 10, ref, at, None, None) == bad
    assert "aligned" in _lib.last_error()
    d.ids, d.ids_stride = at, 5
    assert f(at, _lib.FH_FP32, 1, 10, 10, ref, at, None, None) == bad
    d.ids, d.uniforms = None, None
    assert f(at, _lib.FH_FP32, 1, 10, 10, ref, at, None, None) == bad


def test_params_layout_matches_the_header(tmp_path):
    fields = [f for f, _ in _lib.SampleParams._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "flashhead.h"\n'
                   "int main(void){printf(\"%zu\\n\", sizeof(fh_sample_params));\n"
                   + "".join(f'printf("%zu\\n", offsetof(fh_sample_params, {f}));\n' for f in fields)
                   + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()
    assert int(out[0]) == ctypes.sizeof(_lib.SampleParams)
    for f, off in zip(fields, out[1:]):
        assert getattr(_lib.SampleParams, f).offset == int(off), f
