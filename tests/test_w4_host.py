"""The 4-bit weight on the CPU: its layout, quantisation and refusals."""

from __future__ import annotations

import ctypes
import os
import subprocess

import pytest
import torch

from conftest import REPO
from flash_head import _lib
from flash_head.w4 import W4Weight, w4_block_sparse_logits, w4_logits


def _quantized(V, D, group, zeros=True, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (V, D // 2), generator=g, dtype=torch.uint8)
    s = torch.rand(V, D // group, generator=g).to(dtype)
    z = torch.randint(0, 16, (V, D // group), generator=g, dtype=torch.uint8) if zeros else None
    return q, s, z


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("V,D,group", [(1, 32, 32), (5, 96, 32), (130, 192, 64), (300, 640, 128)])
def test_layout_round_trip(V, D, group, zeros):
    q, s, z = _quantized(V, D, group, zeros)
    w = W4Weight.from_quantized(q, s, z)
    v = torch.stack([q & 15, q >> 4], 2).view(V, -1, group).float()
    want = (v - (8.0 if z is None else z.float().unsqueeze(2))) * s.float().unsqueeze(2)
    assert torch.equal(w.dequantize(), want.view(V, D))
    assert w.shape == (V, D) and w.group_size == group


def test_layout_words():
    """Word j of quad c of row r of block b holds columns 128b + 32j + 8c + e
    (even e in bits 2e.., odd e in bits 16 + 2(e-1)..); padding has scale 0."""
    V, D, group = 20, 256, 64
    q, s, z = _quantized(V, D, group)
    w = W4Weight.from_quantized(q, s, z)
    v = torch.stack([q & 15, q >> 4], 2).view(V, D).tolist()
    assert w.qweight.shape == (1, 2, 4, 128, 4)  # rows padded to 128
    words = w.qweight.tolist()
    for r, b, c, j in [(0, 0, 0, 0), (7, 1, 3, 2), (19, 0, 1, 3), (16, 1, 2, 1)]:
        word = words[r // 128][b][c][r % 128][j] & 0xFFFFFFFF
        for e in range(8):
            at = 4 * (e // 2) + 16 * (e % 2)
            assert (word >> at) & 15 == v[r][128 * b + 32 * j + 8 * c + e]
    assert w.scales[0, 1, 19, 0] == s[19, 2] and w.zeros[0, 1, 19, 1] == z[19, 3]
    assert (w.scales[0, :, 20:] == 0).all() and (w.zeros[0, :, 20:] == 8).all()


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantisation(zeros, dtype):
    g = torch.Generator().manual_seed(1)
    W = (torch.randn(64, 256, generator=g) * 0.02).to(dtype)
    W[3] = 0.0
    w = W4Weight.from_dense(W, 64, zeros)
    assert torch.isfinite(w.dequantize()).all() and (w.dequantize()[3] == 0).all()
    # weights on the grid come back exactly
    grid = (torch.randint(-7, 8, (8, 128), generator=g).float() * 2.0 ** -6).to(dtype)
    grid[:, 0] = 7 * 2.0 ** -6
    if not zeros:
        assert torch.equal(W4Weight.from_dense(grid, 128).dequantize(), grid.float())


def test_refused_weights():
    q, s, z = _quantized(8, 128, 64)
    ok = W4Weight.from_quantized(q, s, z)
    assert ok.nbytes == 128 * 64 + 128 * 2 * 3
    with pytest.raises(ValueError, match="uint8"):
        W4Weight.from_quantized(q.int(), s, z)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        W4Weight.from_quantized(q, s.float(), z)
    with pytest.raises(ValueError, match="do not fit"):
        W4Weight.from_quantized(q, s[:4], None)
    with pytest.raises(ValueError, match="group_size"):
        W4Weight.from_quantized(q, s[:, :1].repeat(1, 8), None)  # groups of 16
    with pytest.raises(ValueError, match="shape of scales"):
        W4Weight.from_quantized(q, s, z[:, :1])
    with pytest.raises(ValueError, match="0..15"):
        W4Weight.from_quantized(q, s, z + 16)
    with pytest.raises(ValueError, match="multiple of group_size"):
        W4Weight.from_dense(torch.zeros(4, 96, dtype=torch.bfloat16), 64)
    with pytest.raises(ValueError, match="exceeds"):
        W4Weight.from_dense(torch.zeros(1, 16384, dtype=torch.bfloat16), 64)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        W4Weight.from_dense(torch.zeros(4, 128), 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        w4_logits(torch.zeros(1, 128, dtype=torch.bfloat16), ok)
    with pytest.raises(RuntimeError, match="no CPU path"):
        w4_block_sparse_logits(torch.zeros(1, 128, dtype=torch.bfloat16), ok,
                               torch.zeros(1, 1, dtype=torch.int64), 1, 8)


@pytest.fixture(scope="module")
def lib():
    from importlib import util
    spec = util.spec_from_file_location("fh_build",
                                        os.path.join(REPO, "flash-head_b200", "build.py"))
    mod = util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.build()
    return _lib.load_library()


def _desc(**kw):
    d = _lib.W4Desc()
    fake = 1 << 20  # aligned, never dereferenced by validation
    d.vocab, d.hidden, d.group_size, d.dtype = 1000, 256, 64, _lib.FH_BF16
    d.qweight, d.scales, d.row_mul = fake, fake, fake
    for k, v in kw.items():
        setattr(d, k, v)
    return ctypes.byref(d)


@pytest.mark.parametrize("field,value,msg", [
    ("vocab", 0, "vocab"), ("hidden", 0, "hidden"), ("hidden", 96, "multiple of group_size"),
    ("hidden", 12288 + 64, "at most"), ("group_size", 48, "group_size"),
    ("dtype", _lib.FH_FP32, "dtype"), ("qweight", None, "null"), ("scales", None, "null"),
    ("row_mul", None, "null"),
    ("qweight", (1 << 20) + 8, "aligned"), ("zeros", (1 << 20) + 1, "aligned")])
def test_refused_descriptors(lib, field, value, msg):
    fake = 1 << 20
    d = _desc(**{field: value})
    assert lib.fh_w4_logits(d, fake, 1, fake, 1000, None, 0, None) == _lib.FH_ERR_INVALID_ARGUMENT
    assert msg in _lib.last_error()
    st = lib.fh_w4_block_sparse_logits(d, fake, 1, fake, 4, 10, 16, fake, None)
    assert st == _lib.FH_ERR_INVALID_ARGUMENT and msg in _lib.last_error()


def test_refused_calls(lib):
    fake, bad = 1 << 20, _lib.FH_ERR_INVALID_ARGUMENT
    d = _desc()
    assert lib.fh_w4_logits(d, None, 0, None, 0, None, 0, None) == _lib.FH_OK
    assert lib.fh_w4_logits(None, fake, 1, fake, 1000, None, 0, None) == bad
    assert lib.fh_w4_logits(d, fake, -1, fake, 1000, None, 0, None) == bad
    assert lib.fh_w4_logits(d, fake + 2, 1, fake, 1000, None, 0, None) == bad
    assert lib.fh_w4_logits(d, fake, 1, fake + 1, 1000, None, 0, None) == bad
    assert lib.fh_w4_logits(d, fake, 1, fake, 999, None, 0, None) == bad
    assert "out_stride" in _lib.last_error()
    # more than 8 rows need a workspace
    assert lib.fh_w4_workspace_bytes(d, 8) == 0 and lib.fh_w4_workspace_bytes(None, 99) == 0
    need = lib.fh_w4_workspace_bytes(d, 20)
    assert need == 256 + 256 + 20 * 256 * 2
    assert lib.fh_w4_logits(d, fake, 20, fake, 1000, fake, need - 1, None) == _lib.FH_ERR_WORKSPACE
    assert lib.fh_w4_logits(d, fake, 20, fake, 1000, None, 0, None) == _lib.FH_ERR_WORKSPACE
    assert lib.fh_w4_logits(d, fake, 20, fake, 1000, fake + 4, need, None) == bad
    blk = lib.fh_w4_block_sparse_logits
    assert blk(d, None, 0, None, 4, 10, 16, None, None) == _lib.FH_OK
    assert blk(d, None, 3, None, 0, 10, 16, None, None) == _lib.FH_OK
    assert blk(d, fake, -1, fake, 0, 10, 16, fake, None) == bad
    assert blk(d, fake, 1, fake, -4, 10, 16, fake, None) == bad
    assert blk(d, fake, 1, None, 4, 10, 16, fake, None) == bad
    assert blk(d, fake, 1, fake, 4, 63, 16, fake, None) == bad
    assert "exceeds vocab" in _lib.last_error()
    assert blk(d, fake, 1, fake, 4, 10, 0, fake, None) == bad
    assert blk(d, fake, 1 << 20, fake, 1 << 20, 10, 16, fake, None) == bad


def test_desc_layout_matches_the_header(tmp_path):
    fields = [f for f, _ in _lib.W4Desc._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "flashhead.h"\n'
                   "int main(void){printf(\"%zu\\n\", sizeof(fh_w4_desc));\n"
                   + "".join(f'printf("%zu\\n", offsetof(fh_w4_desc, {f}));\n' for f in fields)
                   + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()
    assert int(out[0]) == ctypes.sizeof(_lib.W4Desc)
    for f, off in zip(fields, out[1:]):
        assert getattr(_lib.W4Desc, f).offset == int(off), f
