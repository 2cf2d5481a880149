"""Sampling from logits: temperature, min-p, top-k, top-p, given random numbers.

    sample_logits(logits, uniforms, temperature=1.0, top_k=None, top_p=None,
                  min_p=None, ids=None)            -> [B] int64 ids

The entries above -inf (NaN counts as masked) of a row are ordered by falling
logit, then rising column. Every filter keeps a prefix of that order: min-p the
entries with p_i >= min_p * max p, top-k the first k of them, top-p the
shortest prefix that holds top_p of their mass. The draw is the first kept
column, in column order, whose running mass exceeds u * (kept mass): one
uniform number per row, so a row's token depends on its logits, settings and u
alone. Masses are held in 64 bits (``csrc/fh_sample.cuh``).

The reference samples at a temperature alone (``flash_head.py:263-275``).
"""

from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.FH_BF16, torch.float16: _lib.FH_FP16,
           torch.float32: _lib.FH_FP32}
_F32, _F64, _I32, _I64 = torch.float32, torch.float64, torch.int32, torch.int64
_call = None  # fh_sample_logits


def _per_row(name: str, v: torch.Tensor, B: int, dtype: torch.dtype, device) -> torch.Tensor:
    """A setting's [B] values (a single one serves every row) as the kernel reads them."""
    if v.device != device:
        raise ValueError(f"{name} on {v.device}, logits on {device}")
    if v.dtype is dtype and v.dim() == 1 and v.shape[0] == B and v.is_contiguous():
        return v
    if v.numel() == 1 and v.dim() <= 1:
        v = v.reshape(1).expand(B)
    elif v.shape != (B,):
        raise ValueError(f"{name} must be a number or [{B}] values, got {tuple(v.shape)}")
    if dtype is _I32:
        if v.is_floating_point() or v.is_complex():
            raise ValueError(f"{name} must hold integers, got {v.dtype}")
        if v.dtype is _I64:  # beyond 32 bits: every k from n on is the same
            v = v.clamp(-1, 2 ** 31 - 1)
    return v.to(dtype).contiguous()


def _number(name: str, v, low: float, high: float):
    v = float(v)
    if v != v:
        raise ValueError(f"{name} is NaN")
    if not low <= v <= high:
        raise ValueError(f"{name} must be in [{low:g}, {high:g}], got {v}")
    return v


def sample_logits(logits: torch.Tensor, uniforms: torch.Tensor,
                  temperature: Union[float, torch.Tensor] = 1.0,
                  top_k: Union[int, torch.Tensor, None] = None,
                  top_p: Union[float, torch.Tensor, None] = None,
                  min_p: Union[float, torch.Tensor, None] = None,
                  ids: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None, return_prob: bool = False):
    """One id per row of ``logits`` [B, n] (bf16, fp16 or fp32, contiguous rows).

    uniforms: [B] numbers in [0, 1), float64 (float32 is converted).
    temperature, top_k, top_p, min_p: a number, or [B] values on the logits'
        device; temperature 0 is greedy, top_k 0, top_p 1 and min_p 0 (or None)
        switch a filter off. Values outside [0, inf], [0, 2^31), [0, 1] and [0, 1] are
        refused as numbers; in a tensor (not read on the host) those below or above
        switch the filter off, or are greedy, as at the ends.
    ids: int32 [n] or [B, n], the id of every column (default: the column).
    out: [B] int64 for the ids.
    return_prob: also return [B] float32, the drawn entry's share of the kept
        mass.

    A row without an entry above -inf gives -1 (probability 0)."""
    if not logits.is_cuda:
        raise RuntimeError("FlashHead kernels need CUDA tensors (there is no CPU path)")
    if logits.dim() != 2 or logits.dtype not in _DTYPES:
        raise ValueError(f"logits must be [B, n] bf16, fp16 or fp32, got "
                         f"{tuple(logits.shape)} {logits.dtype}")
    B, n = logits.shape
    dev = logits.device
    stride = logits.stride(0)
    if (n > 1 and logits.stride(1) != 1) or (B > 1 and stride < n):
        logits = logits.contiguous()
        stride = n
    if uniforms.shape != (B,) or uniforms.device != dev or not uniforms.is_floating_point():
        raise ValueError(f"uniforms must be [{B}] float64 on {dev}, got "
                         f"{tuple(uniforms.shape)} {uniforms.dtype} on {uniforms.device}")
    if uniforms.dtype is not _F64 or not uniforms.is_contiguous():
        uniforms = uniforms.to(_F64).contiguous()
    tt = kt = pt = mt = None
    t, k, p, m = 1.0, 0, 1.0, 0.0
    if isinstance(temperature, torch.Tensor):
        tt = _per_row("temperature", temperature, B, _F32, dev)
    elif temperature is not None:
        t = _number("temperature", temperature, 0.0, float("inf"))
    if isinstance(top_k, torch.Tensor):
        kt = _per_row("top_k", top_k, B, _I32, dev)
    elif top_k is not None:
        k = int(_number("top_k", top_k, 0, 2 ** 31 - 1))
        if k != top_k:
            raise ValueError(f"top_k must be an integer, got {top_k}")
    if isinstance(top_p, torch.Tensor):
        pt = _per_row("top_p", top_p, B, _F32, dev)
    elif top_p is not None:
        p = _number("top_p", top_p, 0.0, 1.0)
    if isinstance(min_p, torch.Tensor):
        mt = _per_row("min_p", min_p, B, _F32, dev)
    elif min_p is not None:
        m = _number("min_p", min_p, 0.0, 1.0)
    ids_stride = 0
    if ids is not None:
        if ids.dtype is not _I32 or ids.device != dev or ids.shape not in ((n,), (B, n)):
            raise ValueError(f"ids must be int32 [{n}] or [{B}, {n}] on {dev}, got "
                             f"{tuple(ids.shape)} {ids.dtype} on {ids.device}")
        ids = ids.contiguous()
        ids_stride = n if ids.dim() == 2 else 0
    if out is None:
        out = torch.empty(B, dtype=_I64, device=dev)
    elif out.shape != (B,) or out.dtype is not _I64 or out.device != dev \
            or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous [{B}] int64 tensor on {dev}")
    prob = torch.empty(B, dtype=_F32, device=dev) if return_prob else None
    if B:
        global _call
        if _call is None:
            _call = _lib.bound("fh_sample_logits")
        d = _lib.SampleParams(
            None if tt is None else tt.data_ptr(), None if kt is None else kt.data_ptr(),
            None if pt is None else pt.data_ptr(), None if mt is None else mt.data_ptr(),
            uniforms.data_ptr(), None if ids is None else ids.data_ptr(), ids_stride, t, k, p, m)
        with _lib.on_device(dev) as stream:
            st = _call(logits.data_ptr(), _DTYPES[logits.dtype], B, n, max(stride, n),
                       ctypes.byref(d), out.data_ptr(),
                       None if prob is None else prob.data_ptr(), stream)
        _lib.check("fh_sample_logits", st)
    return (out, prob) if return_prob else out
