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

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _per_row(name: str, value, B: int, dtype: torch.dtype, device, off):
    """(tensor or None, scalar) of a setting given as None, a number or [B]."""
    if value is None:
        return None, off
    if not isinstance(value, torch.Tensor):
        value = float(value) if dtype.is_floating_point else int(value)
        if value != value:
            raise ValueError(f"{name} is NaN")
        return None, value
    if value.dim() > 1 or value.numel() not in (1, B) or (value.numel() == 1 and B != 1):
        if value.numel() != 1:
            raise ValueError(f"{name} must be a number or [{B}] values, got {tuple(value.shape)}")
        value = value.reshape(1).expand(B)
    if value.device != device:
        raise ValueError(f"{name} on {value.device}, logits on {device}")
    return value.reshape(B).to(dtype).contiguous(), off


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
        switch a filter off.
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
    if (n > 1 and logits.stride(1) != 1) or (B > 1 and logits.stride(0) < n):
        logits = logits.contiguous()
    if uniforms.shape != (B,) or uniforms.device != dev or not uniforms.is_floating_point():
        raise ValueError(f"uniforms must be [{B}] float64 on {dev}, got "
                         f"{tuple(uniforms.shape)} {uniforms.dtype} on {uniforms.device}")
    uniforms = uniforms.to(torch.float64).contiguous()
    if not isinstance(temperature, torch.Tensor) and float(temperature) < 0:
        raise ValueError(f"temperature must be >= 0, got {temperature}")
    if not isinstance(top_k, torch.Tensor) and top_k is not None and int(top_k) < 0:
        raise ValueError(f"top_k must be >= 0, got {top_k}")
    for name, v in (("top_p", top_p), ("min_p", min_p)):
        if not isinstance(v, torch.Tensor) and v is not None and not 0.0 <= float(v) <= 1.0:
            raise ValueError(f"{name} must be in [0, 1], got {v}")
    d = _lib.SampleParams()
    f32 = torch.float32
    t, d.temperature_all = _per_row("temperature", temperature, B, f32, dev, 1.0)
    k, d.top_k_all = _per_row("top_k", top_k, B, torch.int32, dev, 0)
    p, d.top_p_all = _per_row("top_p", top_p, B, f32, dev, 1.0)
    m, d.min_p_all = _per_row("min_p", min_p, B, f32, dev, 0.0)
    for name, v in (("temperature", t), ("top_k", k), ("top_p", p), ("min_p", m)):
        setattr(d, name, None if v is None else v.data_ptr())
    d.uniforms = uniforms.data_ptr()
    if ids is not None:
        if ids.dtype != torch.int32 or ids.device != dev or ids.shape not in ((n,), (B, n)):
            raise ValueError(f"ids must be int32 [{n}] or [{B}, {n}] on {dev}, got "
                             f"{tuple(ids.shape)} {ids.dtype} on {ids.device}")
        ids = ids.contiguous()
        d.ids, d.ids_stride = ids.data_ptr(), n if ids.dim() == 2 else 0
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=dev)
    elif out.shape != (B,) or out.dtype != torch.int64 or out.device != dev \
            or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous [{B}] int64 tensor on {dev}")
    prob = torch.empty(B, dtype=f32, device=dev) if return_prob else None
    if B:
        with torch.cuda.device(dev):
            _lib.call("fh_sample_logits", logits.data_ptr(), _lib.dtype_code(logits.dtype), B, n,
                      max(logits.stride(0), n), ctypes.byref(d), out.data_ptr(),
                      None if prob is None else prob.data_ptr(), _lib.stream_ptr())
    return (out, prob) if return_prob else out
