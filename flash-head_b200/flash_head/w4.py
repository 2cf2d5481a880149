"""A head weight in 4 bits with group scales, and its products.

    W4Weight.from_dense(weight, group_size=128)       quantise [V, D] bf16/fp16
    W4Weight.from_quantized(q, scales, zeros=None)    a 4-bit checkpoint
    w4_logits(hs, w)                                  [T, V] logits
    w4_block_sparse_logits(hs, w, ci, n_clusters, cluster_size)
                                                      [T, P*cap] logits of probed clusters

w[v, k] = (q[v, k] - z[v, g]) * s[v, g], q in 0..15, one scale (and zero point;
8 without zero points) per group g = k // group_size of a row. The kernels
(``csrc/fh_w4.cuh``) sum exact products of q - z and the hidden states in fp32
and scale each group's sum in fp32; results are rounded once, to the hidden
states' dtype. ``w4_logits`` of more than 8 rows runs on ``csrc/fh_w4_tc.cuh`` or
``csrc/fh_w4_split.cuh``, which sum the same products in another order.
``w4_block_sparse_logits`` is the 4-bit form of
``flash_head.fused.block_sparse_logits`` (reference
``src/flash_head/fused.py:82-93``).
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib

GROUP_SIZES = (32, 64, 128)
MAX_HIDDEN = 12288
_BLOCK = 128       # columns per layout block
_ROWS = 128        # rows per layout tile (the last one is padded)
_CHUNK = 1 << 27   # elements unpacked at a time while laying out


def _check_groups(D: int, group_size: int):
    if group_size not in GROUP_SIZES:
        raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {group_size}")
    if D <= 0 or D % group_size:
        raise ValueError(f"hidden size {D} is not a multiple of group_size {group_size}")
    if D > MAX_HIDDEN:
        raise ValueError(f"hidden size {D} exceeds {MAX_HIDDEN}")


def _pack_words(q: torch.Tensor, nb: int) -> torch.Tensor:
    """[R, D] uint8 values (R a multiple of 128) -> int32 [R/128, nb, 4, 128, 4] words."""
    R, D = q.shape
    if D < nb * _BLOCK:
        q = torch.nn.functional.pad(q, (0, nb * _BLOCK - D), value=8)
    # tile, block, quad, row, word, e
    x = q.view(R // _ROWS, _ROWS, nb, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)
    w = torch.zeros(x.shape[:-1], dtype=torch.int32, device=q.device)
    for e in range(8):
        w |= x[..., e].to(torch.int32) << (4 * (e // 2) + 16 * (e % 2))
    return w.contiguous()


def _unpack_words(w: torch.Tensor, D: int) -> torch.Tensor:
    """The inverse of ``_pack_words``: int32 [t, nb, 4, 128, 4] -> [128 t, D] uint8."""
    x = torch.stack([(w >> (4 * (e // 2) + 16 * (e % 2))) & 15 for e in range(8)], dim=-1)
    t, nb = w.shape[0], w.shape[1]
    x = x.permute(0, 3, 1, 4, 2, 5).reshape(_ROWS * t, nb * _BLOCK)
    return x[:, :D].to(torch.uint8)


def _pack_groups(x: torch.Tensor, V_pad: int, nb: int, gpk: int, fill) -> torch.Tensor:
    """[V, G] per-group values -> [V_pad/128, nb, 128, gpk], padding = fill."""
    V, G = x.shape
    out = torch.full((V_pad, nb * gpk), fill, dtype=x.dtype, device=x.device)
    out[:V, :G] = x
    return out.view(V_pad // _ROWS, _ROWS, nb, gpk).permute(0, 2, 1, 3).contiguous()


class W4Weight:
    """A [V, D] head weight in 4 bits, in the kernels' layout.

    Made by ``from_dense`` or ``from_quantized``; holds ``qweight``, ``scales``
    and ``zeros`` (or None) on one CUDA device (or on the CPU until ``to``)."""

    def __init__(self, qweight, scales, zeros, vocab: int, hidden: int, group_size: int):
        self.qweight, self.scales, self.zeros = qweight, scales, zeros
        self.vocab, self.hidden, self.group_size = int(vocab), int(hidden), int(group_size)
        d = _lib.W4Desc()
        d.vocab, d.hidden, d.group_size = self.vocab, self.hidden, self.group_size
        d.dtype = _lib.dtype_code(scales.dtype)
        d.qweight, d.scales = qweight.data_ptr(), scales.data_ptr()
        d.zeros = None if zeros is None else zeros.data_ptr()
        # rows whose weights may pass the type's largest number, brought down by 2^-4
        top = scales.float().abs().amax(dim=(1, 3)).view(-1)
        limit = 2.0 ** (12 if scales.dtype == torch.float16 else 124)
        self.row_mul = torch.where(torch.isfinite(top) & (top > limit), 2.0 ** -4, 1.0)
        d.row_mul = self.row_mul.data_ptr()
        self.desc, self.ref = d, ctypes.byref(d)

    def __reduce__(self):  # copies and pickles hold no addresses
        return W4Weight, (self.qweight, self.scales, self.zeros, self.vocab, self.hidden,
                          self.group_size)

    # -- making one ----------------------------------------------------------
    @classmethod
    def from_quantized(cls, q: torch.Tensor, scales: torch.Tensor,
                       zeros: Optional[torch.Tensor] = None) -> "W4Weight":
        """q [V, D/2] uint8 (column 2i in the low, 2i+1 in the high nibble of
        byte i), scales [V, D/group_size] bf16 or fp16, zeros the same shape
        uint8 in 0..15 (None: 8 everywhere)."""
        if q.dim() != 2 or q.dtype != torch.uint8:
            raise ValueError(f"q must be a 2-D uint8 tensor, got {tuple(q.shape)} {q.dtype}")
        if scales.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"scales must be bf16 or fp16, got {scales.dtype}")
        V, D = q.shape[0], 2 * q.shape[1]
        if V == 0 or scales.dim() != 2 or scales.shape[0] != V or scales.shape[1] == 0 \
                or D % scales.shape[1]:
            raise ValueError(f"scales {tuple(scales.shape)} do not fit q {tuple(q.shape)}")
        group = D // scales.shape[1]
        _check_groups(D, group)
        if scales.device != q.device:
            raise ValueError("q and scales are on different devices")
        if zeros is not None:
            if zeros.shape != scales.shape or zeros.dtype != torch.uint8 \
                    or zeros.device != q.device:
                raise ValueError("zeros must be uint8 on q's device in the shape of scales")
            if int(zeros.max()) > 15:
                raise ValueError("zero points must be in 0..15")
        nb, gpk = -(-D // _BLOCK), _BLOCK // group
        V_pad = -(-V // _ROWS) * _ROWS
        with torch.no_grad():
            qw = torch.empty((V_pad // _ROWS, nb, 4, _ROWS, 4), dtype=torch.int32, device=q.device)
            step = max(_ROWS, _CHUNK // (nb * _BLOCK) // _ROWS * _ROWS)
            for lo in range(0, V_pad, step):
                n = min(step, V_pad - lo)
                part = q[lo:min(V, lo + n)]
                x = torch.full((n, D), 8, dtype=torch.uint8, device=q.device)
                x[:part.shape[0], 0::2] = part & 15
                x[:part.shape[0], 1::2] = part >> 4
                qw[lo // _ROWS:(lo + n) // _ROWS] = _pack_words(x, nb)
            s = _pack_groups(scales, V_pad, nb, gpk, 0.0)
            z = None if zeros is None else _pack_groups(zeros, V_pad, nb, gpk, 8)
        return cls(qw, s, z, V, D, group)

    @classmethod
    def from_dense(cls, weight: torch.Tensor, group_size: int = 128,
                   zeros: bool = False) -> "W4Weight":
        """Round-to-nearest quantisation of a [V, D] bf16 or fp16 weight.

        Without zero points a group's scale is its largest magnitude / 7; with
        them the group's range (0 included) is spread over 0..15. Scales are
        held in the weight's dtype, at least its smallest normal number, and
        weights are rounded against the held scale. The weight has to be finite."""
        if weight.dim() != 2 or weight.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"weight must be a 2-D bf16 or fp16 tensor, got "
                             f"{tuple(weight.shape)} {weight.dtype}")
        V, D = weight.shape
        _check_groups(D, group_size)
        tiny = torch.finfo(weight.dtype).tiny
        qs, ss, zs = [], [], []
        step = max(1, _CHUNK // D)
        with torch.no_grad():
            for lo in range(0, V, step):
                x = weight[lo:lo + step].float().view(-1, D // group_size, group_size)
                if zeros:
                    low = x.amin(dim=2).clamp_max(0.0)
                    high = x.amax(dim=2).clamp_min(0.0)
                    s = ((high - low) / 15.0).clamp_min(tiny).to(weight.dtype)
                    z = (-low / s.float()).round_().clamp_(0, 15)
                else:
                    s = (x.abs().amax(dim=2) / 7.0).clamp_min(tiny).to(weight.dtype)
                    z = torch.full_like(s, 8.0, dtype=torch.float32)
                if not bool(torch.isfinite(s).all()):
                    raise ValueError("the weight holds numbers that are not finite, or a group "
                                     "whose range is not")
                q = (x / s.float().unsqueeze(2)).round_() + z.unsqueeze(2)
                q = q.clamp_(0, 15).to(torch.uint8).view(-1, D)
                qs.append(q[:, 0::2] | (q[:, 1::2] << 4))
                ss.append(s)
                zs.append(z.to(torch.uint8))
        return cls.from_quantized(torch.cat(qs), torch.cat(ss), torch.cat(zs) if zeros else None)

    # -- reading one ---------------------------------------------------------
    @property
    def shape(self):
        return torch.Size((self.vocab, self.hidden))

    @property
    def dtype(self):
        return self.scales.dtype

    @property
    def device(self):
        return self.qweight.device

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size()
                   for t in (self.qweight, self.scales, self.zeros) if t is not None)

    def to(self, device) -> "W4Weight":
        """This weight on another device (itself if it is there already)."""
        device = torch.device(device)
        if self.device == device or (device.type == "cuda" and device.index is None
                                     and self.device.type == "cuda"):
            return self
        z = None if self.zeros is None else self.zeros.to(device)
        return W4Weight(self.qweight.to(device), self.scales.to(device), z, self.vocab,
                        self.hidden, self.group_size)

    def dequantize(self) -> torch.Tensor:
        """[V, D] fp32 (q - z) * s."""
        G = self.hidden // self.group_size

        def rows(x):  # [tiles, nb, 128, gpk] -> [V, G]
            return x.permute(0, 2, 1, 3).reshape(-1, x.shape[1] * x.shape[3])[:self.vocab, :G]
        q = _unpack_words(self.qweight, self.hidden)[:self.vocab].float()
        q = q.view(self.vocab, G, self.group_size)
        z = 8.0 if self.zeros is None else rows(self.zeros).float().unsqueeze(2)
        return ((q - z) * rows(self.scales).float().unsqueeze(2)).view(self.vocab, self.hidden)

    def __repr__(self):
        return (f"W4Weight(vocab={self.vocab}, hidden={self.hidden}, group_size="
                f"{self.group_size}, zeros={self.zeros is not None}, dtype={self.dtype}, "
                f"device={self.device})")


def _check(hs: torch.Tensor, w: W4Weight) -> torch.Tensor:
    if not hs.is_cuda or not w.qweight.is_cuda:
        raise RuntimeError("FlashHead kernels need CUDA tensors (there is no CPU path)")
    if hs.dim() != 2 or hs.shape[1] != w.hidden:
        raise ValueError(f"hidden states must be [T, {w.hidden}], got {tuple(hs.shape)}")
    if hs.dtype != w.dtype:
        raise ValueError(f"hidden dtype {hs.dtype} != weight scale dtype {w.dtype}")
    if hs.device != w.device:
        raise ValueError(f"hidden states on {hs.device}, weight on {w.device}")
    hs = hs.contiguous()
    return hs if hs.data_ptr() % 16 == 0 else hs.clone()


def w4_logits(hs: torch.Tensor, w: W4Weight, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[T, D] hidden states -> [T, V] logits in their dtype.

    ``out`` may be any [T, V] tensor of that dtype with contiguous rows. Should one
    of the kernels' bounded waits run out (more than 8 rows; none does on a GPU that
    works), the logits that depend on it are NaN, which ``sample_logits`` takes for
    masked: -1 for a row without any other."""
    hs = _check(hs, w)
    T = hs.shape[0]
    if out is None:
        out = torch.empty((T, w.vocab), dtype=hs.dtype, device=hs.device)
    elif out.shape != (T, w.vocab) or out.dtype != hs.dtype or out.device != hs.device \
            or (T > 0 and out.stride(1) != 1 and w.vocab > 1) or (T > 1 and out.stride(0) < w.vocab):
        raise ValueError(f"out must be a [{T}, {w.vocab}] {hs.dtype} tensor on {hs.device} with "
                         "contiguous rows")
    if T == 0:
        return out
    lib = _lib.load_library()
    with _lib.on_device(hs.device) as stream:
        need = lib.fh_w4_workspace_bytes(w.ref, T)
        ws = torch.empty(need, dtype=torch.uint8, device=hs.device) if need else None
        st = lib.fh_w4_logits(w.ref, hs.data_ptr(), T, out.data_ptr(),
                              max(out.stride(0), w.vocab),
                              None if ws is None else ws.data_ptr(), need, stream)
    _lib.check("fh_w4_logits", st)
    return out


def w4_block_sparse_logits(hs: torch.Tensor, w: W4Weight, ci: torch.Tensor, n_clusters: int,
                           cluster_size: int) -> torch.Tensor:
    """[T, P * cluster_size] logits of each row's probed clusters ``ci`` [T, P]
    int64, weight row = cluster * cluster_size + slot. A cluster id outside
    [0, n_clusters) gives -inf."""
    hs = _check(hs, w)
    if ci.dim() != 2 or ci.dtype != torch.int64 or ci.shape[0] != hs.shape[0]:
        raise ValueError(f"ci must be int64 [{hs.shape[0]}, P], got {tuple(ci.shape)} {ci.dtype}")
    if ci.device != hs.device:
        raise ValueError(f"ci on {ci.device}, hidden states on {hs.device}")
    T, P = ci.shape
    ci = ci.contiguous()
    out = torch.empty((T, P * int(cluster_size)), dtype=hs.dtype, device=hs.device)
    lib = _lib.load_library()
    with _lib.on_device(hs.device) as stream:
        st = lib.fh_w4_block_sparse_logits(w.ref, hs.data_ptr(), T, ci.data_ptr(), P,
                                           int(n_clusters), int(cluster_size), out.data_ptr(),
                                           stream)
    _lib.check("fh_w4_block_sparse_logits", st)
    return out
