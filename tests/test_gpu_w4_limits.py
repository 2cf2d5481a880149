"""The bounded waits of the 4-bit many-row kernels: a wait that runs out ends the
call with NaN logits and a bit in the workspace, never with other numbers, and
leaves nothing behind."""

from __future__ import annotations

import ctypes

import pytest
import torch

from flash_head import _lib
from flash_head.sampling import sample_logits
from flash_head.w4 import W4Weight, w4_logits

pytestmark = pytest.mark.gpu


@pytest.fixture
def polls():
    lib = _lib.load_library()
    default = lib.fh_w4_wait_polls(1 << 18)
    assert default == 1 << 18
    yield lib.fh_w4_wait_polls
    lib.fh_w4_wait_polls(default)


def call(w, h):
    """Logits and the workspace's first word."""
    lib = _lib.load_library()
    T = h.shape[0]
    need = lib.fh_w4_workspace_bytes(ctypes.byref(w.desc), T)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((T, w.vocab), 3.0, dtype=h.dtype, device="cuda")
    _lib.call("fh_w4_logits", ctypes.byref(w.desc), h.data_ptr(), T, out.data_ptr(), w.vocab,
              ws.data_ptr(), need, _lib.stream_ptr())
    return out, int(ws[:4].view(torch.int32))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T", [9, 64, 200])
def test_a_wait_that_gives_up(group, T, polls):
    g = torch.Generator().manual_seed(group + T)
    V, D = 5000, 1024
    W = (torch.randn(V, D, generator=g) * 0.02).bfloat16().cuda()
    w = W4Weight.from_dense(W, group, zeros=True)
    h = torch.randn(T, D, generator=g).bfloat16().cuda()
    want, word = call(w, h)
    assert word == 0 and want.isfinite().all()
    polls(0)
    out, word = call(w, h)
    assert word & 2 and out.isnan().all()
    # through Python: NaN, which the sampler takes for masked
    x = w4_logits(h, w)
    assert x.isnan().all()
    u = torch.full((T,), 0.5, dtype=torch.float64, device="cuda")
    assert (sample_logits(x, u) == -1).all()
    polls(1 << 18)
    out, word = call(w, h)
    assert word == 0 and torch.equal(out, want)


@pytest.mark.parametrize("group", [64, 128])
def test_a_wait_that_gives_up_midway(group, polls):
    """With a few polls some CTAs get further than others: what is not NaN is right."""
    g = torch.Generator().manual_seed(group)
    W = (torch.randn(40000, 512, generator=g) * 0.02).bfloat16().cuda()
    w = W4Weight.from_dense(W, group)
    h = torch.randn(40, 512, generator=g).bfloat16().cuda()
    want, _ = call(w, h)
    for n in (1, 4, 16):
        polls(n)
        out, word = call(w, h)
        gone = out.isnan()
        assert bool(gone.any()) == bool(word & 2)
        assert torch.equal(out[~gone], want[~gone])
    polls(1 << 18)
    assert torch.equal(call(w, h)[0], want)
