"""The 4-bit products and the sampler at the same time on several streams, and
over and over: every call gives the bits that it gives alone."""

from __future__ import annotations

import pytest
import torch

from flash_head.sampling import sample_logits
from flash_head.w4 import W4Weight, w4_block_sparse_logits, w4_logits

pytestmark = pytest.mark.gpu


def make(V, D, group, zeros, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=g) * 0.02).to(dtype).cuda()
    return W4Weight.from_dense(w, group, zeros)


def hidden(T, D, dtype, seed):
    return torch.randn(T, D, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def jobs():
    a = make(30000, 1024, 128, True, torch.bfloat16, 1)
    b = make(20008, 1536, 64, False, torch.float16, 2)
    c = make(9000, 800, 32, True, torch.bfloat16, 3)
    ci = torch.randperm(500, generator=torch.Generator().manual_seed(4))[:96].view(1, 96).cuda()
    x = (torch.randn(40, 60000, generator=torch.Generator().manual_seed(5)) * 3).cuda()
    u = torch.rand(40, generator=torch.Generator().manual_seed(6), dtype=torch.float64).cuda()
    calls = []
    for T in (9, 64, 130):
        h = hidden(T, 1024, torch.bfloat16, T)
        calls.append(lambda h=h: w4_logits(h, a))
        h = hidden(T, 1536, torch.float16, T)
        calls.append(lambda h=h: w4_logits(h, b))
        h = hidden(T, 800, torch.bfloat16, T)
        calls.append(lambda h=h: w4_logits(h, c))
    h5 = hidden(5, 1024, torch.bfloat16, 5)
    calls.append(lambda: w4_logits(h5, a))
    calls.append(lambda: w4_block_sparse_logits(h5[:1], a, ci, 500, 16))
    calls.append(lambda: sample_logits(x, u, 0.9, 50, 0.95))
    calls.append(lambda: sample_logits(x, u, 1.1, None, 0.9))
    calls.append(lambda: sample_logits(x, u))
    return calls


def test_streams_at_the_same_time():
    calls = jobs()
    alone = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for r in range(12):
        for i, f in enumerate(calls):
            with torch.cuda.stream(streams[(i + r) % 4]):
                got.append((i, f()))
    torch.cuda.synchronize()
    for i, out in got:
        assert torch.equal(out, alone[i]), i


def test_over_and_over():
    calls = jobs()
    alone = [f() for f in calls]
    for r in range(60):
        bad = [i for i, f in enumerate(calls) if not torch.equal(f(), alone[i])]
        assert not bad, (r, bad)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_number_of_rows(group):
    """1 .. 140 and a few beyond: each row's logits are those of the row in
    another call of more than 8 rows, up to the rounding of the output."""
    V, D = 777, 384
    w = make(V, D, group, True, torch.bfloat16, group)
    h = hidden(300, D, torch.bfloat16, 1)
    want = h.double() @ w.dequantize().double().t()
    mag = h.double().abs() @ w.dequantize().double().abs().t()
    # at most D / 8 + 16 fp32 additions of 2^-22, and one rounding (half a step)
    tol = torch.finfo(torch.bfloat16).eps / 2 * want.abs() + (D / 8 + 16) * 2.0 ** -22 * mag
    for T in list(range(1, 141)) + [255, 256, 257, 300]:
        out = torch.full((T, V), 50.0, dtype=torch.bfloat16, device="cuda")
        w4_logits(h[:T], w, out=out)
        assert ((out.double() - want[:T]).abs() <= tol[:T]).all(), T
