"""Filtered sampling where the draw lies at an end of the row: every row's id
and probability are written, and are the definition's in 64 bits.

An entry counts while e_i is a 64-bit number well above the smallest (the rows
here stay above 2^-1000 of the largest), so u = 0 takes the first kept column
however small its mass. Ids must be equal; the probability is rounded once, to
fp32 (see test_gpu_sampling.py for the 64-bit errors).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from flash_head.sampling import sample_logits
from test_gpu_sampling import logits, oracle_row

pytestmark = pytest.mark.gpu

LAST = 1.0 - 2.0 ** -53


def check(x, u, T=1.0, k=0, p=1.0, m=0.0, alike=False):
    """alike: every row has the same logits and the same u."""
    B = x.shape[0]
    out = torch.full((B,), -77, dtype=torch.int64, device="cuda")
    got, prob = sample_logits(x, u, T, k, p, m, out=out, return_prob=True)
    f32 = [np.float64(np.float32(v)) for v in (T, p, m)]
    some = 1 if alike else B
    xn, un = x[:some].float().cpu().double().numpy(), u.cpu().numpy()
    want = [oracle_row(xn[r], un[r], f32[0], k, f32[1], f32[2]) for r in range(some)]
    want *= B // some
    cols = np.array([c for c, _ in want])
    assert np.array_equal(got.cpu().numpy(), cols), \
        [(int(r), int(got[r]), int(cols[r])) for r in np.flatnonzero(got.cpu().numpy() != cols)[:8]]
    pw = np.array([q for _, q in want])
    assert (np.abs(prob.cpu().double().numpy() - pw) <= pw * (2.0 ** -24 + 2.0 ** -40) + 1e-40).all()


def ends(B):
    """u = 0 and the largest below 1, by turns."""
    return torch.tensor([0.0, LAST], dtype=torch.float64, device="cuda").repeat(B)[:B]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,n", [(2, 128256), (8, 40000), (300, 20000)])
@pytest.mark.parametrize("bits", [60, 80, 300, 800, 940])
def test_a_first_stretch_far_below_the_largest(B, n, bits, dtype):
    """The first eighth of the row lies `bits` binary orders below its largest."""
    T = 0.5
    x = logits(B, n, dtype, 5, sigma=0.5, peak=False)
    x[:, n // 8:] += bits * T * 0.6931472
    u = ends(B)
    check(x, u, T=T)
    check(x, u, T=T, m=1e-30)
    check(x, u, T=T, k=n - 5)
    check(x, u, T=T, p=0.9999999)


@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, LAST])
def test_a_kept_entry_far_below_the_largest(u):
    """Short rows: the list of the candidates has the same rule."""
    B = 4
    for n in (50, 3000, 9000):
        x = torch.full((B, n), float("-inf"))
        x[:, 3] = -120.0
        x[:, n // 2] = 5.0
        x[:, n - 2] = 4.0
        x = x.cuda()
        uu = torch.full((B,), u, dtype=torch.float64, device="cuda")
        for kw in ({}, {"k": 3}, {"k": 2}, {"p": 0.999}, {"T": 0.25, "k": 3}):
            check(x, uu, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("left", [1, 3, 2100 * 8, 60000])
def test_a_masked_tail_of_a_long_segment(left, dtype):
    """One CTA per row, so that a warp's segment is walked in several pieces;
    the row's last entries are masked, and u is at its end."""
    B, n = 300, 151936
    x = logits(B, n, dtype, 8, sigma=1.5, peak=False)
    x[:, left:] = float("-inf")
    u = torch.full((B,), LAST, dtype=torch.float64, device="cuda")
    check(x, u)
    check(x, u, m=1e-6)
    check(x, torch.full_like(u, 1.5))


@pytest.mark.parametrize("B,n", [(1, 151936), (300, 151936), (3, 128256)])
@pytest.mark.parametrize("T,low,top", [
    (0.1, 1.6745601, 9.715551), (0.1, 1.0, 9.3), (0.05, -3.0, 1.2), (0.2, 0.0, 17.0),
    (1.0, 0.0, 80.0), (1.0, -20.0, 10.0)])
def test_top_p_next_to_a_border_at_low_temperatures(B, n, T, low, top):
    """A few equal logits hold all the mass, and top_p is the next number above
    (below) the share of some of them: the cut is decided exactly. (Where top_p is
    that share, the others' mass decides, which is above 0 and less than a step of
    64 bits: one entry more by the definition, none more by its sums in 64 bits.)"""
    for count, kept in ((2, 1), (4, 2), (8, 2), (8, 4)):
        x = torch.full((1, n), low)
        x[:, ::3] -= 1.0
        x[:, [17 + i * (n // count) + 5 * i for i in range(count)]] = top
        x = x.cuda().repeat(B, 1)
        share = np.float32(kept / count)
        for p in (np.nextafter(share, np.float32(1)), share, np.nextafter(share, np.float32(0))):
            for u in (0.2, 0.99):
                uu = torch.full((B,), u, dtype=torch.float64, device="cuda")
                if p != share:
                    check(x, uu, T=T, p=float(p), alike=True)
                    continue
                got, prob = sample_logits(x, uu, T, top_p=float(p), return_prob=True)
                some = [c for c in (kept, kept + 1) if abs(float(prob[0]) * c - 1) < 1e-6]
                assert some and (prob == prob[0]).all()
                assert (got == x[0].topk(count).indices.sort().values[int(u * some[0])]).all()


@pytest.mark.parametrize("B,n", [(1, 151936), (40, 151936), (300, 151936)])
@pytest.mark.parametrize("T,low,top", [
    (0.1, 1.6745601, 9.715551), (0.1, 1.1, 9.6), (0.07, -3.1, 2.4), (0.2, 0.3, 17.1),
    (1.0, 0.7, 83.1), (0.9, -20.3, 30.2), (0.1, 1.6745601, 5.1), (0.05, 2.3, 4.7)])
def test_top_p_above_what_a_sample_shows(B, n, T, low, top):
    """The few logits that hold the mass lie between the vectors that the kernel
    samples for its reference, up to 127 binary orders above it."""
    g = torch.Generator().manual_seed(2)
    base = low - 0.5 * torch.rand(1, n, generator=g)
    base[0, 0] = low
    for count, kept in ((2, 1), (4, 2), (8, 2), (8, 4)):
        x = base.clone()
        x[:, [17 + i * (n // count) + 5 * i for i in range(count)]] = top
        x = x.cuda().repeat(B, 1)
        share = np.float32(kept / count)
        for p in (np.nextafter(share, np.float32(1)), np.nextafter(share, np.float32(0))):
            for u in (0.2, 0.99):
                uu = torch.full((B,), u, dtype=torch.float64, device="cuda")
                check(x, uu, T=T, p=float(p), alike=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,n", [(2, 128256), (300, 40000)])
@pytest.mark.parametrize("T,level", [(1.0, -30.0), (1.0, -80.0), (0.1, -90.0), (1.0, -2000.0)])
def test_masked_beginnings_and_logits_far_below_zero(B, n, T, level, dtype):
    """Log-probabilities, and a mask over the first entries of every warp's
    segment: what is left lies far from the 0 that a mask leaves as a reference."""
    x = logits(B, n, dtype, 6, sigma=1.0, peak=False) + level
    segments = 64 if B == 2 else 8
    at = torch.arange(n, device="cuda") % (n // segments)
    x[:, at < 400] = float("-inf")
    g = torch.Generator().manual_seed(4)
    u = torch.rand(B, generator=g, dtype=torch.float64).cuda()
    check(x, u, T=T)
    check(x, torch.zeros_like(u), T=T)
    # At 1 - 2^-53 the mass behind the draw is no more than the rounding of the
    # sums (n of them, half a step each): any of the columns there will do.
    got = sample_logits(x, torch.full_like(u, LAST), T,
                        out=torch.full((B,), -77, dtype=torch.int64, device="cuda"))
    e = torch.exp((x.double() - x.double().amax(1, keepdim=True)) / float(np.float32(T)))
    share = (e.cumsum(1) / e.sum(1, keepdim=True)).gather(1, got.clamp_min(0).view(B, 1))
    assert (got >= 0).all() and (share >= 1 - n * 2.0 ** -52).all()
    assert (x.gather(1, got.view(B, 1)) > float("-inf")).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,n", [(3, 1580), (2, 4217), (5, 9000), (2, 150000)])
def test_nan_masks_where_the_cut_descends_by_keys(B, n, dtype):
    """A top-k beyond the list of candidates, or a cut among thousands of equal
    logits: a NaN is not counted among the entries above it, whatever its bits."""
    x = logits(B, n, torch.float32, 9, sigma=1.0, peak=False)
    gone = torch.rand(B, n, generator=torch.Generator().manual_seed(5)).cuda() < 0.3
    left = int((~gone).sum(1).min())
    u = torch.rand(B, generator=torch.Generator().manual_seed(6), dtype=torch.float64).cuda()
    for y in (x, x.round()):
        y = y.to(dtype)
        bits = y.view(torch.int16 if dtype != torch.float32 else torch.int32)
        for negative in (True, False):
            y[gone] = float("nan")
            if negative:
                bits[gone] = -1  # every bit set
            for k in (1025, left - 1, left, left + 1, n - 1):
                check(y, u, T=2.0, k=k)
                check(y, u, T=2.0, k=k, p=0.9)
            check(y, u, T=50.0, p=0.7)
            check(y, u, T=2.0, p=0.7, m=1e-3)
