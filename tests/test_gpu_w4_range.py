"""Dense 4-bit logits over the range of scales and hidden states, and the same
for every number of rows.

Tolerance. The products (q - z) * h are exact; a group's fp32 sum and the groups'
scaled sums are at most group / 16 + G + 16 additions, each off by 2^-22 of
A = sum |w| |h| at worst. Calls of more than 8 rows with groups below 128 sum the
exact products of a weight's two parts instead, 16 columns at a time: D / 8
additions (of which an accumulator sees half). Then one rounding to the output type, half a step. Nothing is rounded
to 16 bits before that.
"""

from __future__ import annotations

import pytest
import torch

from flash_head.w4 import W4Weight, w4_logits

pytestmark = pytest.mark.gpu

ROWS = (1, 8, 9, 16, 17, 33, 64, 65, 97, 128, 129, 200, 256)


def weight(V, D, group, zeros, dtype, seed, scale):
    """Random nibbles (and zero points) under the given scales [V, groups]."""
    g = torch.Generator().manual_seed(seed)
    v = torch.randint(0, 16, (V, D), generator=g, dtype=torch.uint8)
    z = torch.randint(0, 16, (V, D // group), generator=g, dtype=torch.uint8) if zeros else None
    return v, scale.to(dtype), z


def build(v, s, z):
    q = v[:, 0::2] | (v[:, 1::2] << 4)
    w = W4Weight.from_quantized(q.cuda(), s.cuda(), None if z is None else z.cuda())
    group = v.shape[1] // s.shape[1]
    x = v.double().view(v.shape[0], -1, group) - (8.0 if z is None else z.double().unsqueeze(2))
    return w, (x * s.double().unsqueeze(2)).view(v.shape).cuda(), group


def check(got, h, W, group, rows=None):
    """rows: of the call, when h holds some of them."""
    hd = h.double()
    want, mag = hd @ W.t(), hd.abs() @ W.abs().t()
    info = torch.finfo(h.dtype)
    # below the smallest normal number a step no longer shrinks with the value
    D = h.shape[1]
    adds = D / 8 if (rows or h.shape[0]) > 8 and group < 128 else group / 16 + D / group + 16
    tol = info.eps / 2 * want.abs().clamp_min(info.tiny) + adds * 2.0 ** -22 * mag
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), float((err / tol).max()))


def hidden(T, D, dtype, seed):
    g = torch.Generator().manual_seed(900 + seed)
    return torch.randn(T, D, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,D,group,zeros", [
    (700, 1024, 128, True), (700, 1024, 128, False), (389, 1056, 32, True), (1500, 576, 64, True)])
def test_no_weight_is_rounded(V, D, group, zeros, dtype):
    """Every number of rows has the row product's error."""
    g = torch.Generator().manual_seed(D)
    s = 0.002 + 0.02 * torch.rand(V, D // group, generator=g)
    w, W, group = build(*weight(V, D, group, zeros, dtype, V, s))
    for T in ROWS:
        h = hidden(T, D, dtype, T).cuda()
        check(w4_logits(h, w), h, W, group)


@pytest.mark.parametrize("T", [8, 9, 40, 100])
@pytest.mark.parametrize("dtype,span", [(torch.bfloat16, 40), (torch.float16, 14)])
def test_scales_far_apart(T, dtype, span):
    """The groups' scales fall by 2^span within a row, and the hidden states
    that meet them grow as much: every group has its share of the logit."""
    V, D, group = 300, 1024, 64
    G = D // group
    fall = torch.linspace(0, span, G).round()
    g = torch.Generator().manual_seed(3)
    s = (1.0 + torch.rand(V, G, generator=g)) * 2.0 ** -fall
    if dtype == torch.float16:
        s = s * 0.25
    w, W, group = build(*weight(V, D, group, True, dtype, 5, s))
    h = (hidden(T, D, torch.float32, T) * 0.25).view(T, G, group)
    h = (h * (2.0 ** fall).view(1, G, 1)).view(T, D).to(dtype).cuda()
    check(w4_logits(h, w), h, W, group)


@pytest.mark.parametrize("T", [8, 9, 40, 100])
def test_hidden_states_far_apart(T):
    """A hidden state 2^50 times its row's others meets weights of zero: the
    others alone are the logit."""
    V, D, group = 300, 512, 128
    v, s, z = weight(V, D, group, False, torch.bfloat16, 7, torch.full((V, D // group), 0.01))
    v[:, 200] = 8
    w, W, group = build(v, s, z)
    h = hidden(T, D, torch.float32, T)
    h[:, 200] = 2.0 ** 50
    h = h.to(torch.bfloat16).cuda()
    got = w4_logits(h, w)
    check(got, h, W, group)
    assert (got != 0).float().mean() > 0.99


@pytest.mark.parametrize("T", [8, 9, 40])
@pytest.mark.parametrize("top", [1.5 * 2.0 ** -128, 2.0 ** -133, 2.0 ** 100])
def test_smallest_and_largest_scales(T, top):
    """Rows whose largest scale is a subnormal bf16 number, and large ones,
    next to hidden states of the other end: neither NaN nor zero."""
    V, D, group = 130, 256, 128
    s = torch.full((V, D // group), top, dtype=torch.float64).to(torch.bfloat16)
    w, W, group = build(*weight(V, D, group, True, torch.bfloat16, 9, s))
    h = (hidden(T, D, torch.float32, T) * (2.0 ** 60 if top < 1 else 2.0 ** -100))
    h = h.to(torch.bfloat16).cuda()
    check(w4_logits(h, w), h, W, group)


@pytest.mark.parametrize("T", [8, 9, 70])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype,top,small", [
    (torch.float16, 60000.0, 2.0 ** -12), (torch.bfloat16, 2.0 ** 126, 2.0 ** -126)])
def test_weights_beyond_the_largest_number(dtype, top, small, group, T):
    """15 times the scale is no number of the type; the logits are."""
    V, D = 200, 256
    s = torch.full((V, D // group), top, dtype=torch.float64)
    s[::2] = 1.0
    w, W, group = build(*weight(V, D, group, True, dtype, 11, s))
    h = (hidden(T, D, torch.float32, T) * small).to(dtype).cuda()
    check(w4_logits(h, w), h, W, group)


@pytest.mark.parametrize("T", [3, 9, 40, 140])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_infinite_hidden_states(group, dtype, T):
    """An infinite hidden state makes infinite logits of the weight's sign, and NaN
    where its weight is zero; other rows are as they were."""
    V, D = 300, 256
    g = torch.Generator().manual_seed(5)
    s = 0.002 + 0.02 * torch.rand(V, D // group, generator=g)
    w, W, group = build(*weight(V, D, group, True, dtype, 13, s))
    h = hidden(T, D, dtype, T).cuda()
    h[1, 77], h[2, 200] = float("inf"), float("-inf")
    got = w4_logits(h, w)
    for r, k in ((1, 77), (2, 200)):
        want = W[:, k] * h[r, k].double()
        assert want.isnan().any() and want.isinf().any()
        assert torch.equal(got[r].isnan(), want.isnan())
        assert torch.equal(got[r][~want.isnan()].double(), want[~want.isnan()])
    keep = [r for r in range(T) if r not in (1, 2)]
    check(got[keep], h[keep], W, group, rows=T)
