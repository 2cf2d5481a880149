"""Products with a 4-bit head weight on the GPU against their definition in
64 bits.

Tolerance. The products (q - z) * h are exact in fp32. A group's sum is a chain
of group/16 tensor-core steps, the groups' scaled sums another chain, and up to
16 warps' partial sums are added: at most group/16 + G + 16 additions, each of
which rounds (or truncates) a partial sum of magnitude at most
A = sum |w| |h| by 2^-22 relative at worst. Then one rounding to the output
type: half a step, eps / 2 relative.

Dense calls of more than 8 rows round each weight to f16: half a step, 2^-11
relative. The hidden states are symmetric around 0 and independent, so the
errors e_k w_k h_k, |e_k| <= 2^-11, are independent, have mean 0 and are bounded
by b_k = 2^-11 |w_k h_k|: by Hoeffding's inequality their sum passes
t = 7 sqrt(sum b_k^2) with a probability below 2 exp(-t^2 / (2 sum b_k^2)) =
5e-11, 5e-4 over 10^7 outputs.
"""

from __future__ import annotations

import pytest
import torch

from flash_head.w4 import W4Weight, w4_block_sparse_logits, w4_logits

pytestmark = pytest.mark.gpu


def make_weight(V, D, group, zeros, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (V, D // 2), generator=g, dtype=torch.uint8)
    s = (0.002 + 0.02 * torch.rand(V, D // group, generator=g)).to(dtype)
    z = torch.randint(0, 16, (V, D // group), generator=g, dtype=torch.uint8) if zeros else None
    w = W4Weight.from_quantized(q.cuda(), s.cuda(), None if z is None else z.cuda())
    v = torch.empty(V, D, dtype=torch.float64)
    v[:, 0::2] = (q & 15).double()
    v[:, 1::2] = (q >> 4).double()
    v = v.view(V, -1, group) - (8.0 if z is None else z.double().unsqueeze(2))
    return w, (v * s.double().unsqueeze(2)).view(V, D).cuda()


def make_hidden(T, D, dtype, seed):
    g = torch.Generator().manual_seed(1000 + seed)
    return (torch.randn(T, D, generator=g) * 0.5).to(dtype).cuda()


def check(got, h, W, group, dtype, rows=None):
    """got [T, V] against h @ W^T in 64 bits (W [V, D] or [T, V, D]); rows: of
    the call, when that is not T."""
    hd = h.double()
    rounded = 0.0
    if W.dim() == 2:
        want, mag = hd @ W.t(), hd.abs() @ W.abs().t()
        if (rows or h.shape[0]) > 8:
            rounded = 7 * 2.0 ** -11 * (hd.square() @ W.square().t()).sqrt()
    else:
        want = (W * hd.unsqueeze(1)).sum(2)
        mag = (W.abs() * hd.abs().unsqueeze(1)).sum(2)
    D = h.shape[1]
    tol = (torch.finfo(dtype).eps / 2) * want.abs() \
        + (group / 16 + D / group + 16) * 2.0 ** -22 * mag + rounded + torch.finfo(dtype).tiny
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), float((err / tol).max()))


SHAPES = [  # V, D, group
    (1, 32, 32), (15, 96, 32), (17, 128, 128), (33, 64, 64), (100, 192, 64), (129, 160, 32),
    (1000, 640, 128), (2000, 1536, 64), (4099, 2048, 128), (777, 4096, 32), (260, 8192, 128),
    (64, 12288, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("V,D,group", SHAPES)
def test_logits(V, D, group, zeros, dtype):
    w, W = make_weight(V, D, group, zeros, dtype, seed=V + D)
    for T in (1, 3, 8, 9, 16, 17, 40):
        h = make_hidden(T, D, dtype, T)
        check(w4_logits(h, w), h, W, group, dtype)


@pytest.mark.parametrize("T", [64, 128, 129, 256, 300])
@pytest.mark.parametrize("V,D,group,zeros,dtype", [
    (3000, 512, 64, True, torch.bfloat16), (20000, 2048, 128, False, torch.bfloat16),
    (1234, 1056, 32, True, torch.float16), (5000, 896, 128, True, torch.float16)])
def test_logits_many_rows(T, V, D, group, zeros, dtype):
    w, W = make_weight(V, D, group, zeros, dtype, seed=T)
    h = make_hidden(T, D, dtype, T)
    check(w4_logits(h, w), h, W, group, dtype)


def test_logits_large_head():
    """The 2048 x 128256 head: every SM, several units per warp."""
    w, W = make_weight(128256, 2048, 128, False, torch.bfloat16, seed=5)
    for T in (1, 8, 64):
        h = make_hidden(T, 2048, torch.bfloat16, T)
        check(w4_logits(h, w), h, W, 128, torch.bfloat16)


@pytest.mark.parametrize("T", [2, 24, 80])
def test_logits_into_a_strided_out(T):
    """Columns and rows around the output are left as they were; a hidden
    state slice that is not 16-byte aligned is accepted."""
    w, W = make_weight(1001, 256, 64, True, torch.bfloat16, seed=2)
    big = torch.full((T + 2, 1501), 7.0, dtype=torch.bfloat16, device="cuda")
    out = big[1:T + 1, 300:1301]
    buf = torch.zeros(T * 256 + 3, dtype=torch.bfloat16, device="cuda")
    h = buf[3:].view(T, 256)
    h.copy_(make_hidden(T, 256, torch.bfloat16, 3))
    assert w4_logits(h, w, out=out).data_ptr() == out.data_ptr()
    check(out, h, W, 64, torch.bfloat16)
    assert (big[0] == 7).all() and (big[-1] == 7).all()
    assert (big[:, :300] == 7).all() and (big[:, 1301:] == 7).all()


@pytest.mark.parametrize("T", [4, 33])
def test_rows_do_not_touch_each_other(T):
    """Infinities and NaN in one hidden row stay in that row's logits."""
    w, W = make_weight(500, 384, 128, True, torch.float16, seed=9)
    h = make_hidden(T, 384, torch.float16, 1)
    h[1, 5] = float("inf")
    h[2, 7] = float("nan")
    got = w4_logits(h, w)
    keep = [r for r in range(T) if r not in (1, 2)]
    check(got[keep], h[keep], W, 128, torch.float16, rows=T)
    assert got[2].isnan().all() and not got[1].isfinite().any()


@pytest.mark.parametrize("T", [1, 20])
def test_large_and_small_values(T):
    """Hidden states over the whole range of bf16 exponents, scales far apart:
    the products neither overflow nor vanish on the way."""
    V, D, group = 400, 512, 128
    w, W = make_weight(V, D, group, True, torch.bfloat16, seed=4)
    for scale in (2.0 ** -60, 2.0 ** 40):
        h = make_hidden(T, D, torch.bfloat16, 2) * scale
        check(w4_logits(h, w), h, W, group, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("K,cap,D,group,P", [
    (8, 16, 128, 128, 8), (37, 4, 1024, 64, 5), (50, 24, 160, 32, 13), (300, 16, 4096, 64, 64),
    (128, 1, 96, 32, 40), (600, 16, 2048, 128, 256), (20, 5, 8192, 32, 3), (4, 31, 576, 64, 4)])
def test_block_sparse(K, cap, D, group, P, zeros, dtype):
    V = K * cap + (3 if cap == 5 else 0)
    w, W = make_weight(V, D, group, zeros, dtype, seed=K)
    for T in (1, 2, 7):
        h = make_hidden(T, D, dtype, T)
        g = torch.Generator().manual_seed(T)
        ci = torch.stack([torch.randperm(K, generator=g)[:P] for _ in range(T)]).cuda()
        got = w4_block_sparse_logits(h, w, ci, K, cap)
        rows = (ci.unsqueeze(2) * cap + torch.arange(cap, device="cuda")).view(T, -1)
        check(got, h, W[rows], group, dtype)


def test_block_sparse_repeated_and_invalid_ids():
    K, cap, D = 10, 16, 256
    w, W = make_weight(K * cap, D, 64, True, torch.bfloat16, seed=1)
    h = make_hidden(3, D, torch.bfloat16, 1)
    ci = torch.tensor([[4, 4, 4], [-1, 9, 10], [0, 2 ** 40, -2 ** 40]], device="cuda")
    got = w4_block_sparse_logits(h, w, ci, K, cap).view(3, 3, cap)
    ok = (ci >= 0) & (ci < K)
    assert (got[~ok] == float("-inf")).all()
    rows = (ci.clamp(0, K - 1).unsqueeze(2) * cap + torch.arange(cap, device="cuda")).view(3, -1)
    want_ok = ok.unsqueeze(2).expand(3, 3, cap).reshape(3, -1)
    full = got.view(3, -1).masked_fill(~want_ok, 0.0)
    Wm = W[rows] * want_ok.unsqueeze(2)
    check(full, h, Wm, 64, torch.bfloat16)
    # the dense form gives the same rows
    assert torch.equal(got[0, 0], got[0, 1])


@pytest.mark.parametrize("T", [0, 1, 30])
def test_empty_calls(T):
    w, _ = make_weight(64, 64, 64, False, torch.bfloat16, seed=1)
    h = make_hidden(T, 64, torch.bfloat16, 1)
    assert w4_logits(h[:0], w).shape == (0, 64)
    ci = torch.zeros((T, 0), dtype=torch.int64, device="cuda")
    assert w4_block_sparse_logits(h, w, ci, 4, 16).shape == (T, 0)


@pytest.mark.parametrize("T", [1, 12, 48])
def test_side_stream_and_graph(T):
    """Calls on another stream than the default, and captured and replayed
    with new hidden states in place."""
    w, W = make_weight(3000, 1024, 128, True, torch.bfloat16, seed=8)
    h = make_hidden(T, 1024, torch.bfloat16, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = w4_logits(h, w)
        out = torch.empty_like(got)
        w4_logits(h, w, out=out)
    s.synchronize()
    check(got, h, W, 128, torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        w4_logits(h, w, out=out)
    for seed in (5, 6):
        h.copy_(make_hidden(T, 1024, torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        check(out, h, W, 128, torch.bfloat16)
        assert torch.equal(out, w4_logits(h, w))


def test_workspace_word_is_clear():
    """No bounded wait of the tensor-core kernel runs out."""
    import ctypes

    from flash_head import _lib
    for dtype in (torch.bfloat16, torch.float16):
        w, W = make_weight(40000, 1024, 64, True, dtype, seed=3)
        h = make_hidden(100, 1024, dtype, 3)
        lib = _lib.load_library()
        need = lib.fh_w4_workspace_bytes(ctypes.byref(w.desc), 100)
        ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        out = torch.empty(100, 40000, dtype=dtype, device="cuda")
        _lib.call("fh_w4_logits", ctypes.byref(w.desc), h.data_ptr(), 100, out.data_ptr(), 40000,
                  ws.data_ptr(), need, _lib.stream_ptr())
        torch.cuda.synchronize()
        assert int(ws[:4].view(torch.int32)) == 0
        check(out, h, W, 64, dtype)


@pytest.mark.parametrize("zeros,bound", [(False, 1 / 7), (True, 1 / 15)])
def test_from_dense(zeros, bound):
    """A quantised weight is within half a step of the original (a step is a
    group's largest magnitude / 7, or its range / 15), plus the rounding of
    the scale and of the zero point."""
    g = torch.Generator().manual_seed(3)
    W = (torch.randn(200, 256, generator=g) * 0.02).bfloat16().cuda()
    w = W4Weight.from_dense(W, 64, zeros)
    back = w.dequantize().view(200, 4, 64)
    x = W.float().view(200, 4, 64)
    if zeros:
        span = x.amax(2).clamp_min(0) - x.amin(2).clamp_max(0)
    else:
        span = x.abs().amax(2)
    step = span * bound
    # half a step of rounding, half a step of the zero point's rounding, and
    # the scale's own rounding (2^-8) over up to 15 steps
    tol = step * (0.5 + (0.5 if zeros else 0.0) + 15 * 2.0 ** -8 + 1e-3)
    assert ((back - x).abs() <= tol.unsqueeze(2)).all()
    h = make_hidden(2, 256, torch.bfloat16, 1)
    check(w4_logits(h, w), h, w.dequantize().double(), 64, torch.bfloat16)
