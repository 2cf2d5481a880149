"""Filtered sampling on the GPU against its definition in 64 bits, row by row.

Ids must be equal: both sides decide by 64-bit sums, whose errors (about 1e-15
of the mass) put a border between them with a probability of about
n * 1e-15 per row. The returned probability is rounded to fp32 once: half a
step, 2^-24 relative, next to the 64-bit errors of e_i and of the mass (fewer
than 2^-40).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from flash_head.sampling import sample_logits

pytestmark = pytest.mark.gpu


def oracle_row(x, u, T, k, p, m):
    """(column, probability) of one row of float64 logits, by the definition."""
    cols = np.flatnonzero(x > -np.inf)
    if cols.size == 0:
        return -1, 0.0
    order = cols[np.argsort(-x[cols], kind="stable")]
    if not T > 0:
        return int(order[0]), 1.0
    top = x[order[0]]
    if top == np.inf:
        e = (x[order] == np.inf).astype(np.float64)
    else:
        e = np.exp((x[order] - top) / T)
    n = order.size
    if m > 0:
        n = max(1, int((e >= min(m, 1.0)).sum()))
    if k > 0:
        n = min(n, int(k))
    if p < 1:
        run = np.concatenate([[0.0], np.cumsum(e[:n])])
        n = max(1, int((run[:n] < p * run[n]).sum()))
    by_col = np.argsort(order[:n])
    run = np.cumsum(e[:n][by_col])
    u = u if u > 0 else 0.0
    hit = np.flatnonzero(run > u * run[-1])
    j = hit[0] if hit.size else np.flatnonzero(e[:n][by_col] > 0)[-1]
    return int(order[:n][by_col[j]]), float(e[:n][by_col[j]] / run[-1])


def check(x, u, T=1.0, k=0, p=1.0, m=0.0, ids=None, **kw):
    B = x.shape[0]
    got, prob = sample_logits(x, u, T, k, p, m, ids=ids, return_prob=True, **kw)

    def host(v):
        v = v.float() if isinstance(v, torch.Tensor) else torch.full((B,), float(v))
        return v.cpu().double().numpy()
    xn, un = x.float().cpu().double().numpy(), u.double().cpu().numpy()
    Tn, kn, pn, mn = host(T), host(k), host(p), host(m)
    want = [oracle_row(xn[r], un[r], Tn[r], kn[r], pn[r], mn[r]) for r in range(B)]
    cols = np.array([c for c, _ in want])
    if ids is not None:
        i = ids.cpu().numpy()
        i = np.broadcast_to(i, xn.shape)
        cols = np.where(cols < 0, -1, i[np.arange(B), np.maximum(cols, 0)])
    assert np.array_equal(got.cpu().numpy(), cols), np.flatnonzero(got.cpu().numpy() != cols)[:8]
    pw = np.array([q for _, q in want])
    assert (np.abs(prob.cpu().double().numpy() - pw) <= pw * (2.0 ** -24 + 2.0 ** -40) + 1e-40).all()
    return got


def logits(B, n, dtype, seed, sigma=2.5, peak=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, n, generator=g) * sigma
    if peak:
        for r in range(B):
            at = torch.randperm(n, generator=g)[:30]
            x[r, at] += 12.0 - 2.0 * torch.log(torch.arange(1, at.numel() + 1).float())
    return x.to(dtype).cuda()


def uniforms(B, seed):
    g = torch.Generator().manual_seed(77 + seed)
    return torch.rand(B, generator=g, dtype=torch.float64).cuda()


def settings(B, seed):
    """Every filter on, off and at its ends, mixed over the rows."""
    g = torch.Generator().manual_seed(177 + seed)

    def pick(vals, dt):
        return torch.tensor(vals, dtype=dt)[torch.randint(len(vals), (B,), generator=g)].cuda()
    return {"T": pick([0.0, 0.3, 0.7, 1.0, 1.0, 1.7], torch.float32),
            "k": pick([0, 0, 1, 2, 5, 50, 400, 10 ** 6], torch.int32),
            "p": pick([1.0, 1.0, 0.1, 0.5, 0.9, 0.999, 0.0], torch.float32),
            "m": pick([0.0, 0.0, 0.0, 0.02, 0.3, 1.0], torch.float32)}


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 31, 255, 1000, 4096, 4111, 9001, 32003])
def test_sizes(n, dtype):
    for B, seed in ((1, 0), (5, 1), (40, 2)):
        x = logits(B, n, dtype, seed)
        check(x, uniforms(B, seed), **settings(B, seed))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,n", [(1, 128256), (3, 151936), (20, 128256), (80, 50003)])
@pytest.mark.parametrize("sigma,peak", [(0.4, False), (2.5, True)])
def test_vocabularies(B, n, dtype, sigma, peak):
    """Flat rows (every filter reaches deep into the row) and peaked ones."""
    x = logits(B, n, dtype, n + B, sigma, peak)
    u = uniforms(B, n)
    check(x, u)
    check(x, u, T=0.7, p=0.9)
    check(x, u, T=1.3, k=50, p=0.95, m=0.01)
    check(x, u, k=3000)
    check(x, u, **settings(B, B))


@pytest.mark.parametrize("B", [1, 6, 150, 300])
def test_batches(B):
    x = logits(B, 2000, torch.bfloat16, B)
    check(x, uniforms(B, B), **settings(B, B))


def test_a_row_does_not_depend_on_its_batch():
    x = logits(200, 30000, torch.bfloat16, 5)
    u, s = uniforms(200, 5), settings(200, 5)
    whole = check(x, u, **s)
    for r in (0, 17, 199):
        one = sample_logits(x[r:r + 1], u[r:r + 1], *(s[c][r:r + 1] for c in "Tkpm"))
        assert one[0] == whole[r]


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties(dtype):
    """Few distinct logits: every cut falls among equal ones; ties go by column."""
    g = torch.Generator().manual_seed(2)
    B, n = 64, 20001
    x = torch.randint(0, 4, (B, n), generator=g).to(dtype).cuda()
    u = uniforms(B, 9)
    for kw in ({}, {"k": 7}, {"k": 9000}, {"p": 0.3}, {"p": 0.95, "k": 12000}, {"p": 0.7, "m": 0.2},
               {"T": 0.0}):
        check(x, u, **kw)
    same = torch.full((4, n), -3.25, dtype=dtype, device="cuda")
    for kw in ({}, {"k": 5}, {"p": 0.25}, {"p": 0.25, "k": 100}, {"m": 1.0}, {"T": 0.0}):
        check(same, uniforms(4, 1), **kw)


def test_signed_zeros_are_equal():
    x = torch.tensor([[-0.0, 0.0, -0.0, -1.0]], device="cuda").repeat(5, 1)
    u = torch.tensor([0.0, 0.34, 0.67, 0.9, 0.999], dtype=torch.float64, device="cuda")
    check(x, u, k=3)
    check(x, u, k=2)
    check(x, u, T=0.0)
    # a threshold at zero keeps zeros of both signs
    check(x, u, m=1.0)
    check(x, u, k=3, m=0.9, p=0.7)
    y = torch.zeros(5, 3000, device="cuda")
    y[:, 1::2] = -0.0
    y[:, ::7] = -2.0
    for kw in ({"m": 1.0}, {"k": 900}, {"m": 0.5, "p": 0.4}, {"p": 0.9}):
        check(y, u, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masks(dtype):
    """-inf, NaN and the type's lowest value as masks; rows left with one entry
    or none; +inf entries take all the mass."""
    n = 5003
    x = logits(12, n, dtype, 3)
    low, inf, nan = torch.finfo(dtype).min, float("inf"), float("nan")
    x[0] = -inf
    x[1] = nan
    x[2] = -inf
    x[2, 4321] = -7.0
    x[3] = low
    x[3, 17] = -3.0
    x[4] = low
    x[5, ::2] = nan
    x[6, 1::3] = -inf
    x[7, 50:] = low
    x[8, 11] = x[8, 4000] = x[8, 4001] = inf
    x[9] = nan
    x[9, n - 1] = -inf
    x[10] = -inf
    x[10, 0] = low
    for kw in ({}, {"k": 3}, {"p": 0.8}, {"m": 0.1}, {"k": 40, "p": 0.9, "m": 0.01}, {"T": 0.0},
               {"T": 5.0, "p": 0.99}):
        for seed in range(3):
            got = check(x, uniforms(12, seed), **kw)
            assert got[[0, 1, 9]].tolist() == [-1, -1, -1] and got[2] == 4321
            assert got[3] == 17 and got[8] in (11, 4000, 4001) and got[10] == 0


@pytest.mark.parametrize("T", [1e-30, 1e-4, 0.05, 20.0, 1e20])
def test_temperatures(T):
    x = logits(30, 8000, torch.float32, 4)
    u = uniforms(30, 4)
    check(x, u, T=T)
    check(x, u, T=T, k=20)
    check(x, u, T=T, p=0.6)
    check(x, u, T=T, m=0.5)


def test_extreme_logits():
    """Logits over the whole fp32 range: nothing overflows."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(8, 3001, generator=g) * 1e38).clamp(-3.3e38, 3.3e38).cuda()
    check(x, uniforms(8, 1))
    check(x, uniforms(8, 1), T=1e38, p=0.9)
    check(x * 1e-45, uniforms(8, 2), T=1e-8, k=5)
    check(x * 1e-38 * 1e-7, uniforms(8, 3), p=0.5)


def test_uniforms_at_and_beyond_their_ends():
    x = logits(6, 3000, torch.bfloat16, 8)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -53, 1.0, 1.5, -0.5, float("nan")], dtype=torch.float64,
                     device="cuda")
    for kw in ({}, {"k": 10}, {"p": 0.9}):
        check(x, u, **kw)
    got = sample_logits(x[:1].repeat(3, 1), torch.tensor([0.1, 0.5, 0.9], device="cuda"))
    want = sample_logits(x[:1].repeat(3, 1),
                         torch.tensor([0.1, 0.5, 0.9], device="cuda").double())
    assert torch.equal(got, want)  # fp32 uniforms are converted


def test_draws_follow_the_distribution():
    """Evenly spaced uniforms: an entry of probability q is drawn q B times, to one."""
    B, n = 4000, 600
    x = logits(1, n, torch.float32, 6).repeat(B, 1)
    u = (torch.arange(B, dtype=torch.float64, device="cuda") + 0.5) / B
    got = sample_logits(x, u, temperature=1.2, top_k=100)
    keep = x[0].double().topk(100)
    q = torch.softmax(keep.values / np.float64(np.float32(1.2)), 0) * B
    count = torch.bincount(got, minlength=n)
    assert (count[keep.indices].double() - q).abs().max() <= 1.0 and count.sum() == B
    assert count.sum() == count[keep.indices].sum()


def test_views_strides_and_ids():
    """Rows at odd addresses, a row pitch, columns mapped to ids (shared and per row)."""
    n = 4097
    for dtype in DTYPES:
        big = torch.full((9, n + 50), 99.0, dtype=dtype, device="cuda")
        for off in (1, 2, 3, 5, 8):
            x = big[1:8, off:off + n]
            x.copy_(logits(7, n, dtype, off))
            u = uniforms(7, off)
            check(x, u, **settings(7, off))
            g = torch.Generator().manual_seed(off)
            ids = torch.randint(0, 200000, (7, n), generator=g, dtype=torch.int32).cuda()
            check(x, u, k=40, ids=ids)
            check(x, u, p=0.9, ids=ids[0].contiguous())
            big.fill_(99.0)
    xt = logits(n, 5, torch.float32, 1).t()  # columns are strided
    check(xt, uniforms(5, 1), p=0.9)
    out = torch.full((5,), -5, dtype=torch.int64, device="cuda")
    assert sample_logits(xt, uniforms(5, 1), out=out).data_ptr() == out.data_ptr()
    assert (out >= 0).all()


def test_empty():
    assert sample_logits(torch.zeros(0, 10, device="cuda"), uniforms(0, 0)).shape == (0,)
    got, prob = sample_logits(torch.zeros(3, 0, device="cuda"), uniforms(3, 0), return_prob=True)
    assert got.tolist() == [-1, -1, -1] and prob.tolist() == [0, 0, 0]


def test_side_stream_and_graph():
    B, n = 4, 40000
    x, u, s = logits(B, n, torch.bfloat16, 1), uniforms(B, 1), settings(B, 1)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    out = torch.empty(B, dtype=torch.int64, device="cuda")
    with torch.cuda.stream(st):
        sample_logits(x, u, *(s[c] for c in "Tkpm"), out=out)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        sample_logits(x, u, *(s[c] for c in "Tkpm"), out=out)
    for seed in (3, 4, 5):
        x.copy_(logits(B, n, torch.bfloat16, seed))
        u.copy_(uniforms(B, seed))
        for c, v in settings(B, seed).items():
            s[c].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, check(x, u, **s))


def test_repeated_calls_agree():
    x = logits(64, 60000, torch.float32, 2, sigma=1.0, peak=False)
    u, s = uniforms(64, 2), settings(64, 2)
    first = check(x, u, **s)
    for _ in range(5):
        assert torch.equal(first, sample_logits(x, u, *(s[c] for c in "Tkpm")))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,B", [(4111, 60), (50003, 60), (151936, 6)])
def test_cuts_at_every_depth(n, B, dtype):
    """Top-p alone, from the first entry to the last, on rows from flat to sharp."""
    for s, sigma in enumerate((1e-3, 0.3, 1.0, 3.0)):
        x = logits(B, n, dtype, 300 + s, sigma, peak=s % 2 == 1)
        p = torch.linspace(1e-4, 0.99999, B).cuda()
        check(x, uniforms(B, s), T=0.9, p=p)
        check(x, uniforms(B, s + 9), T=0.9, p=p, m=1e-7)


@pytest.mark.parametrize("dtype", DTYPES)
def test_heavy_entries_side_by_side(dtype):
    """The entries above the cut fill one stretch of the row, and few values."""
    B, n = 12, 60013
    x = logits(B, n, dtype, 41, 1.0, peak=False)
    p = torch.tensor([0.3, 0.6, 0.9, 0.99] * 3).cuda()
    for first, count in ((0, 1500), (30001, 700), (58000, 2013), (100, 5000)):
        y = x.clone()
        y[:, first:first + count] += 9.0
        check(y, uniforms(B, first), p=p)
        check((y * 4).round() / 4, uniforms(B, first + 1), T=1.3, p=p)


@pytest.mark.parametrize("shift", [0.0, 1e4, -1e4, 3e37])
def test_cuts_far_from_zero(shift):
    """Logits whose spread is a few steps of their type, and large ones."""
    B, n = 16, 40000
    p = torch.linspace(0.05, 0.999, B).cuda()
    x = logits(B, n, torch.float32, 51, 2.0) + shift
    check(x, uniforms(B, 3), p=p)
    check(x, uniforms(B, 4), T=max(1.0, abs(shift) / 1e4), p=p)
