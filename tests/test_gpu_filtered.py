"""A FlashHead step with filtered sampling: probes, candidate logits (16-bit or
4-bit weight), special tokens and the draw, run together.

Candidate logits are compared with products in 64 bits of the weights the
kernels read: fp32 sums of at most D + 16 terms, each addition off by 2^-22 of
the sum of magnitudes at worst (2^-23 for a fused one), then one rounding to the
head's dtype (half a step). The drawn ids are those of the definition in 64 bits
applied to the candidate logits themselves.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from headutil import build_head
from test_gpu_sampling import oracle_row, settings, uniforms

pytestmark = pytest.mark.gpu

D, K, CAP, P = 512, 256, 16, 24


def make(dtype=torch.bfloat16, specials=(3, 77, 4000), quantise=None):
    from flash_head.synthetic import HeadShape, make_head
    h = make_head(HeadShape(hidden=D, vocab=K * CAP, n_clusters=K, n_probes=P), seed=12)
    fh = build_head(h.weight, h.centroids, h.assignments, P, specials=list(specials),
                    stage1="model", dtype=dtype)
    if quantise:
        fh.quantize_head(*quantise)
    return fh


def hidden(n, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, D, generator=g) * 3.0).to(dtype).cuda()


def weight64(fh):
    w4 = fh.quantized()
    return w4.dequantize().double() if w4 is not None else fh.w_perm.view(-1, D).double()


def check_ids(logits, ids, got, prob, u, s):
    x, i, un = logits.float().double().cpu().numpy(), ids.cpu().numpy(), u.cpu().numpy()
    s = {c: v.float().double().cpu().numpy() for c, v in s.items()}
    for r in range(x.shape[0]):
        col, q = oracle_row(x[r], un[r], s["T"][r], s["k"][r], s["p"][r], s["m"][r])
        assert int(got[r]) == i[min(r, i.shape[0] - 1)][col], r
        assert abs(float(prob[r]) - q) <= q * (2.0 ** -24 + 2.0 ** -40) + 1e-40


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("quantise", [None, (128, False), (64, True)])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_step(dtype, quantise, n):
    fh = make(dtype, quantise=quantise)
    h = hidden(n, dtype, n)
    logits, ids = fh.candidate_logits(h)
    probes = fh.native().top_clusters(h).long()
    assert logits.shape == ids.shape == (n, P * CAP + 3) and logits.dtype == dtype
    # the candidates' ids and logits
    W = weight64(fh)
    slots = torch.cat([(probes.unsqueeze(2) * CAP + torch.arange(CAP, device="cuda")).view(n, -1),
                       fh.native().bufs["special_slots"].long().expand(n, 3)], 1)
    assert torch.equal(ids.long(), fh.vocab_maps.view(-1)[slots])
    rows = W[slots]
    want = (rows * h.double().unsqueeze(1)).sum(2)
    mag = (rows.abs() * h.double().abs().unsqueeze(1)).sum(2)
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (D + 16) * 2.0 ** -22 * mag
    special = torch.zeros_like(want, dtype=torch.bool)
    special[:, -3:] = ((slots[:, -3:] // CAP).unsqueeze(2) == probes.unsqueeze(1)).any(2)
    assert torch.equal(logits == float("-inf"), special)
    assert ((logits.double() - want).abs() <= tol)[~special].all()
    # the draw
    u, s = uniforms(n, n), settings(n, n)
    got, prob = fh.get_next_token_filtered(h, u, s["T"], s["k"], s["p"], s["m"], return_prob=True)
    check_ids(logits, ids, got, prob, u, s)


def test_whole_head():
    """The dense form draws from the 4-bit head's whole vocabulary."""
    fh = make(quantise=(128, True))
    for n in (1, 30):
        h = hidden(n, torch.bfloat16, 9)
        logits = fh.head_logits(h)
        u, s = uniforms(n, 3), settings(n, 3)
        got, prob = fh.get_next_token_filtered(h, u, s["T"], s["k"], s["p"], s["m"], dense=True,
                                               return_prob=True)
        check_ids(logits, fh.vocab_maps.view(1, -1), got, prob, u, s)


def test_greedy_rows_match_the_greedy_step():
    """At temperature 0 the 16-bit head's filtered step gives the greedy step's
    tokens, up to candidates whose logits round to the same value."""
    fh = make()
    h = hidden(64, torch.bfloat16, 4)
    got = fh.get_next_token_filtered(h, temperature=0.0)
    greedy = fh.get_next_token_batched(h)
    logits, ids = fh.candidate_logits(h)
    for r in torch.nonzero(got != greedy).view(-1).tolist():
        at = logits[r][(ids[r] == greedy[r])]
        assert at.max() == logits[r].max()
    assert (got == greedy).float().mean() > 0.8


def test_default_uniforms_follow_torch_seed():
    fh = make()
    h = hidden(8, torch.bfloat16, 5)
    torch.manual_seed(11)
    a = fh.get_next_token_filtered(h, temperature=1.5, top_k=20)
    torch.manual_seed(11)
    assert torch.equal(a, fh.get_next_token_filtered(h, temperature=1.5, top_k=20))


@pytest.mark.parametrize("quantise", [None, (128, False)])
def test_captured_step(quantise):
    fh = make(quantise=quantise)
    n = 3
    fh.prepare(n)
    h, u = hidden(n, torch.bfloat16, 1), uniforms(n, 1)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        fh.get_next_token_filtered(h, u, 0.8, 30, 0.9, 0.02)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        out = fh.get_next_token_filtered(h, u, 0.8, 30, 0.9, 0.02)
    for seed in (2, 3, 4):
        h.copy_(hidden(n, torch.bfloat16, seed))
        u.copy_(uniforms(n, seed))
        graph.replay()
        torch.cuda.synchronize()
        want = fh.get_next_token_filtered(h, u, 0.8, 30, 0.9, 0.02)
        assert torch.equal(out, want)
        x, ids = fh.candidate_logits(h)
        x = x.float().double().cpu().numpy()
        for r in range(n):
            col, _ = oracle_row(x[r], float(u[r]), np.float64(np.float32(0.8)), 30,
                                np.float64(np.float32(0.9)), np.float64(np.float32(0.02)))
            assert int(out[r]) == int(ids[r, col])
