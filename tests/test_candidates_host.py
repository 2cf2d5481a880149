"""FlashHead.candidate_logits' own arithmetic on the CPU, with a stand-in for the
kernels: given probes of every kind, and no rows at all."""

from __future__ import annotations

import pytest
import torch
from torch import nn

import flash_head.fused as fused
from flash_head.flash_head import FlashHead

D, K, CAP, P = 16, 6, 4, 3
INF = float("inf")


class Native:
    def __init__(self, fh, specials):
        self.fh = fh
        self.bufs = {"vocab_map": fh.vocab_maps.view(-1).to(torch.int32),
                     "special_slots": specials}

    def _h(self, hidden):
        return hidden.reshape(-1, D)

    def top_clusters(self, h):
        return torch.arange(P, dtype=torch.int32).expand(h.shape[0], P).contiguous()


def logits_16(hs, w_perm_flat, ci, n_clusters, cluster_size):
    """What the kernel does: a cluster id outside the head leaves its outputs as
    they were (here 99)."""
    w = w_perm_flat.view(n_clusters, cluster_size, D).float()
    ok = (ci >= 0) & (ci < n_clusters)
    x = torch.einsum("npcd,nd->npc", w[ci.clamp(0, n_clusters - 1)], hs.float())
    return torch.where(ok.unsqueeze(2), x, torch.tensor(99.0)).view(
        hs.shape[0], ci.shape[1] * cluster_size).to(hs.dtype)


@pytest.fixture
def head(monkeypatch):
    torch.manual_seed(3)
    lm = nn.Linear(D, K * CAP, bias=False).to(torch.bfloat16)
    fh = FlashHead(lm, torch.randn(D, K), torch.randperm(K * CAP).view(K, CAP), n_probes=P)
    monkeypatch.setattr(fused, "block_sparse_logits", logits_16)
    nat = Native(fh, torch.tensor([1, 21], dtype=torch.int32))
    monkeypatch.setattr(fh, "native", lambda: nat)
    return fh


def rows(n):
    return torch.randn(n, D, generator=torch.Generator().manual_seed(n)).to(torch.bfloat16)


def test_probes_that_name_no_cluster(head):
    """An index outside the head must not reach an indexing kernel (on a GPU its
    assertion ends the process), nor leave what was in memory as a logit."""
    h = rows(2)
    probes = torch.tensor([[2, -1, 4], [K, 0, 2 ** 40]])
    logits, ids = head.candidate_logits(h, probes)
    assert logits.shape == ids.shape == (2, P * CAP + 2)
    x = logits[:, :P * CAP].view(2, P, CAP)
    ok = torch.tensor([[True, False, True], [False, True, False]])
    assert (x[~ok] == -INF).all() and x[ok].isfinite().all()
    want, want_ids = head.candidate_logits(h, torch.tensor([[2, 3, 4], [1, 0, 5]]))
    w = want[:, :P * CAP].view(2, P, CAP)
    assert torch.equal(x[ok], w[ok])
    assert torch.equal(ids[:, :P * CAP].view(2, P, CAP)[ok],
                       want_ids[:, :P * CAP].view(2, P, CAP)[ok])


def test_a_cluster_named_twice_counts_once(head):
    h = rows(2)
    logits, _ = head.candidate_logits(h, torch.tensor([[3, 3, 1], [5, 0, 5]]))
    x = logits[:, :P * CAP].view(2, P, CAP)
    assert (x[0, 1] == -INF).all() and (x[1, 2] == -INF).all()
    assert x[0, [0, 2]].isfinite().all() and x[1, [0, 1]].isfinite().all()


def test_probes_of_other_shapes_are_refused(head):
    for bad in (torch.zeros(3, P, dtype=torch.int64), torch.zeros(P, dtype=torch.int64),
                torch.zeros(2, P)):
        with pytest.raises(ValueError, match="probes"):
            head.candidate_logits(rows(2), bad)
    logits, _ = head.candidate_logits(rows(2), torch.zeros(2, 1, dtype=torch.int32))
    assert logits.shape == (2, CAP + 2)


def test_no_rows(head):
    logits, ids = head.candidate_logits(rows(0))
    assert logits.shape == ids.shape == (0, P * CAP + 2)
    logits, ids = head.candidate_logits(rows(0), torch.zeros(0, 2, dtype=torch.int64))
    assert logits.shape == ids.shape == (0, 2 * CAP + 2)


def test_a_special_token_given_twice_is_one_candidate():
    lm = nn.Linear(D, K * CAP, bias=False).to(torch.bfloat16)
    fh = FlashHead(lm, torch.randn(D, K), torch.arange(K * CAP).view(K, CAP), n_probes=P,
                   special_token_ids=[7, 21, 7, 21, 3])
    assert fh.special_token_ids_tensor.tolist() == [7, 21, 3]


def test_block_sparse_probes_of_other_rows_are_refused():
    """(Their rows would be read past the end.)"""
    h, w = torch.zeros(3, D), torch.zeros(K * CAP * D)
    ci = torch.zeros(2, P, dtype=torch.int64)
    for call in (lambda: fused.block_sparse_logits(h, w, ci, K, CAP),
                 lambda: fused.block_sparse_logits_argmax(h, w, ci, torch.zeros(K * CAP), K, CAP),
                 lambda: fused.block_sparse_argmax_atomic(h, w, ci, torch.zeros(K * CAP), K, CAP)):
        with pytest.raises(ValueError, match="does not fit"):
            call()
