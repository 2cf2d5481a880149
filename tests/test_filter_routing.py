"""The vLLM hook sends each request down the path of its own settings, whatever
its neighbours in the step have set (CPU, a fake head)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from flash_head.patches import logits_processor as lp
from test_filtered_host import FakeHead, metadata


class Head(FakeHead):
    original_shape = (1000, 8)

    def get_next_token_batched(self, h, do_sample=False, temperature=1.0, seed=0, offset=0):
        self.plain.append((h[:, 0].tolist(), temperature, seed))
        return torch.full((h.shape[0],), 7, dtype=torch.int64)


@pytest.fixture
def step(monkeypatch):
    head = Head()
    h = torch.arange(4.0).view(4, 1).expand(4, 8).contiguous()
    monkeypatch.setattr(lp, "_flash_head", head)
    monkeypatch.setattr(lp, "_last_hidden", h)
    return head, torch.tensor([1, 2, 3, 4], dtype=torch.int32)


def gens():
    return {r: torch.Generator().manual_seed(40 + r) for r in (1, 2, 3)}


def test_only_rows_that_set_a_filter_change_path(step):
    head, greedy = step
    # row 1 has nothing set: vLLM's values for that in every tensor
    out = lp.step_sampled_ids(greedy, metadata(
        top_k=torch.tensor([1000, 1000, 50, 1000]), top_p=torch.tensor([1.0, 1.0, 1.0, 0.9]),
        generators=gens()))
    (hs, u, t, k, p, m), = head.filtered
    assert hs[:, 0].tolist() == [2.0, 3.0] and k.tolist() == [50, 1000] and m is None
    assert torch.allclose(p, torch.tensor([1.0, 0.9])) and torch.allclose(t, torch.tensor([1.3, 0.9]))
    assert [(rows, round(t, 3)) for rows, t, _ in head.plain] == [([1.0], 0.7)]
    assert out.tolist() == [1, 7, 100, 101]


def test_a_seeded_request_does_not_see_its_neighbours_filters(step):
    """The temperature-only request's call, seed included, is the same with and
    without filtered neighbours; so is a filtered request's uniform."""
    head, greedy = step
    temps = torch.tensor([0.0, 0.7, 0.0, 0.9])
    lp.step_sampled_ids(greedy, metadata(temperature=temps, generators=gens()))
    alone = [c for c in head.plain if c[0] == [1.0]]
    head.plain.clear()
    lp.step_sampled_ids(greedy, metadata(temperature=temps, top_p=torch.tensor([1.0, 1.0, 1.0, 0.5]),
                                         generators=gens()))
    assert alone and [c for c in head.plain if c[0] == [1.0]] == alone
    u = head.filtered[0][1]
    head.filtered.clear()
    lp.step_sampled_ids(greedy, metadata(temperature=torch.tensor([0.0, 0.0, 0.0, 0.9]),
                                         top_p=torch.tensor([1.0, 1.0, 1.0, 0.5]),
                                         generators=gens()))
    assert torch.equal(head.filtered[0][1], u)


def test_values_that_keep_everything_are_no_filter(step):
    head, greedy = step
    lp.step_sampled_ids(greedy, metadata(top_k=torch.tensor([1000, 0, -1, 5000]),
                                         top_p=torch.ones(4)))
    assert not head.filtered and len(head.plain) == 3


def test_a_min_p_shorter_than_the_step_is_kept_for_its_rows(step, caplog):
    """It used to be dropped for every row, without a word."""
    head, greedy = step
    lp._warned.clear()
    proc = SimpleNamespace(min_p=torch.tensor([[0.1], [0.2]]), min_p_count=2)
    with caplog.at_level("WARNING"):
        for _ in range(2):
            lp.step_sampled_ids(greedy, metadata(
                logitsprocs=SimpleNamespace(argmax_invariant=[proc])))
    hs, _, _, k, p, m = head.filtered[0]
    assert hs[:, 0].tolist() == [1.0] and k is None and p is None
    assert torch.allclose(m, torch.tensor([0.2]))
    assert [c[0] for c in head.plain[:2]] == [[3.0], [2.0]]  # rows 3 and 2, by temperature
    assert sum("min-p" in r.getMessage() for r in caplog.records) == 1
