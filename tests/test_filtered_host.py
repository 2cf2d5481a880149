"""Routing of vLLM's per-request sampling settings to FlashHead's filtered
sampling, and refusals of the head's own entry points, on the CPU."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from flash_head.patches import logits_processor as lp


class FakeHead:
    def __init__(self):
        self.filtered, self.plain = [], []

    def get_next_token_filtered(self, h, uniforms, temperature, top_k, top_p, min_p):
        self.filtered.append((h, uniforms, temperature, top_k, top_p, min_p))
        return torch.arange(h.shape[0], dtype=torch.int64) + 100

    def get_next_token_batched(self, h, do_sample=False, temperature=1.0, seed=0, offset=0):
        self.plain.append((h.shape[0], temperature))
        return torch.full((h.shape[0],), 7, dtype=torch.int64)


@pytest.fixture
def step(monkeypatch):
    head = FakeHead()
    h = torch.arange(4.0).view(4, 1).expand(4, 8).contiguous()
    monkeypatch.setattr(lp, "_flash_head", head)
    monkeypatch.setattr(lp, "_last_hidden", h)
    return head, h, torch.tensor([1, 2, 3, 4], dtype=torch.int32)


def metadata(**kw):
    base = dict(all_greedy=False, temperature=torch.tensor([0.0, 0.7, 1.3, 0.9]), top_k=None,
                top_p=None, generators={})
    return SimpleNamespace(**{**base, **kw})


def test_filters_go_to_one_call_over_the_random_rows(step):
    head, h, greedy = step
    gen = torch.Generator().manual_seed(5)
    want_u = torch.rand((), generator=torch.Generator().manual_seed(5), dtype=torch.float64)
    out = lp.step_sampled_ids(greedy, metadata(
        top_k=torch.tensor([5, 6, 7, 8]), top_p=torch.tensor([0.5, 0.6, 0.7, 0.8]),
        generators={2: gen}))
    assert out.tolist() == [1, 100, 101, 102]  # the greedy row keeps its id
    (hs, u, t, k, p, m), = head.filtered
    assert hs[:, 0].tolist() == [1.0, 2.0, 3.0] and k.tolist() == [6, 7, 8] and m is None
    assert torch.allclose(t, torch.tensor([0.7, 1.3, 0.9]))
    assert torch.allclose(p, torch.tensor([0.6, 0.7, 0.8]))
    assert u.dtype == torch.float64 and u.shape == (3,) and u[1] == want_u
    assert not head.plain


def test_min_p_of_the_logits_processors(step):
    head, _, greedy = step
    proc = SimpleNamespace(min_p=torch.tensor([[0.1], [0.2], [0.3], [0.4]]), min_p_count=2)
    off = SimpleNamespace(min_p=torch.ones(4, 1), min_p_count=0)
    lp.step_sampled_ids(greedy, metadata(
        logitsprocs=SimpleNamespace(argmax_invariant=[SimpleNamespace(), off, proc])))
    _, _, _, k, p, m = head.filtered[0]
    assert k is None and p is None and torch.allclose(m, torch.tensor([0.2, 0.3, 0.4]))


def test_temperatures_alone_stay_on_their_path(step):
    head, _, greedy = step
    out = lp.step_sampled_ids(greedy, metadata())
    assert out.tolist() == [1, 7, 7, 7] and not head.filtered and len(head.plain) == 3
    # no random row: nothing is sampled
    head.plain.clear()
    out = lp.step_sampled_ids(greedy, metadata(temperature=torch.zeros(4),
                                               top_p=torch.full((4,), 0.9)))
    assert out.tolist() == [1, 2, 3, 4] and not head.filtered and not head.plain


def test_head_logits_need_a_quantised_head():
    from torch import nn

    from flash_head.flash_head import FlashHead
    lm = nn.Linear(64, 32, bias=False).to(torch.bfloat16)
    fh = FlashHead(lm, torch.randn(64, 4), torch.arange(32).view(4, 8), n_probes=2)
    with pytest.raises(RuntimeError, match="quantize_head"):
        fh.head_logits(torch.zeros(1, 64))
    w = fh.quantize_head(group_size=32)
    assert fh.quantized() is w and w.shape == (32, 64)
    fh.to(torch.float16)  # another weight
    assert fh.quantized() is None


def test_a_4_bit_weight_is_of_the_weight_as_it_is():
    """Written to, replaced or copied: the old 4-bit weight no longer serves."""
    import copy

    from torch import nn

    from flash_head.flash_head import FlashHead
    lm = nn.Linear(64, 32, bias=False).to(torch.bfloat16)
    fh = FlashHead(lm, torch.randn(64, 4), torch.arange(32).view(4, 8), n_probes=2)
    w = fh.quantize_head(group_size=32)
    assert fh.quantized() is w
    with torch.no_grad():
        fh.w_perm.mul_(2)
    assert fh.quantized() is None
    w = fh.quantize_head(group_size=32)
    state = {k: v * 3 for k, v in fh.state_dict().items()}
    if "w_perm" in state:
        fh.load_state_dict(state)
        assert fh.quantized() is None
        w = fh.quantize_head(group_size=32)
    twin = copy.deepcopy(fh)
    assert fh.quantized() is w and twin.quantized() is None
    assert torch.equal(copy.deepcopy(w).dequantize(), w.dequantize())
    fh.w_perm = fh.w_perm.clone()
    assert fh.quantized() is None


def test_copies_of_vllms_top_k():
    """int64 values beyond 32 bits keep their meaning; numbers that are none are refused."""
    from flash_head.sampling import _per_row
    v = torch.tensor([2 ** 40, -2 ** 40, 7, -1, 2 ** 32 + 1])
    got = _per_row("top_k", v, 5, torch.int32, v.device)
    assert got.dtype == torch.int32 and got.tolist() == [2 ** 31 - 1, -1, 7, -1, 2 ** 31 - 1]
    with pytest.raises(ValueError, match="integers"):
        _per_row("top_k", v.double(), 5, torch.int32, v.device)
