"""vLLM end to end with top-k, top-p and min-p: a request's filters reach
FlashHead's sampling kernels (tests/test_gpu_vllm.py has the model and the
driver)."""

from __future__ import annotations

import pytest

import test_gpu_vllm as base
from test_gpu_vllm import served  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu


def test_vllm_filters_are_applied(served, monkeypatch):  # noqa: F811
    """With top_k=3 every token is one of the three largest logits of its step
    (or a near-tie of the third: vLLM's hidden states are bf16), through the
    filtered path, and the seed repeats the run."""
    import torch
    from transformers import LlamaForCausalLM
    model_dir, site, oracle = served
    driver = base._DRIVER.replace("ignore_eos=True,", "ignore_eos=True, top_k=3, top_p=0.97, "
                                                      "min_p=0.001,")
    driver = driver.replace("sampled = []\n", "sampled = []\ncalls = []\n"
                            "from flash_head.flash_head import FlashHead\n"
                            "inner_f = FlashHead.get_next_token_filtered\n"
                            "def counted_f(self, h, *a, **kw):\n"
                            "    calls.append((int(h.shape[0]), sorted(k for k, v in kw.items()"
                            " if v is not None)))\n"
                            "    return inner_f(self, h, *a, **kw)\n"
                            "FlashHead.get_next_token_filtered = counted_f\n", 1)
    driver = driver.replace('"sampled": sampled,', '"sampled": sampled, "calls": calls,')
    monkeypatch.setattr(base, "_DRIVER", driver)
    prompts = [[1, 17, 305, 2201, 44]]
    runs = [base._run_vllm(model_dir, site, prompts, max_tokens=12, temperature=1.5, seed=3)
            for _ in range(2)]
    for out in runs:
        # the prompt's last position and every decode step
        assert len(out["calls"]) == 12 and all(n == 1 for n, _ in out["calls"])
        assert all({"temperature", "top_k", "top_p"} <= set(kw) for _, kw in out["calls"])
    assert runs[0]["tokens"] == runs[1]["tokens"]
    ref = LlamaForCausalLM.from_pretrained(model_dir, torch_dtype=torch.float32).eval()
    toks = runs[0]["tokens"][0]
    seq = prompts[0] + toks
    with torch.no_grad():
        hs = ref.model(torch.tensor([seq])).last_hidden_state[0].numpy()
    for i, t in enumerate(toks):
        x = oracle.W.astype("float64") @ hs[len(prompts[0]) + i - 1].astype("float64")
        third = sorted(x)[-3]
        assert x[t] >= third - 2e-2 * abs(third), (i, t, x[t], third)
