"""Host logic of the model's paged path on the CPU (tests/paged_model_cpu.py has the kernels' calls as plain torch)."""

import pytest
import torch

from paged_model_cpu import PlainModel, prompt, use_plain_calls


@pytest.fixture
def plain(monkeypatch):
    use_plain_calls(monkeypatch.setattr)


def test_any_token_may_stand_in_an_inactive_slot(plain):
    model = PlainModel(seed=1)
    runs = []
    for other in (0, -1, 1 << 40):
        cache = model.new_cache(pages=20, page_size=16, format="bf16", sequences=3, max_tokens=64)
        first = model.prefill_paged(prompt(20, 2), cache, 1).argmax()
        tokens = torch.full((3,), other)
        tokens[1] = first
        runs.append(model.decode_paged(tokens, cache)[1])
        assert cache.lengths == [-1, 21, -1] and cache.starts.tolist() == cache.lengths
    assert runs[0].isfinite().all() and torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
