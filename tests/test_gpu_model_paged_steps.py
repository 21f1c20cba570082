"""Steps of the paged model: tokens of inactive slots, and a step that does not end."""

import pytest
import torch

from exp3_b200 import _capi, ops
from exp3_b200.attention import METHODS
from exp3_b200.model import AttentionSettings, Qwen2Model
from test_gpu_model_paged import CFG, prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
def test_any_token_may_stand_in_an_inactive_slot(graph):
    model = Qwen2Model(CFG, seed=26, attention=AttentionSettings("dense"))
    runs = []
    for other in (0, -1, 1 << 40):
        cache = model.new_cache(pages=20, page_size=16, format="int4", sequences=3, max_tokens=64)
        tokens = torch.full((3,), other, device="cuda")
        tokens[1] = model.prefill_paged(prompt(20, 2), cache, 1).argmax()
        if graph:
            runs.append(model.decode_paged_graph(tokens, 5, cache)[:, 1])
            assert cache.lengths == [-1, 24, -1]
        else:
            runs.append(model.decode_paged(tokens, cache)[1])
            assert cache.lengths == [-1, 21, -1]
        assert cache.starts.tolist() == cache.lengths
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
    assert _capi.device_error() == 0


@pytest.mark.parametrize("fails", [1, 2])
def test_a_step_that_raises_leaves_the_cache_as_the_last_whole_one(fails, monkeypatch):
    """The first call of the graphed decode's step runs, the second is captured: whichever raises, host and device agree on the lengths,
    and decoding goes on from there."""
    model = Qwen2Model(CFG, seed=27, attention=AttentionSettings("dense"))
    cache, other = (model.new_cache(pages=20, page_size=16, format="int4", sequences=2, max_tokens=64) for _ in range(2))
    tokens = torch.zeros(2, dtype=torch.int64, device="cuda")
    for c in (cache, other):
        tokens[1] = model.prefill_paged(prompt(20, 3), c, 1).argmax()
    step, calls = Qwen2Model._paged_step, []

    def failing(self, *args):
        calls.append(1)
        if len(calls) == fails:
            raise RuntimeError("out of memory")
        return step(self, *args)

    monkeypatch.setattr(Qwen2Model, "_paged_step", failing)
    with pytest.raises(RuntimeError, match="out of memory"):
        model.decode_paged_graph(tokens, 6, cache)
    monkeypatch.undo()
    done = fails - 1
    assert cache.lengths == [-1, 20 + done] and cache.starts.tolist() == cache.lengths
    for _ in range(done):
        tokens = model.decode_paged(tokens, other).argmax(-1)
    assert torch.equal(model.decode_paged(tokens, cache)[1], model.decode_paged(tokens, other)[1])


@pytest.mark.parametrize("reuse", [128, 700, 1100])
@pytest.mark.parametrize("method,alpha", [(m, a) for m in METHODS for a in (0.08, 0.3)])
def test_a_reused_prefix_is_read_as_keys_alone(method, alpha, reuse, monkeypatch):
    """The prefix's queries are never computed. Whatever their memory holds (NaN here), the new rows' attention, with tiles left out and
    tails, has the bits of a call on full queries."""
    model = Qwen2Model(CFG, seed=28, attention=AttentionSettings(method, alpha, sink=1, window=1, last_full=1))
    ids = prompt(1300, 51)
    cache = model.new_cache(pages=30, format="bf16", max_tokens=1400)
    model.prefill_paged(ids[:reuse], cache)
    calls = []
    kernel = ops.prefill_attention

    def spy(q, k, v, *args, tile_range=None):
        prefix = 128 * tile_range[0]
        assert prefix == reuse // 128 * 128
        full = torch.randn_like(q)
        full[:, prefix:] = q[:, prefix:]
        q[:, :prefix] = float("nan")
        got = kernel(q, k, v, *args, tile_range=tile_range)
        want = kernel(full, k, v, *args)
        calls.append(torch.equal(got[:, prefix:], want[:, prefix:]))
        return got

    monkeypatch.setattr(ops, "prefill_attention", spy)
    logits = model.prefill_paged(ids, cache, reuse=reuse)
    assert calls == [True] * CFG.num_hidden_layers and logits.isfinite().all()
    assert _capi.device_error() == 0
