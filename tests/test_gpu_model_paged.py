"""The model on a paged cache against its dense path, and the paged step's own forms against each other."""

import pytest
import torch

from exp3_b200 import _capi, decode, paged
from exp3_b200.model import AttentionSettings, Qwen2Config, Qwen2Model

pytestmark = pytest.mark.gpu
CFG = Qwen2Config(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                  num_attention_heads=4, num_key_value_heads=2)


def prompt(n, seed):
    return torch.randint(0, CFG.vocab_size, (n,), generator=torch.Generator().manual_seed(seed)).cuda()


def close(a, b, rel=3e-2):
    err, scale = (a - b).abs().max().item(), b.abs().max().item()
    cos = torch.nn.functional.cosine_similarity(a.flatten(), b.flatten(), dim=0).item()
    assert err <= rel * scale + 1e-3 and cos > 0.999, (err, scale, cos)


@pytest.mark.parametrize("method", ["dense", "mean_native"])
def test_batch_on_bf16_pages_matches_the_dense_cache(method):
    """Prompts of different lengths decode together; an empty slot among them."""
    settings = AttentionSettings(method, 0.08)
    model, dense = (Qwen2Model(CFG, seed=21, attention=settings) for _ in range(2))
    cache = model.new_cache(pages=60, page_size=32, format="bf16", sequences=4, max_tokens=1024)
    prompts = {0: prompt(333, 1), 1: prompt(17, 2), 3: prompt(800, 3)}
    tokens = torch.zeros(4, dtype=torch.int64, device="cuda")
    want = {}
    for s, ids in prompts.items():
        want[s] = [dense.prefill_logits(ids, 8)]
        close(model.prefill_paged(ids, cache, s), want[s][0])
        tokens[s] = want[s][0].argmax()
        for _ in range(3):
            with torch.inference_mode():
                want[s].append(dense._forward(want[s][-1].argmax().view(1), dense.length, decoding=True))
            dense.length += 1
    for step in range(1, 4):
        logits = model.decode_paged(tokens, cache)
        for s in prompts:
            close(logits[s], want[s][step])
            tokens[s] = want[s][step].argmax()  # both follow the dense path's tokens
    assert cache.lengths == [336, 20, -1, 803] and cache.starts.tolist() == cache.lengths
    assert _capi.device_error() == 0


def test_int4_step_attends_to_what_the_pages_hold():
    """The step's logits equal a forward whose attention reads the same pages back dense."""
    model = Qwen2Model(CFG, seed=22, attention=AttentionSettings("dense"))
    cache = model.new_cache(pages=40, format="int4", sequences=2, max_tokens=512)
    for s, n in ((0, 200), (1, 63)):
        model.prefill_paged(prompt(n, 30 + s), cache, s)
    tokens = torch.tensor([5, 9], device="cuda")
    before = cache.starts.clone()
    logits = model.decode_paged(tokens, cache)
    table = model._table(cache)
    with torch.inference_mode():
        h = torch.nn.functional.embedding(tokens, model.embed)
        x = model._rmsnorm(h, model.layers[0].ln1)
        for i in range(CFG.num_hidden_layers):
            if i:
                x = model._rmsnorm(down, model.layers[i].ln1, residual=h)
            q, k, v = model._qkv(i, x, 2)
            where = (cache.pools[i], cache.page_table)
            q = paged.paged_append(k, v, *where, before, q=q, rope=table)
            attn = torch.empty_like(q)
            for s in range(2):
                n = int(before[s]) + 1
                kd, vd = paged.paged_gather(cache.pools[i], cache.page_table[s:s + 1], torch.zeros_like(before[:1]), None, n)
                attn[s:s + 1] = decode.decode_attention(q[s:s + 1], kd, vd, model.scale)
            h, down = model._paged_rest(i, h, attn.view(2, -1))
        close(logits, model._logits(down, h), rel=1e-2)


@pytest.mark.parametrize("format", ["int4", "bf16"])
def test_graph_steps_equal_eager_steps(format):
    model = Qwen2Model(CFG, seed=23, attention=AttentionSettings("mean_native"))
    runs = []
    for graph in (False, True):
        cache = model.new_cache(pages=64, page_size=16, format=format, sequences=3, max_tokens=256)
        first = torch.zeros(3, dtype=torch.int64, device="cuda")
        for s, n in ((0, 40), (2, 130)):
            first[s] = model.prefill_paged(prompt(n, 40 + s), cache, s).argmax()
        if graph:
            out = model.decode_paged_graph(first, 10, cache)
        else:
            out = [first]
            for _ in range(9):
                out.append(model.decode_paged(out[-1], cache).argmax(-1))
            out = torch.stack(out)
        runs.append((out[:, [0, 2]], list(cache.lengths), cache.starts.tolist()))
    assert torch.equal(runs[0][0], runs[1][0]) and runs[0][1:] == runs[1][1:]
    assert runs[0][1] == [49, -1, 139]


@pytest.mark.parametrize("format,reuse,method", [("bf16", 300, "dense"), ("int4", 300, "dense"), ("bf16", 128, "mean_native"),
                                                 ("bf16", 60, "dense"), ("bf16", 700, "cgf_mean")])
def test_a_following_prompt_reuses_its_prefix(format, reuse, method):
    """The second turn from a cached prefix gives the whole prompt's logits (bf16: to the rounding of a prefill;
    int4: the prefix is what the pages hold, each row about a tenth off, which 300 rows of attention average), and
    leaves the same pages behind for its own rows."""
    model = Qwen2Model(CFG, seed=24, attention=AttentionSettings(method, 0.0))  # every causal block: no routing ties
    ids = prompt(700, 50)
    whole = model.new_cache(pages=30, format=format, max_tokens=1024)
    want = model.prefill_paged(ids, whole)
    turns = model.new_cache(pages=30, format=format, max_tokens=1024)
    model.prefill_paged(ids[:max(reuse, 1)], turns)
    got = model.prefill_paged(ids, turns, reuse=reuse)
    assert turns.lengths == [700]
    if format == "bf16":
        close(got, want)
        for i in range(CFG.num_hidden_layers):
            zero = torch.zeros(1, dtype=torch.int32, device="cuda")
            for a, b in zip(paged.paged_gather(turns.pools[i], turns.page_table, zero, None, 700),
                            paged.paged_gather(whole.pools[i], whole.page_table, zero, None, 700)):
                close(a.float(), b.float())
    else:
        assert torch.nn.functional.cosine_similarity(got, want, dim=0) > 0.95
    with pytest.raises(ValueError):
        model.prefill_paged(ids, turns, reuse=701)


def test_slots_are_reused():
    """A released slot's pages serve the next sequence, with its results as in a fresh cache."""
    model = Qwen2Model(CFG, seed=25, attention=AttentionSettings("dense"))
    cache = model.new_cache(pages=6, format="int4", sequences=2, max_tokens=256)
    model.prefill_paged(prompt(256, 60), cache, 0)
    with pytest.raises(_capi.FpxError):
        model.prefill_paged(prompt(200, 61), cache, 1)
    cache.release(0)
    got = model.prefill_paged(prompt(200, 61), cache, 1)
    fresh = model.new_cache(pages=6, format="int4", sequences=2, max_tokens=256)
    assert torch.equal(got, model.prefill_paged(prompt(200, 61), fresh, 1))
    token = torch.zeros(2, dtype=torch.int64, device="cuda")
    token[1] = got.argmax()
    assert torch.equal(model.decode_paged(token, cache)[1], model.decode_paged(token, fresh)[1])
