"""Host logic of the model's paged path on the CPU (tests/paged_model_cpu.py has the kernels' calls as plain torch)."""

import datetime

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

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


def decode_run(model):
    """Two prompts, one of them continued from its prefix, an empty slot, three steps: all logits."""
    cache = model.new_cache(pages=40, page_size=16, format="bf16", sequences=3, max_tokens=256)
    out = [model.prefill_paged(prompt(140, 5), cache, 0), model.prefill_paged(prompt(9, 6), cache, 2)]
    out.append(model.prefill_paged(torch.cat((prompt(140, 5), prompt(12, 7))), cache, 0, reuse=140))
    for tokens in ([3, -1, 5], [60, 7, 11], [0, -1, 63]):
        logits = model.decode_paged(torch.tensor(tokens), cache)
        out += [logits[0], logits[2]]
    assert cache.lengths == [155, -1, 12]
    return torch.stack(out)


def tensor_parallel_rank(rank, world, path):
    torch.set_num_threads(2)
    dist.init_process_group("gloo", init_method=f"file://{path}/store", rank=rank, world_size=world,
                            timeout=datetime.timedelta(seconds=120))
    try:
        use_plain_calls(setattr)
        model = PlainModel(seed=4, tp_rank=rank, tp_size=world)
        assert model.vocab_sharded and len(model.kv) == max(1, 2 // world)
        torch.save(decode_run(model), f"{path}/{rank}.pt")
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 4])
def test_tensor_parallel_paged_decode(plain, tmp_path, world):
    """Ranks that share KV heads out (2) and that share one group's query heads out (4) give one rank's logits, over the whole vocabulary in
    its order, on every rank alike.

    A rank's partial products round to bf16 (half a step 2^-8 of each) before they are summed, four times in the two layers, and
    rounding of the residual stream adds as much: logits agree to a few 2^-8 of their size; shards in another order would not at all."""
    want = decode_run(PlainModel(seed=4))
    ctx = mp.get_context("spawn")
    procs = [ctx.Process(target=tensor_parallel_rank, args=(r, world, str(tmp_path))) for r in range(world)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(timeout=300)
    assert [p.exitcode for p in procs] == [0] * world
    got = [torch.load(tmp_path / f"{r}.pt") for r in range(world)]
    assert all(torch.equal(got[0], g) for g in got[1:])
    off = (got[0] - want).square().sum(-1).sqrt() / want.square().sum(-1).sqrt()
    assert (off <= 12 * 2.0 ** -8).all(), off


@pytest.mark.parametrize("reuse,length", [(0, -1), (140, 128)])
def test_a_prefill_that_raises_leaves_what_is_whole(plain, monkeypatch, reuse, length):
    """Rows behind the reused tiles are overwritten layer by layer: a slot whose prefill raised holds those tiles, or nothing."""
    import exp3_b200.model as model_module

    model = PlainModel(seed=6)
    cache = model.new_cache(pages=40, page_size=16, format="bf16", sequences=2, max_tokens=256)
    model.prefill_paged(prompt(140, 5), cache, 1)
    longer = torch.cat((prompt(140, 5), prompt(12, 7)))
    want = model.prefill_paged(longer, model.new_cache(pages=40, page_size=16, format="bf16", max_tokens=256))
    ops, calls = model_module.ops, []

    class Failing(ops):
        @staticmethod
        def prefill_attention(*args, **kw):
            calls.append(1)
            if len(calls) == 2:
                raise RuntimeError("out of memory")
            return ops.prefill_attention(*args, **kw)

    monkeypatch.setattr(model_module, "ops", Failing)
    with pytest.raises(RuntimeError, match="out of memory"):
        model.prefill_paged(longer, cache, 1, reuse=reuse)
    assert cache.lengths == [-1, length] and cache.starts.tolist() == cache.lengths
    got = model.prefill_paged(longer, cache, 1, reuse=max(length, 0))
    assert cache.lengths == [-1, 152] and torch.allclose(got, want, atol=2e-2 * want.abs().max().item())
