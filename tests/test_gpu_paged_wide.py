"""Decode attention over 4-bit pages with many (query row, head) columns a KV head: the tcgen05 kernel, which long tables
of more than 16 columns take. Bounds as in test_gpu_paged.py."""

import math

import pytest
import torch

from exp3_b200 import _capi, paged
from test_gpu_paged import Cache, DEV, attend, cached_values, check, ints, no_device_error, randn  # noqa: F401

pytestmark = pytest.mark.gpu
LONG = 1 << 17  # tokens of a table: whatever the lengths, the kernel for long ones


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("rows,heads,kv_heads", [(17, 1, 1), (5, 8, 2), (4, 28, 4), (16, 2, 1), (3, 11, 1), (5, 7, 1), (8, 8, 1), (13, 5, 1), (64, 16, 1)])
def test_columns(dim, rows, heads, kv_heads):
    """Blocks of 32 and 64, full and not, one and several."""
    attend("int4", [rows, rows + 1, 129, 700], rows, heads, kv_heads, dim, 32, seed=rows, table_tokens=LONG)


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("heads", [6, 12])
@pytest.mark.parametrize("length", [3, 15, 16, 17, 127, 128, 129, 255, 256, 257, 1000, 20011])
def test_lengths(dim, heads, length):
    attend("int4", [length], 3, heads, 1, dim, 16, seed=length, table_tokens=LONG)


@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("heads", [12, 32])
def test_ragged_batch_with_padding_and_inactive_sequences(page, heads):
    lengths = [300, 2, 1500, 1, 77, 1024, 33]
    counts = [3, 2, 0, 1, 3, 2, 1]
    starts = [297, 0, 1500, 0, -1, 1022, 32]
    attend("int4", lengths, 3, heads, 2, 128, page, seed=page, counts=counts, starts=starts, table_tokens=LONG)


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("table", [0, LONG])
def test_many_sequences(dim, table):
    """More than 32 of them; with short tables, a CTA takes a unit."""
    lengths = [3 + (37 * i) % 300 for i in range(170)]
    counts = [1 + i % 3 for i in range(170)]
    counts[7] = 0
    starts = [n - c for n, c in zip(lengths, counts)]
    starts[9] = -1
    attend("int4", lengths, 3, 24, 2, dim, 16, seed=9, counts=counts, starts=starts, table_tokens=table)


@pytest.mark.parametrize("k_size,v_size,q_size", [(1.0, 1e-6, 1.0), (1.0, 1e6, 1.0), (8.0, 1.0, 2.0), (1e-3, 1e-30, 1.0), (1.0, 1e30, 0.0)])
def test_sizes(k_size, v_size, q_size):
    attend("int4", [900], 5, 8, 2, 128, 64, seed=2, k_size=k_size, v_size=v_size, q_size=q_size, table_tokens=LONG)


@pytest.mark.parametrize("direction", [1, -1])
@pytest.mark.parametrize("heads", [6, 16])
def test_logits_that_rise_and_fall_along_the_sequence(direction, heads):
    """From -200 to 200 and back, so that the softmax's reference moves in many tiles of a CTA."""
    g = torch.Generator().manual_seed(31)
    n, rows = 30000, 3
    ramp = torch.linspace(-direction, direction, n)
    axis = randn(g, 128).float()
    k = ((torch.randn(1, n, 1, 128, generator=g) * 0.5) + 200 * ramp[None, :, None, None] * axis / axis.square().sum()).to(torch.bfloat16)
    v = randn(g, 1, n, 1, 128)
    q = (axis + torch.randn(1, rows, heads, 128, generator=g) * 0.05).to(torch.bfloat16).to(DEV)
    cache = Cache("int4", [n], 1, 128, 64, table_tokens=LONG)
    paged.paged_append(k.to(DEV), v.to(DEV), cache.pool, cache.table, ints([0]))
    lse = torch.empty(1, rows, heads, device=DEV)
    out = paged.paged_decode_attention(q, cache.pool, cache.table, ints([n - rows]), 1.0, lse=lse)
    check(cache, [n], [n - rows], [rows], q, [cached_values("int4", k[0].float(), v[0])], 1.0, out, lse)


def test_keys_whose_groups_differ_in_size():
    """A group 2^20 times as large as the others, which the queries do not read: the others count in full."""
    g = torch.Generator().manual_seed(32)
    n, rows, heads = 600, 4, 7
    k, v, q = randn(g, 1, n, 1, 128), randn(g, 1, n, 1, 128), randn(g, 1, rows, heads, 128)
    k[..., 32:64] *= 2.0 ** 20
    q[..., 32:64] = 0
    cache = Cache("int4", [n], 1, 128, 64, table_tokens=LONG)
    paged.paged_append(k.to(DEV), v.to(DEV), cache.pool, cache.table, ints([0]))
    lse = torch.empty(1, rows, heads, device=DEV)
    out = paged.paged_decode_attention(q.to(DEV), cache.pool, cache.table, ints([n - rows]), 0.088, lse=lse)
    kc, vc = cached_values("int4", k[0].float(), v[0])
    kc[..., 32:64] = 0
    check(cache, [n], [n - rows], [rows], q.to(DEV), [(kc, vc)], 0.088, out, lse)


def test_nan_stays_where_it_is_and_unseen_rows_hold_anything():
    g = torch.Generator().manual_seed(33)
    n, rows, heads = 500, 3, 14
    k, v, q = randn(g, 2, n, 2, 128), randn(g, 2, n, 2, 128), randn(g, 2, rows, heads, 128)
    outs = []
    for dirty in (False, True):
        if dirty:
            q[0, 1, 2, 5] = math.nan
            k[1, 40, 1, 3] = math.nan
            k[0, 402:], v[0, 402:] = math.nan, math.inf  # behind sequence 0's last row
        cache = Cache("int4", [n, n], 2, 128, 16, table_tokens=LONG)
        paged.paged_append(k.to(DEV), v.to(DEV), cache.pool, cache.table, ints([0, 0]))
        outs.append(paged.paged_decode_attention(q.to(DEV), cache.pool, cache.table, ints([399, 497]), 0.1))
    clean, got = outs
    assert clean.isfinite().all()
    assert got[0, 1, 2].isnan().all() and got[1, :, 7:].isnan().all()
    got[0, 1, 2] = clean[0, 1, 2]
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1, :, :7], clean[1, :, :7])


def test_huge_queries_pick_one_key():
    """The output is the value of the largest logit: its weight is 1 and the others' 0, so what is left is the value's two
    roundings, of code x scale to fp16 (11 + 3 bits to 11) and of the sum to bf16: (1 + 2^-11) (1 + 2^-8) - 1 < 2^-8 + 2^-11 +
    2^-18 of it (one rounding of the exact value alone, as one column's kernel has it, would be equality)."""
    g = torch.Generator().manual_seed(26)
    k, v, q = randn(g, 1, 300, 1, 128), randn(g, 1, 300, 1, 128), randn(g, 1, 2, 16, 128)
    cache = Cache("int4", [300], 1, 128, 64, table_tokens=LONG)
    paged.paged_append(k.to(DEV), v.to(DEV), cache.pool, cache.table, ints([0]))
    kc, vc = cached_values("int4", k[0].float(), v[0])
    logits = torch.einsum("rhd,td->rht", q[0].double(), kc[:, 0].double())
    logits[0, :, 299:] = -math.inf
    best = logits.argmax(-1)
    for size in (2.0 ** 40, 2.0 ** 100, 2.0 ** 115, 2.0 ** 124):
        out = paged.paged_decode_attention((q * size).to(DEV), cache.pool, cache.table, ints([298]), 1.0 if size < 1e30 else 2.0 ** -20)
        off = (out[0].cpu().double() - vc[best, 0].double()).abs()
        assert (off <= (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -18) * vc[best, 0].double().abs()).all(), size


@pytest.mark.parametrize("lost", [[2], [0, 1, 2, 3, 4, 5, 6, 7, 8], list(range(19))])
def test_missing_pages_are_skipped_and_reported(lost):
    """One in the middle; the first two tiles and a bit; all of them."""
    cache, q, out, lse, starts, counts, kv = attend("int4", [600, 96], 5, 8, 2, 128, 32, seed=12, table_tokens=LONG)
    table = cache.table.clone()
    table[0, lost] = -1
    got_lse = torch.empty_like(lse)
    got = paged.paged_decode_attention(q, cache.pool, table, ints(starts), 128 ** -0.5, lse=got_lse)
    assert _capi.device_error() == 2 and _capi.device_error() == 0
    torch.testing.assert_close(got[1], out[1], rtol=2.0 ** -7, atol=1e-6)  # perhaps another split
    keep = torch.tensor([t for t in range(600) if t // 32 not in lost], dtype=torch.long)
    if len(keep) == 0:
        assert (got[0] == 0).all() and (got_lse[0] == -math.inf).all()
    else:
        m = len(keep)
        check(cache, [m], [m - 5], [5], q[:1], [(kv[0][0][keep], kv[0][1][keep])], 128 ** -0.5, got[:1], got_lse[:1])


def test_other_strides_output_in_place_and_no_rows_touched():
    """Queries from a fused projection's output, results into them."""
    cache, q, out, *_ = attend("int4", [700, 50], 4, 14, 2, 128, 64, seed=40, table_tokens=LONG)
    fused = torch.full((2, 4, 20 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    view = fused.unflatten(-1, (20, 128))[:, :, :14]
    view.copy_(q)
    assert paged.paged_decode_attention(view, cache.pool, cache.table, ints([696, 46]), 128 ** -0.5, out=view) is view
    assert torch.equal(view, out) and (fused[..., 14 * 128:] == 7).all()


def test_again_on_two_streams_and_replayed():
    a = attend("int4", [6000, 40], 4, 28, 4, 128, 64, seed=15, table_tokens=LONG)
    b = attend("int4", [4000, 900], 9, 8, 2, 256, 32, seed=16, table_tokens=LONG)
    starts = [ints(a[4]), ints(b[4])]
    calls = [lambda: paged.paged_decode_attention(a[1], a[0].pool, a[0].table, starts[0], 128 ** -0.5),
             lambda: paged.paged_decode_attention(b[1], b[0].pool, b[0].table, starts[1], 256 ** -0.5)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(calls[i]())
    torch.cuda.synchronize()
    for got, c in zip(outs, (a, b)):
        assert all(torch.equal(x, c[2]) for x in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [calls[0](), calls[1](), calls[0]()]
    for _ in range(3):
        for x in got:
            x.zero_()
        graph.replay()
        assert torch.equal(got[0], a[2]) and torch.equal(got[1], b[2]) and torch.equal(got[2], a[2])


def test_few_and_many_columns_agree():
    """A draft's rows together and one by one."""
    cache, q, out, *_ = attend("int4", [9000], 6, 28, 4, 128, 64, seed=41, table_tokens=LONG)
    for r in range(6):
        one = paged.paged_decode_attention(q[:, r:r + 1].contiguous(), cache.pool, cache.table, ints([8994 + r]), 128 ** -0.5)
        torch.testing.assert_close(one[:, 0], out[:, r], rtol=2.0 ** -7, atol=2.0 ** -10)
