"""The paged KV cache's operators against a plain restatement (tests/paged_reference.py).

Tolerances. Append and gather do the documented fp32 arithmetic operation by operation: equal
bits. Attention: with half steps h16 = 2^-11 (fp16) and h = 2^-8 (bf16),

    |out - exact| <= h |exact| + (2 h16 + 2 delta + 2^-18) sum_t p_t |v_t|

from the output's rounding; the probabilities' two fp16 roundings (int4; the two bf16 terms of
bf16 pages keep 2^-16); exp2's and the sums' fp32 error; and delta, the logits' error, twice (it moves the
weights and their sum). A logit adds d products in fp32: each addition is off by at most 2^-23 of the partial
sum, which int4's offset codes (fp16 1024 + n) bring to 1039 sum |q| over a group, so

    delta <= scale * 36 * 2^-23 * 1039 * sum_groups s_group sum_group |q|   (int4)
    delta <= scale * d * 2^-23 * sum |q k|                                  (bf16)

taken at the largest scales of a sequence. lse is off by delta, and by fp32 rounding.

fp16 below 2^-14 rounds by up to 2^-25 however small the number. The int4 kernel's probability u_t is
weight_t 2^e_t over the largest such of the sequence (or up to 2^8 more), its product with the group's
scale r < 2 rounds once more, and a code is at most 7: a token adds at most 7 (2 + 1) 2^-25 in units of
max_t weight_t 2^e_t <= max_t weight_t amax_t / 7. So T tokens add at most 3 T 2^-25 max_t weight_t amax_t, which
matters only in dims where the token of the largest weighted values has none.
"""

import math

import pytest
import torch

from exp3_b200 import _capi, paged
from paged_reference import attention, int4_keys, int4_values, rotate

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def no_device_error():
    _capi.device_error()
    yield
    assert _capi.device_error() == 0


def randn(g, *shape, size=1.0):
    return (torch.randn(*shape, generator=g) * size).to(torch.bfloat16)


class Cache:
    """A pool of unwritten memory (NaN scales) with a shuffled page table; entries past a sequence's
    pages name no page."""

    def __init__(self, form, lengths, kv_heads, dim, page, seed=0, table_tokens=0):
        g = torch.Generator().manual_seed(seed + 77)
        need = [max(1, -(-n // page)) for n in lengths]
        total = sum(need) + 2
        self.pool = paged.new_pool(total, kv_heads, dim, page, form, DEV)
        self.pool.view(torch.uint8).fill_(255)
        order = torch.randperm(total, generator=g).tolist()
        table = torch.full((len(lengths), max(max(need) + 1, table_tokens // page)), 1 << 30, dtype=torch.int32)
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor([order.pop() for _ in range(n)])
        self.table = table.to(DEV)
        self.form, self.dim, self.kv_heads = form, dim, kv_heads


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def cached_values(form, k, v):
    """What pages give back of k (fp32, rotated) and v."""
    if form == "int4":
        return int4_keys(k), int4_values(v.float())
    return k.to(torch.bfloat16).float(), v.float()


# ------------------------------------------------------------------------------ append, gather


@pytest.mark.parametrize("form", ["int4", "bf16"])
@pytest.mark.parametrize("dim,rotary,heads,kv_heads", [(128, 128, 7, 1), (128, 64, 4, 2), (256, 256, 4, 4), (256, 64, 5, 1),
                                                       (256, 8, 2, 1), (128, None, 3, 3)])
@pytest.mark.parametrize("page", [16, 64])
def test_append_then_gather_gives_the_documented_bits(form, dim, rotary, heads, kv_heads, page):
    g = torch.Generator().manual_seed(dim + page)
    starts, counts, length = [0, 5, 33, -1, 100], [37, 1, 0, 12, 37], 37
    cache = Cache(form, [s + n for s, n in zip(starts, counts)], kv_heads, dim, page)
    batch = len(starts)
    qkv = randn(g, batch, length, (heads + 2 * kv_heads) * dim + 4).to(DEV)[..., 4:]  # 8-byte aligned rows
    q = qkv[..., : heads * dim].unflatten(-1, (heads, dim))
    k = qkv[..., heads * dim:(heads + kv_heads) * dim].unflatten(-1, (kv_heads, dim))
    v = qkv[..., (heads + kv_heads) * dim:].unflatten(-1, (kv_heads, dim))
    table = None if rotary is None else paged.rope_table(140, rotary, 1e4, DEV)
    k_out = torch.full_like(k, 7.0)
    where = (cache.pool, cache.table, ints(starts))
    q_out = torch.full(q.shape, 9.0, dtype=q.dtype, device=DEV)
    assert paged.paged_append(k, v, *where, ints(counts), q, table, q_out=q_out, k_out=k_out) is q_out
    fresh = paged.paged_append(k, v, *where, ints(counts), q, table)  # the same rows again: the same cache
    kept = [torch.full((batch, length + 3, kv_heads, dim), 5.0, dtype=torch.bfloat16, device=DEV)[:, 1:-2] for _ in range(2)]
    paged.paged_gather(*where, ints(counts), length, *kept)
    new = paged.paged_gather(*where, ints(counts), length)
    for b, (s, n) in enumerate(zip(starts, counts)):
        n = 0 if s < 0 else n
        at = torch.arange(s, s + n)
        turn = (lambda x: x.float()) if rotary is None else (lambda x: rotate(x, at, table.cpu()))
        kr = turn(k[b, :n].cpu())
        kc, vc = cached_values(form, kr, v[b, :n].cpu())
        for got, want, pad in ((q_out, turn(q[b, :n].cpu()), 9.0), (fresh, turn(q[b, :n].cpu()), 0.0), (k_out, kr, 7.0),
                               (kept[0], kc, 5.0), (kept[1], vc, 5.0), (new[0], kc, 0.0), (new[1], vc, 0.0)):
            assert torch.equal(got[b, :n].cpu(), want.to(torch.bfloat16))
            assert (got[b, n:] == pad).all()


def test_append_in_place_and_row_by_row():
    """A prompt row by row, rotated in place, leaves the same bytes as in one call."""
    g = torch.Generator().manual_seed(3)
    k, v, q = randn(g, 1, 40, 2, 128).to(DEV), randn(g, 1, 40, 2, 128).to(DEV), randn(g, 1, 40, 6, 128).to(DEV)
    table = paged.rope_table(64, device=DEV)
    one, many = (Cache("int4", [40], 2, 128, 16) for _ in range(2))
    out = paged.paged_append(k, v, one.pool, one.table, ints([0]), q=q, rope=table)
    k2, q2 = k.clone(), q.clone()
    for i in range(40):
        paged.paged_append(k2[:, i:i + 1], v[:, i:i + 1], many.pool, many.table, ints([i]), q=q2[:, i:i + 1], rope=table,
                           q_out=q2[:, i:i + 1], k_out=k2[:, i:i + 1])
    assert torch.equal(one.pool, many.pool) and torch.equal(q2, out)
    assert torch.equal(k2[0].cpu(), rotate(k[0].cpu(), torch.arange(40), table.cpu()).to(torch.bfloat16))


def test_int4_rows_of_extreme_values():
    rows = torch.zeros(10, 128)
    g = torch.Generator().manual_seed(5)
    rows[1] = torch.randn(128, generator=g) * 1e-30
    rows[2] = torch.randn(128, generator=g) * 1e30
    rows[3, 17] = 3.0                                   # one element in the row
    rows[4] = torch.randn(128, generator=g)
    rows[4, 64:96] *= 1e-6                              # groups of very different sizes
    rows[5] = torch.linspace(-7, 7, 128)                # halves: ties go to the even code
    rows[6] = 3.0e38
    rows[7] = torch.randn(128, generator=g) * 1e-39     # subnormal
    rows[8] = torch.randn(128, generator=g); rows[8, 40] = math.inf
    rows[9] = torch.randn(128, generator=g); rows[9, 100] = math.nan
    rows = rows.to(torch.bfloat16)[None, :, None].expand(1, 10, 2, 128)
    cache = Cache("int4", [10], 2, 128, 16)
    where = (cache.pool, cache.table, ints([0]))
    paged.paged_append(rows.to(DEV), rows.to(DEV), *where)
    k, v = (x.cpu() for x in paged.paged_gather(*where, None, 10))
    kw, vw = int4_keys(rows[0].float()), int4_values(rows[0].float())
    for got, want in ((k[0], kw), (v[0], vw)):
        torch.testing.assert_close(got, want.to(torch.bfloat16), rtol=0, atol=0, equal_nan=True)
        assert got[8, :, 32:64].isnan().all() and got[9, :, 96:].isnan().all() and got[:8].isfinite().all()
    assert k[0, 8, :, 64:].isfinite().all() and v[0, 9, :, :96].isfinite().all()


# ----------------------------------------------------------------------------------- attention


def check(cache, lengths, starts, counts, q, kv, scale, out, lse):
    """kv[b]: the fp32 rows that the cache stands for."""
    h16, h = 2.0 ** -11, 2.0 ** -8
    for b in range(q.shape[0]):
        n = 0 if starts[b] < 0 else min(counts[b], q.shape[1])
        assert (out[b, n:] == 0).all() and (lse[b, n:] == -math.inf).all()
        if n == 0:
            continue
        k, v = (x[:lengths[b]] for x in kv[b])
        group = q.shape[2] // cache.kv_heads
        want, want_lse, size, most = attention(q[b, :n].cpu(), k, v, starts[b], scale)
        absq = q[b, :n].cpu().double().abs().unflatten(1, (cache.kv_heads, group))
        if cache.form == "int4":
            s = (k.abs().unflatten(-1, (-1, 32)).amax(-1) / 7).amax(0).double()  # [Hkv, groups]
            delta = 36 * 2.0 ** -23 * 1039 * torch.einsum("nhgj,hj->nhg", absq.unflatten(-1, (-1, 32)).sum(-1), s * 1.01)
        else:
            delta = cache.dim * 2.0 ** -23 * torch.einsum("nhgd,hd->nhg", absq, k.abs().amax(0).double())
        delta = (delta * scale + 2.0 ** -20).flatten(1)
        room = h * want.abs() + (2 * h16 + 2 * delta[..., None] + 2.0 ** -18) * size
        if cache.form == "int4":
            room += 3 * len(k) * 2.0 ** -25 * most[..., None]
        off = (out[b, :n].cpu().double() - want).abs()
        assert (off <= room).all(), (b, (off / room).max())
        # as a whole: roundings of size h and h16 are uniform, so their 2-norm is 1 / sqrt(3) of them at most, and
        # the 36 additions' errors add up as their squares do
        total = off.square().sum().sqrt() / want.square().sum().sqrt().clamp_min(1e-30)
        weight = size.square().sum().sqrt() / want.square().sum().sqrt().clamp_min(1e-30)
        assert total <= 1.2 * (h / 3 ** 0.5) + weight * (2 * h16 / 3 ** 0.5 + 2 * delta.max() / 6), total
        lse_off = (lse[b, :n].cpu().double() - want_lse).abs()
        assert (lse_off <= delta + 2.0 ** -17 * (1 + want_lse.abs())).all(), lse_off.max()


def attend(form, lengths, rows, heads, kv_heads, dim, page, seed=0, counts=None, starts=None, k_size=1.0, v_size=1.0,
           scale=None, q_size=1.0, table_tokens=0):
    g = torch.Generator().manual_seed(seed)
    batch = len(lengths)
    cache = Cache(form, lengths, kv_heads, dim, page, seed, table_tokens)
    counts = counts or [rows] * batch
    starts = starts or [n - c for n, c in zip(lengths, counts)]
    longest = max(lengths)
    k, v = randn(g, batch, longest, kv_heads, dim, size=k_size), randn(g, batch, longest, kv_heads, dim, size=v_size)
    k += randn(g, 1, 1, kv_heads, dim, size=k_size)
    paged.paged_append(k.to(DEV), v.to(DEV), cache.pool, cache.table, ints([0] * batch), ints(lengths))
    q = randn(g, batch, rows, heads, dim, size=q_size).to(DEV)
    scale = scale or dim ** -0.5
    lse = torch.full((batch, rows, heads), 3.0, device=DEV)
    out = paged.paged_decode_attention(q, cache.pool, cache.table, ints(starts), scale, ints(counts), lse=lse)
    kv = [cached_values(form, k[b].float(), v[b]) for b in range(batch)]
    check(cache, lengths, starts, counts, q, kv, scale, out, lse)
    return cache, q, out, lse, starts, counts, kv


@pytest.mark.parametrize("form", ["int4", "bf16"])
@pytest.mark.parametrize("length", [1, 15, 16, 17, 63, 64, 65, 257, 1000])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 7, 1), (128, 8, 4), (256, 4, 1), (128, 32, 2)])
def test_decode_lengths(form, length, dim, heads, kv_heads):
    attend(form, [length], 1, heads, kv_heads, dim, 16, seed=length)


@pytest.mark.parametrize("form", ["int4", "bf16"])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("rows,heads,kv_heads", [(2, 3, 1), (5, 4, 1), (4, 28, 4), (17, 2, 2), (64, 1, 1)])
def test_rows_are_causal_by_position(form, dim, rows, heads, kv_heads):
    attend(form, [rows, rows + 1, 131, 400], rows, heads, kv_heads, dim, 32, seed=rows)


@pytest.mark.parametrize("form", ["int4", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 128, 1024])
def test_ragged_batch_with_padding_and_inactive_sequences(form, page):
    lengths = [300, 2, 1500, 1, 77, 1024, 33]
    counts = [3, 2, 0, 1, 3, 2, 1]
    starts = [297, 0, 1500, 0, -1, 1022, 32]
    attend(form, lengths, 3, 12, 2, 128, page, seed=page, counts=counts, starts=starts)


@pytest.mark.parametrize("form", ["int4", "bf16"])
@pytest.mark.parametrize("longest", [40, 1500])
def test_many_sequences_share_the_launch(form, longest):
    """More units than CTAs, most of one granule; with a long table, whose work is split, and a short one."""
    lengths = [1 + (37 * i) % 40 for i in range(333)]
    lengths[200] = longest
    attend(form, lengths, 1, 8, 4, 128, 16, seed=9)


@pytest.mark.parametrize("form", ["int4", "bf16"])
@pytest.mark.parametrize("dim,heads", [(128, 4), (128, 24), (256, 10)])
def test_padding_and_inactive_sequences_of_short_tables(form, dim, heads):
    counts, starts = [3, 2, 0, 1, 3, 2, 1], [97, 0, 100, 0, -1, 22, 32]
    attend(form, [100, 2, 100, 1, 77, 24, 33], 3, heads, 2, dim, 16, seed=dim, counts=counts, starts=starts)


@pytest.mark.parametrize("form,dim,heads,kv_heads", [("int4", 128, 7, 1), ("int4", 256, 16, 4), ("bf16", 128, 5, 1), ("int4", 128, 16, 1)])
def test_one_long_sequence_over_all_ctas(form, dim, heads, kv_heads):
    attend(form, [40011], 1, heads, kv_heads, dim, 64, seed=1)


@pytest.mark.parametrize("form", ["int4", "bf16"])
@pytest.mark.parametrize("k_size,v_size,q_size", [(1.0, 1e-6, 1.0), (1.0, 1e6, 1.0), (8.0, 1.0, 2.0), (1e-3, 1e-30, 1.0), (1.0, 1e30, 0.0)])
def test_sizes_of_keys_and_values(form, k_size, v_size, q_size):
    attend(form, [700], 2, 4, 2, 128, 64, seed=2, k_size=k_size, v_size=v_size, q_size=q_size)


def test_values_of_mixed_sizes_weigh_as_they_should():
    """Tokens whose values are tiny or zero still take their weight: the first takes most of the softmax."""
    g = torch.Generator().manual_seed(21)
    k, v = randn(g, 1, 200, 1, 128), randn(g, 1, 200, 1, 128)
    q = randn(g, 1, 1, 4, 128)
    k[0, 0] = q[0, 0, 0] * 1.5
    v[0, 0] = 0
    v[0, 1] *= 1e-9
    v[0, 2] *= 1e9
    k[0, 2] = -q[0, 0, 0] * 3
    cache = Cache("int4", [200], 1, 128, 64)
    where = (cache.pool, cache.table)
    paged.paged_append(k.to(DEV), v.to(DEV), *where, ints([0]))
    lse = torch.empty(1, 1, 4, device=DEV)
    out = paged.paged_decode_attention(q.to(DEV), *where, ints([199]), 128 ** -0.5, lse=lse)
    check(cache, [200], [199], [1], q.to(DEV), [cached_values("int4", k[0].float(), v[0])], 128 ** -0.5, out, lse)


@pytest.mark.parametrize("form", ["int4", "bf16"])
def test_nan_and_infinity_stay_where_they_are(form):
    """A NaN in a query or a key reaches the heads that read it, and no other."""
    g = torch.Generator().manual_seed(4)
    k, v, q = randn(g, 2, 90, 2, 128), randn(g, 2, 90, 2, 128), randn(g, 2, 1, 6, 128)
    clean_cache = Cache(form, [90, 90], 2, 128, 16)
    where = (clean_cache.pool, clean_cache.table)
    paged.paged_append(k.to(DEV), v.to(DEV), *where, ints([0, 0]))
    clean = paged.paged_decode_attention(q.to(DEV), *where, ints([89, 89]), 0.1)
    q[0, 0, 1, 5] = math.nan
    k[1, 40, 1, 3] = math.nan
    v[1, 80, 0, 100] = math.inf
    dirty_cache = Cache(form, [90, 90], 2, 128, 16)
    where = (dirty_cache.pool, dirty_cache.table)
    paged.paged_append(k.to(DEV), v.to(DEV), *where, ints([0, 0]))
    out = paged.paged_decode_attention(q.to(DEV), *where, ints([89, 89]), 0.1)
    assert out[0, 0, 1].isnan().all() and out[1, 0, 3:].isnan().all()
    same = [(0, h) for h in (0, 2, 3, 4, 5)]
    assert all(torch.equal(out[b, 0, h], clean[b, 0, h]) for b, h in same)
    assert not out[1, 0, :3, 96:].isfinite().all(-1).any()
    early = paged.paged_decode_attention(q.to(DEV), *where, ints([38, 38]), 0.1)  # positions before the NaN
    assert early[1].isfinite().all()


@pytest.mark.parametrize("form", ["int4", "bf16"])
def test_huge_queries_pick_one_key(form):
    """Logits far apart: the output is the value of the largest, up to the largest bf16 queries. bf16 pages sum q k in
    fp32 before the scale: 128 products of 2^124 and 1 have a sum of about 2^124 128^0.5 2^2 > 2^128, which fp32 does not
    hold, so there the sizes end before (int4 brings the query to 2^15 first)."""
    g = torch.Generator().manual_seed(26)
    k, v = randn(g, 1, 300, 1, 128), randn(g, 1, 300, 1, 128)
    q = randn(g, 1, 1, 4, 128)
    cache = Cache(form, [300], 1, 128, 64)
    paged.paged_append(k.to(DEV), v.to(DEV), cache.pool, cache.table, ints([0]))
    kc, vc = cached_values(form, k[0].float(), v[0])
    best = torch.einsum("hd,td->ht", q[0, 0].double(), kc[:, 0].double()).argmax(-1)
    for size in (2.0 ** 40, 2.0 ** 100, 2.0 ** 115) + ((2.0 ** 124,) if form == "int4" else ()):
        out = paged.paged_decode_attention((q * size).to(DEV), cache.pool, cache.table, ints([299]), 1.0 if size < 1e30 else 2.0 ** -20)
        assert torch.equal(out[0, 0].cpu(), vc[best, 0].to(torch.bfloat16)), size


def test_shared_pages_and_output_in_place():
    """Two sequences with a common prefix in the same pages; the output may be the queries' tensor."""
    g = torch.Generator().manual_seed(27)
    k, v = randn(g, 1, 1300, 2, 128).to(DEV), randn(g, 1, 1300, 2, 128).to(DEV)
    q = randn(g, 2, 2, 8, 128).to(DEV)
    cache = Cache("int4", [1300], 2, 128, 64)
    paged.paged_append(k, v, cache.pool, cache.table, ints([0]))
    both = cache.table.expand(2, -1).contiguous()
    starts = ints([1298, 640])
    want = [paged.paged_decode_attention(q[b:b + 1], cache.pool, cache.table, starts[b:b + 1], 0.1) for b in range(2)]
    assert paged.paged_decode_attention(q, cache.pool, both, starts, 0.1, out=q) is q
    for b in range(2):
        torch.testing.assert_close(q[b], want[b][0], rtol=2.0 ** -7, atol=1e-6)  # another split of the keys


def test_unseen_rows_of_a_granule_hold_anything():
    """NaN and infinities stored behind a row's position, in its own granule, do not reach it."""
    g = torch.Generator().manual_seed(28)
    k, v, q = randn(g, 1, 64, 1, 128), randn(g, 1, 64, 1, 128), randn(g, 1, 4, 4, 128).to(DEV)
    for form in ("int4", "bf16"):
        outs = []
        for dirty in (False, True):
            kd, vd = k.clone(), v.clone()
            if dirty:
                kd[0, 41:], vd[0, 41:] = math.nan, math.inf
            cache = Cache(form, [64], 1, 128, 16)
            paged.paged_append(kd.to(DEV), vd.to(DEV), cache.pool, cache.table, ints([0]))
            outs.append(paged.paged_decode_attention(q, cache.pool, cache.table, ints([37]), 0.1))
        assert outs[0].isfinite().all() and torch.equal(*outs)


def test_pool_beyond_four_gigabytes():
    """Pages whose byte offsets pass 32 bits."""
    g = torch.Generator().manual_seed(6)
    pool = paged.new_pool(60000, 8, 128, 64, "int4", DEV)  # 4.5 GB
    table = ints([[59999, 3, 59990]])
    k, v, q = randn(g, 1, 150, 8, 128), randn(g, 1, 150, 8, 128), randn(g, 1, 1, 8, 128).to(DEV)
    paged.paged_append(k.to(DEV), v.to(DEV), pool, table, ints([0]))
    kg, vg = paged.paged_gather(pool, table, ints([0]), None, 150)
    kv = cached_values("int4", k[0].float(), v[0])
    assert torch.equal(kg[0].cpu(), kv[0].to(torch.bfloat16)) and torch.equal(vg[0].cpu(), kv[1].to(torch.bfloat16))
    lse = torch.empty(1, 1, 8, device=DEV)
    out = paged.paged_decode_attention(q, pool, table, ints([149]), 0.088, lse=lse)
    holder = Cache("int4", [16], 8, 128, 16)
    check(holder, [150], [149], [1], q, [kv], 0.088, out, lse)


# ------------------------------------------------------- indices that name nothing, streams, graphs


def test_missing_pages_are_skipped_and_reported():
    cache, q, out, lse, starts, counts, kv = attend("int4", [160, 96], 1, 4, 1, 128, 32, seed=12)
    for bad in (-1, cache.pool.shape[0], -(1 << 31)):
        table = cache.table.clone()
        table[0, 2] = bad  # tokens 64 .. 95 of sequence 0
        got_lse = torch.empty_like(lse)
        got = paged.paged_decode_attention(q, cache.pool, table, ints(starts), 128 ** -0.5, lse=got_lse)
        assert _capi.device_error() == 2 and _capi.device_error() == 0
        assert torch.equal(got[1], out[1])
        keep = torch.cat((torch.arange(64), torch.arange(96, 160)))
        check(cache, [128], [127], [1], q[:1], [(kv[0][0][keep], kv[0][1][keep])], 128 ** -0.5, got[:1], got_lse[:1])
        k, v = paged.paged_gather(cache.pool, table, ints([0, 0]), None, 160)
        assert _capi.device_error() == 2
        assert (k[0, 64:96] == 0).all() and (v[0, 64:96] == 0).all()
        assert torch.equal(k[0, 96:].cpu(), kv[0][0][96:160].to(torch.bfloat16))


def test_positions_past_the_table_write_nothing():
    g = torch.Generator().manual_seed(8)
    k, v, q = randn(g, 1, 40, 1, 128).to(DEV), randn(g, 1, 40, 1, 128).to(DEV), randn(g, 1, 40, 2, 128).to(DEV)
    cache = Cache("bf16", [32], 1, 128, 16)
    cache.table = cache.table[:, :2].contiguous()  # 32 tokens
    before = cache.pool.clone()
    paged.paged_append(k, v, cache.pool, cache.table, ints([0]))  # rows 32 .. 39 have no page
    assert _capi.device_error() == 2
    got, _ = paged.paged_gather(cache.pool, cache.table, ints([0]), None, 32)
    assert torch.equal(got, k[:, :32])
    paged.paged_append(k, v, cache.pool, cache.table, ints([2**31 - 20]))
    assert _capi.device_error() == 2
    untouched = cache.table[0].tolist()
    rest = [i for i in range(cache.pool.shape[0]) if i not in untouched]
    assert torch.equal(cache.pool[rest].view(torch.int16), before[rest].view(torch.int16))
    table = paged.rope_table(10, device=DEV)  # rows 10 .. have no rotation
    out = paged.paged_append(k[:, :16], v[:, :16], cache.pool, cache.table, ints([0]), q=q[:, :16], rope=table)
    assert _capi.device_error() == 2
    assert torch.equal(out[0, :10].cpu(), rotate(q[0, :10].cpu(), torch.arange(10), table.cpu()).to(torch.bfloat16))
    assert (out[0, 10:] == 0).all()


def test_a_bad_index_does_not_stop_other_kernels():
    """The report of a missing page leaves the prefill kernels, which stop after a wait that gave up, at work."""
    from exp3_b200 import ops
    g = torch.Generator().manual_seed(29)
    q, k = randn(g, 1, 300, 4, 128).to(DEV), randn(g, 1, 300, 2, 128).to(DEV)
    want = ops.prefill_attention(q, k, k, "fp_v1_rescue", 0.08, 0.088)
    cache = Cache("int4", [40], 2, 128, 16)
    paged.paged_append(k[:, :40], k[:, :40], cache.pool, torch.full_like(cache.table, -1), ints([0]))
    got = ops.prefill_attention(q, k, k, "fp_v1_rescue", 0.08, 0.088, out=torch.zeros_like(q))
    assert torch.equal(got, want)
    assert _capi.device_error() == 2


def test_results_do_not_depend_on_timing():
    cache, q, out, lse, starts, counts, _ = attend("int4", [5000, 3000, 20], 1, 28, 4, 128, 64, seed=14)
    for _ in range(5):
        again_lse = torch.empty_like(lse)
        again = paged.paged_decode_attention(q, cache.pool, cache.table, ints(starts), 128 ** -0.5, lse=again_lse)
        assert torch.equal(again, out) and torch.equal(again_lse, lse)


def test_two_streams_at_once():
    a = attend("int4", [6000], 1, 28, 4, 128, 64, seed=15)
    b = attend("bf16", [4000, 100], 2, 8, 2, 128, 32, seed=16)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, (c, s) in enumerate(zip((a, b), streams)):
            with torch.cuda.stream(s):
                outs[i].append(paged.paged_decode_attention(c[1], c[0].pool, c[0].table, ints(c[4]), 128 ** -0.5))
    torch.cuda.synchronize()
    for got, c in zip(outs, (a, b)):
        assert all(torch.equal(x, c[2]) for x in got)


def test_a_captured_step_follows_its_tensors():
    """Append + attention captured once, replayed as positions and counts change; two graphs of one pool."""
    g = torch.Generator().manual_seed(18)
    steps, batch = 24, 3
    k, v, q = (randn(g, steps, batch, 1, n, 128).to(DEV) for n in (2, 2, 6))
    table = paged.rope_table(steps, device=DEV)
    eager, graphed = (Cache("int4", [steps] * batch, 2, 128, 16, seed=18) for _ in range(2))
    counts = [[1, 1, int(i % 3 > 0)] for i in range(steps)]
    starts = [[i, i, sum(c[2] for c in counts[:i])] for i in range(steps)]

    def step(cache, k, v, q, s, c):
        qr = paged.paged_append(k, v, cache.pool, cache.table, s, c, q, table)
        return paged.paged_decode_attention(qr, cache.pool, cache.table, s, 128 ** -0.5, c)

    want = [step(eager, k[i], v[i], q[i], ints(starts[i]), ints(counts[i])) for i in range(steps)]
    slots = [(torch.empty_like(k[0]), torch.empty_like(v[0]), torch.empty_like(q[0]), ints([0] * 3), ints([0] * 3)) for _ in range(2)]
    graphs, outs = [], []
    for slot in slots:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(graphed, *slot))
        graphs.append(graph)
    graphed.pool.copy_(torch.full_like(graphed.pool, 255))
    for i in range(steps):
        for dst, src in zip(slots[i & 1], (k[i], v[i], q[i], ints(starts[i]), ints(counts[i]))):
            dst.copy_(src)
        graphs[i & 1].replay()
        assert torch.equal(outs[i & 1], want[i]), i
    assert torch.equal(eager.pool, graphed.pool)


def test_opcheck():
    cache, q, *_ = attend("int4", [40, 20], 1, 4, 2, 128, 16, seed=19)
    g = torch.Generator().manual_seed(20)
    k, v = randn(g, 2, 3, 2, 128).to(DEV), randn(g, 2, 3, 2, 128).to(DEV)
    where = (cache.pool, cache.table, ints([0, 1]))
    tests = ("test_schema", "test_faketensor")
    torch.library.opcheck(torch.ops.fpx.paged_append, (k, v, *where, ints([3, 2]), None, None), test_utils=tests)
    torch.library.opcheck(torch.ops.fpx.paged_append, (k, v, *where, None, q.expand(2, 3, 4, 128).contiguous(),
                                                       paged.rope_table(64, device=DEV)), test_utils=tests)
    torch.library.opcheck(torch.ops.fpx.paged_gather, (*where, ints([3, 2]), 3), test_utils=tests)
    torch.library.opcheck(torch.ops.fpx.paged_decode_attention, (q, *where, None, 0.1), test_utils=tests)
