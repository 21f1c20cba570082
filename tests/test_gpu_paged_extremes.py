"""Decode attention over pages where sizes lie far apart: weights, groups of a value row, value rows; values that are no
numbers. Half steps h16 = 2^-11 (fp16) and h = 2^-8 (bf16)."""

import math

import pytest
import torch

from exp3_b200 import paged
from paged_reference import attention
from test_gpu_paged import Cache, DEV, cached_values, check, ints, no_device_error, randn  # noqa: F401

pytestmark = pytest.mark.gpu
H16, H = 2.0 ** -11, 2.0 ** -8


def whole_keys(g, n, dim):
    """Keys of whole numbers times 2^-9 that the 4-bit form holds exactly: each group has a 7. Against queries of 1 and -1 every
    product and sum of the logits is exact."""
    k = torch.randint(-7, 8, (1, n, 1, dim), generator=g).float()
    k.unflatten(-1, (-1, 32))[..., 0] = 7
    return (k * 2.0 ** -9).to(torch.bfloat16)


@pytest.mark.parametrize("nats", [12, 14])
@pytest.mark.parametrize("dim,rows,heads", [(128, 1, 2), (128, 5, 2), (256, 1, 2), (128, 9, 2), (256, 9, 4)])
def test_small_groups_keep_the_weight_of_many_unlikely_tokens(dim, rows, heads, nats):
    """One key far above 131071 others, which together weigh as much or an eighth; groups of values 64 and 256 times smaller
    than the row's largest. 450 sequences share the pages, so that a warp's run is long: what it loses, it loses of a quarter of the
    tokens or more.

    A product of probability and scale below 2^-14 rounds by up to 2^-25, so does a probability; the largest weight times value
    exponent stands for at least 2^10. A code is at most 7, and 7 times the exponent is at most the row's largest value:
    a token adds at most 3 * 2^-35 of the largest weighted value. Logits are exact here; 2^-16 is left for the exponentials and sums."""
    g = torch.Generator().manual_seed(50)
    n, batch, at = 131072, 450, 70001
    k, v = whole_keys(g, n, dim), 1 + 0.25 * torch.randn(1, n, 1, dim, generator=g)
    q = torch.where(torch.randn(dim, generator=g) > 0, 1.0, -1.0)
    top = torch.full((dim,), 6.0)
    top.unflatten(-1, (-1, 32))[..., 0] = 7.0
    k[0, at, 0] = (q * top * 2.0 ** -6 * (128 / dim)).to(torch.bfloat16)  # 12.06 in all
    scale = nats / 12.0
    v *= torch.tensor([1.0, 1 / 64, 1 / 256, 1 / 4] * (dim // 128)).repeat_interleave(32)
    v = v.to(torch.bfloat16)
    cache = Cache("int4", [n], 1, dim, 64, seed=50)
    paged.paged_append(k.to(DEV), v.to(DEV), cache.pool, cache.table, ints([0]))
    kc, vc = cached_values("int4", k[0].float(), v[0])
    assert torch.equal(kc, k[0].float())
    queries = q.to(torch.bfloat16).expand(1, rows, heads, dim)
    lse = torch.empty(batch, rows, heads, device=DEV)
    out = paged.paged_decode_attention(queries.expand(batch, -1, -1, -1).to(DEV).contiguous(), cache.pool,
                                       cache.table.expand(batch, -1).contiguous(), ints([n - rows] * batch), scale, lse=lse)
    want, want_lse, size, most = attention(queries[0], kc, vc, n - rows, scale)
    room = H * want.abs() + (2 * H16 + 2.0 ** -16) * size + 3 * n * 2.0 ** -35 * most[..., None]
    off = (out.cpu().double() - want).abs()
    assert (off <= room).all(), (off / room).amax((0, 1, 2))
    assert ((lse.cpu().double() - want_lse).abs() <= 2.0 ** -17 * (1 + want_lse.abs())).all()


@pytest.mark.parametrize("exponent", [30, 70, 100, 124])
@pytest.mark.parametrize("dim,rows,heads", [(128, 1, 4), (128, 3, 4), (256, 1, 4), (128, 3, 8), (256, 5, 8)])
@pytest.mark.parametrize("n", [300, 20011])
def test_value_rows_of_far_apart_sizes_weigh_as_they_should(exponent, dim, rows, heads, n):
    """Rows of values about 2^exponent among rows of 1e-20 (exponent -60) and of zeros: each takes its weight, whose sum
    divides the large ones. A first, a middle and a late one, so that sums stand before, between and behind them, in one
    CTA and in pieces. Bounds as in test_gpu_paged.py's `check`."""
    g = torch.Generator().manual_seed(51)
    k, v, q = randn(g, 1, n, 1, dim), randn(g, 1, n, 1, dim, size=1e-20), randn(g, 1, rows, heads, dim)
    v[:, ::3] = 0
    for at, size in ((n // 2, 1.0), (n - rows - 3, 0.25), (n // 2 + 40, 0.5)):
        v[:, at] = (randn(g, 1, dim).float().sign() * size * 2.0 ** exponent).to(torch.bfloat16)
    cache = Cache("int4", [n], 1, dim, 64, seed=51, table_tokens=(1 << 17) * (rows * heads > 16))  # wide: tcgen05
    paged.paged_append(k.to(DEV), v.to(DEV), cache.pool, cache.table, ints([0]))
    for first, last in ((0, n), (n // 2 + 1, n), (n // 2 - 40, n // 2 + 1)):  # tokens from the first on and up to the last one
        if (first, last) == (0, n):
            table, shift = cache.table, 0
        else:
            table, shift = cache.table[:, first // 64:].contiguous(), first // 64 * 64
        start = last - shift - rows
        lse = torch.empty(1, rows, heads, device=DEV)
        out = paged.paged_decode_attention(q.to(DEV), cache.pool, table, ints([start]), dim ** -0.5, lse=lse)
        kv = [tuple(x[shift:last] for x in cached_values("int4", k[0].float(), v[0]))]
        check(cache, [last - shift], [start], [rows], q.to(DEV), kv, dim ** -0.5, out, lse)


@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("dim,rows,heads", [(128, 1, 4), (128, 3, 4), (256, 1, 4), (128, 3, 8), (256, 5, 8)])
@pytest.mark.parametrize("n", [300, 20011])
def test_a_value_that_is_no_number_spoils_its_group_alone(value, dim, rows, heads, n):
    """The group's dims are NaN for the rows that see it; the others are the sum of all other rows (this one reads back as
    zero there), and so is the log-sum. Bounds as in test_gpu_paged.py's `check`."""
    g = torch.Generator().manual_seed(52)
    k, v, q = randn(g, 1, n, 1, dim), randn(g, 1, n, 1, dim), randn(g, 1, rows, heads, dim)
    v[0, n // 3, 0, 40] = value
    cache = Cache("int4", [n], 1, dim, 64, seed=52, table_tokens=(1 << 17) * (rows * heads > 16))
    paged.paged_append(k.to(DEV), v.to(DEV), cache.pool, cache.table, ints([0]))
    lse = torch.empty(1, rows, heads, device=DEV)
    out = paged.paged_decode_attention(q.to(DEV), cache.pool, cache.table, ints([n - rows]), dim ** -0.5, lse=lse)
    assert out[..., 32:64].isnan().all()
    kc, vc = cached_values("int4", k[0].float(), v[0])
    assert vc[n // 3, 0, 32:64].isnan().all() and (vc[n // 3, 0, :32] == 0).all() and (vc[n // 3, 0, 64:] == 0).all()
    vc[..., 32:64] = 0
    out[..., 32:64] = 0
    check(cache, [n], [n - rows], [rows], q.to(DEV), [(kc, vc)], dim ** -0.5, out, lse)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("form,dim,rows,heads", [("int4", 128, 4, 2), ("int4", 128, 5, 3), ("int4", 256, 4, 2), ("int4", 256, 3, 5), ("int4", 128, 7, 4), ("int4", 128, 5, 7),
                                                 ("int4", 256, 9, 4), ("bf16", 128, 4, 2), ("bf16", 128, 7, 4), ("bf16", 256, 4, 2),
                                                 ("bf16", 256, 9, 4)])
@pytest.mark.parametrize("n", [40, 300, 20011])
def test_a_value_that_is_no_number_reaches_no_row_before_it(value, form, dim, rows, heads, n):
    """In the call's own rows, as a draft's tokens are: the rows before it are as they are without it; those that see it are spoilt
    in its group (bf16 pages: its dim) alone. Bounds as in test_gpu_paged.py's `check`. An infinity in bf16 pages comes out as itself or
    as NaN: its probability is a sum of two bf16 terms h + l with l of either sign or zero, and where l <= 0, h inf + l inf is NaN."""
    g = torch.Generator().manual_seed(53)
    k, v, q = randn(g, 1, n, 1, dim), randn(g, 1, n, 1, dim), randn(g, 1, rows, heads, dim)
    for own in (rows // 2, rows - 1):
        v2 = v.clone()
        at = n - rows + own
        v2[0, at, 0, 41] = value
        cache = Cache(form, [n], 1, dim, 16, seed=53, table_tokens=(1 << 17) * (rows * heads > 16 and n > 40))
        paged.paged_append(k.to(DEV), v2.to(DEV), cache.pool, cache.table, ints([0]))
        lse = torch.empty(1, rows, heads, device=DEV)
        out = paged.paged_decode_attention(q.to(DEV), cache.pool, cache.table, ints([n - rows]), dim ** -0.5, lse=lse)
        kc, vc = cached_values(form, k[0].float(), v2[0])
        spoilt = slice(32, 64) if form == "int4" else slice(41, 42)
        assert not out[0, own:, :, spoilt].isfinite().any()
        vc[at, :, spoilt] = 0  # the rows before it do not read it
        where = (cache, [n], [n - rows], [own], q[:, :own].to(DEV), [(kc, vc)], dim ** -0.5, out[:, :own], lse[:, :own])
        check(*where)
        vc = vc.clone()
        vc[..., spoilt] = 0
        out[0, own:, :, spoilt] = 0
        check(cache, [n], [n - rows + own], [rows - own], q[:, own:].to(DEV), [(kc, vc)], dim ** -0.5, out[:, own:], lse[:, own:])


@pytest.mark.parametrize("form", ["int4", "bf16"])
@pytest.mark.parametrize("dim,rows,heads", [(128, 1, 4), (256, 2, 4), (128, 3, 8)])
@pytest.mark.parametrize("exponent", [110, 118, 122])
def test_large_queries_under_a_small_scale(form, dim, rows, heads, exponent):
    """The scale brings their logits to ordinary sizes; bf16 pages sum 256 products of up to 2^122 * 2^4, below 2^128. Bounds as in test_gpu_paged.py's `check`."""
    g = torch.Generator().manual_seed(54)
    n = 500
    k, v, q = randn(g, 1, n, 1, dim, size=0.5), randn(g, 1, n, 1, dim), randn(g, 1, rows, heads, dim) * 2.0 ** exponent
    cache = Cache(form, [n], 1, dim, 64, seed=54, table_tokens=(1 << 17) * (rows * heads > 16))
    paged.paged_append(k.to(DEV), v.to(DEV), cache.pool, cache.table, ints([0]))
    lse = torch.empty(1, rows, heads, device=DEV)
    scale = dim ** -0.5 * 2.0 ** -exponent
    out = paged.paged_decode_attention(q.to(DEV), cache.pool, cache.table, ints([n - rows]), scale, lse=lse)
    check(cache, [n], [n - rows], [rows], q.to(DEV), [cached_values(form, k[0].float(), v[0])], scale, out, lse)


@pytest.mark.parametrize("dim,rotary", [(128, 128), (256, 64)])
def test_large_values_beside_one_that_is_no_number_keep_their_bits(dim, rotary):
    """Equal to the restatement's: such a row has the largest exponent, at which values below 2^101 * 7 have no bits and larger ones some."""
    g = torch.Generator().manual_seed(55)
    k, v = randn(g, 1, 40, 2, dim), randn(g, 1, 40, 2, dim)
    for t in range(40):
        v[0, t, :, 32:64] *= 2.0 ** (90 + t)
        v[0, t, t % 2, 64 if t % 3 else 96] = (math.inf, math.nan, -math.inf)[t % 3]
    cache = Cache("int4", [40], 2, dim, 16, seed=55)
    where = (cache.pool, cache.table, ints([0]))
    paged.paged_append(k.to(DEV), v.to(DEV), *where, rope=paged.rope_table(40, rotary, device=DEV))
    got = paged.paged_gather(*where, None, 40)[1][0].cpu()
    want = cached_values("int4", k[0].float(), v[0])[1].to(torch.bfloat16)
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)
    assert want.isnan().any(-1).any(1).all() and (want[:, :, 32:64] != 0).any(-1).any(1).tolist().count(True) > 20


@pytest.mark.parametrize("dim,rows,heads", [(128, 1, 4), (256, 1, 4), (128, 3, 8)])
def test_tiny_values_beside_one_that_is_no_number(dim, rows, heads):
    """The row that holds it weighs as one of zeros does: values of 1e-12 in the other rows keep their bits."""
    g = torch.Generator().manual_seed(56)
    n = 300
    k, v, q = randn(g, 1, n, 1, dim), randn(g, 1, n, 1, dim, size=1e-12), randn(g, 1, rows, heads, dim)
    v[0, n // 3, 0, 40] = math.inf
    cache = Cache("int4", [n], 1, dim, 64, seed=56, table_tokens=(1 << 17) * (rows * heads > 16))
    paged.paged_append(k.to(DEV), v.to(DEV), cache.pool, cache.table, ints([0]))
    lse = torch.empty(1, rows, heads, device=DEV)
    out = paged.paged_decode_attention(q.to(DEV), cache.pool, cache.table, ints([n - rows]), dim ** -0.5, lse=lse)
    assert out[..., 32:64].isnan().all()
    kc, vc = cached_values("int4", k[0].float(), v[0])
    vc[..., 32:64] = 0
    out[..., 32:64] = 0
    check(cache, [n], [n - rows], [rows], q.to(DEV), [(kc, vc)], dim ** -0.5, out, lse)
