"""Host checks of the paged cache's calls (no GPU): sizes, refusals before any launch, fake ops."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from exp3_b200 import _capi, paged

A = ctypes.c_void_p(1 << 20)  # an aligned address that no refused call reads


def test_page_bytes():
    f = _capi.lib().fpx_paged_page_bytes
    assert f(0, 4, 128, 64) == 4 * 64 * 512 and f(1, 4, 128, 64) == 4 * 64 * 146
    assert f(1, 1, 256, 16) == 16 * 290 and f(0, 1, 256, 16) == 16 * 1024
    for bad in ((2, 4, 128, 64), (1, 0, 128, 64), (1, 4, 64, 64), (1, 4, 128, 48), (1, 4, 128, 8), (1, 4, 128, 2048)):
        assert f(*bad) == 0
    pool = paged.new_pool(3, 4, 128, 64, "int4", "cpu", layers=2)
    assert pool.shape == (2, 3, 4, 64, 146) and pool[0].numel() == 3 * f(1, 4, 128, 64)
    assert paged.new_pool(3, 4, 256, 16, "bf16", "cpu").shape == (3, 4, 16, 512)
    with pytest.raises(_capi.FpxError):
        paged.new_pool(3, 4, 128, 48, device="cpu")
    with pytest.raises(_capi.FpxError):
        paged.new_pool(3, 4, 64, device="cpu")
    with pytest.raises(ValueError):
        paged.new_pool(3, 4, format="int8", device="cpu")
    with pytest.raises(ValueError):
        paged.new_pool(0, 4, device="cpu")


def test_workspace_bytes_do_not_depend_on_lengths_and_refuse_what_is_not_compiled():
    f = _capi.lib().fpx_paged_decode_workspace_bytes
    assert 0 < f(1, 1, 1, 28, 4, 128) < f(1, 64, 1, 28, 4, 128) < f(1, 64, 8, 28, 4, 128)
    for bad in ((2, 1, 1, 28, 4, 128), (1, 0, 1, 28, 4, 128), (1, 1, 65, 28, 4, 128), (1, 1, 1, 28, 3, 128),
                (1, 1, 1, 34, 2, 128), (1, 1, 1, 28, 4, 64), (1, 1 << 24, 1, 2, 1, 128)):
        assert f(*bad) == 0


def append(**change):
    a = dict(format=1, q=A, qs=(0, 256, 128), k=A, ks=(0, 128, 128), v=A, vs=(0, 128, 128), B=1, L=4, H=2, Hkv=1, d=128,
             rope=A, rope_len=8, rotary=128, pool=A, pages=4, page_size=16, table=A, stride=4, max_pages=4, starts=A,
             counts=None, q_out=A, qo=(0, 256, 128), k_out=None, ko=(0, 0, 0))
    a.update(change)
    return _capi.lib().fpx_paged_append(
        a["format"], a["q"], *a["qs"], a["k"], *a["ks"], a["v"], *a["vs"], a["B"], a["L"], a["H"], a["Hkv"], a["d"],
        a["rope"], a["rope_len"], a["rotary"], a["pool"], a["pages"], a["page_size"], a["table"], a["stride"],
        a["max_pages"], a["starts"], a["counts"], a["q_out"], *a["qo"], a["k_out"], *a["ko"], 0, None)


ODD = ctypes.c_void_p((1 << 20) + 2)


@pytest.mark.parametrize("status,change", [
    (-1, dict(format=2)), (-1, dict(k=None)), (-1, dict(v=None)), (-1, dict(pool=None)), (-1, dict(table=None)),
    (-1, dict(starts=None)), (-1, dict(B=0)), (-1, dict(L=-1)), (-1, dict(Hkv=0)), (-1, dict(H=-1)), (-1, dict(pages=0)),
    (-1, dict(max_pages=0)), (-1, dict(q=None)), (-1, dict(q_out=None)), (-1, dict(H=0)), (-1, dict(rope_len=0)),
    (-3, dict(d=64)), (-3, dict(page_size=24)), (-3, dict(page_size=8)), (-3, dict(page_size=2048)),
    (-2, dict(stride=3)), (-2, dict(rotary=12)), (-2, dict(rotary=136)), (-2, dict(rotary=0)), (-2, dict(k=ODD)),
    (-2, dict(ks=(0, 130, 128))), (-2, dict(Hkv=2, vs=(0, 256, 2))), (-2, dict(qs=(0, 257, 128))), (-2, dict(B=2, qo=(1, 256, 128))),
    (-2, dict(k_out=ODD)), (-2, dict(k_out=A, ko=(0, 2, 128))), (-2, dict(pool=ctypes.c_void_p((1 << 20) + 8))),
    (-2, dict(rope=ctypes.c_void_p((1 << 20) + 4)))])
def test_append_refuses(status, change):
    assert append(**change) == status


def gather(**change):
    a = dict(format=0, pool=A, pages=4, page_size=16, table=A, stride=4, max_pages=4, starts=A, counts=None, B=1, L=4, Hkv=1,
             d=128, k=A, ks=(0, 128, 128), v=A, vs=(0, 128, 128))
    a.update(change)
    return _capi.lib().fpx_paged_gather(
        a["format"], a["pool"], a["pages"], a["page_size"], a["table"], a["stride"], a["max_pages"], a["starts"], a["counts"],
        a["B"], a["L"], a["Hkv"], a["d"], a["k"], *a["ks"], a["v"], *a["vs"], 0, None)


@pytest.mark.parametrize("status,change", [
    (-1, dict(format=-1)), (-1, dict(k=None)), (-1, dict(v=None)), (-1, dict(pool=None)), (-1, dict(L=0)), (-1, dict(B=-2)),
    (-3, dict(d=192)), (-3, dict(page_size=17)), (-2, dict(stride=2)), (-2, dict(k=ODD)), (-2, dict(vs=(0, 129, 128)))])
def test_gather_refuses(status, change):
    assert gather(**change) == status


def decode(**change):
    a = dict(format=1, q=A, qs=(0, 256, 128), B=1, Lq=1, H=2, Hkv=1, d=128, scale=0.1, pool=A, pages=4, page_size=16, table=A,
             stride=4, max_pages=4, starts=A, counts=None, out=A, os=(0, 256, 128), lse=None, ws=A, ws_bytes=1 << 40)
    a.update(change)
    return _capi.lib().fpx_paged_decode_attention(
        a["format"], a["q"], *a["qs"], a["B"], a["Lq"], a["H"], a["Hkv"], a["d"], a["scale"], a["pool"], a["pages"],
        a["page_size"], a["table"], a["stride"], a["max_pages"], a["starts"], a["counts"], a["out"], *a["os"], a["lse"],
        a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("status,change", [
    (-1, dict(q=None)), (-1, dict(out=None)), (-1, dict(Lq=0)), (-1, dict(format=3)), (-1, dict(pool=None)),
    (-1, dict(starts=None)), (-2, dict(H=3, Hkv=2)), (-3, dict(Lq=65)), (-3, dict(H=17)), (-3, dict(d=64)),
    (-3, dict(B=1 << 24)), (-2, dict(Lq=2, qs=(0, 260, 128))), (-2, dict(q=ctypes.c_void_p((1 << 20) + 8))), (-5, dict(max_pages=33, stride=33, ws=None)),
    (-5, dict(max_pages=33, stride=33, ws_bytes=1000)), (-5, dict(Lq=16, max_pages=8192, stride=8192, ws=None)),
    (-5, dict(Lq=40, max_pages=8192, stride=8192, ws_bytes=148 * 64 * 128 * 4)), (-5, dict(max_pages=33, stride=33, ws=ctypes.c_void_p((1 << 20) + 8)))])
def test_decode_refuses(status, change):
    assert decode(**change) == status


def test_python_refusals():
    pool = paged.new_pool(4, 2, 128, 16, "int4", "cpu")
    k = torch.zeros(1, 4, 2, 128, dtype=torch.bfloat16)
    table, starts = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(_capi.FpxError):  # CPU tensors
        paged.paged_append(k, k, pool, table, starts)
    with pytest.raises(_capi.FpxError):
        paged.paged_gather(pool, table, starts, None, 4)
    with pytest.raises(_capi.FpxError):
        paged.paged_decode_attention(k[:, :1], pool, table, starts, 0.1)
    fit = paged._binding().check_where
    assert fit(pool, table, starts, None, 1, 2, 128) == 1
    assert paged.paged_decode_workspace_bytes(pool, 3, 2, 6) == _capi.lib().fpx_paged_decode_workspace_bytes(1, 3, 2, 6, 2, 128)
    for args in ((pool, table, starts, None, 1, 3, 128), (pool, table, starts, None, 1, 2, 256), (pool, table, starts, None, 2, 2, 128),
                 (pool[..., :-1], table, starts, None, 1, 2, 128), (pool.transpose(0, 1), table, starts, None, 1, 4, 128),
                 (pool[0], table, starts, None, 1, 2, 128), (pool, table, starts[None], None, 1, 2, 128),
                 (pool, table.t(), starts, None, 4, 2, 128), (pool, table, starts, torch.zeros(2, dtype=torch.int32), 1, 2, 128)):
        with pytest.raises(_capi.FpxError):
            fit(*args)
    for args in ((pool.float(), table, starts, None, 1, 2, 128), (pool, table.long(), starts, None, 1, 2, 128),
                 (pool, table, starts.long(), None, 1, 2, 128), (pool, table, starts, starts.long(), 1, 2, 128)):
        with pytest.raises(TypeError):
            fit(*args)


def test_fake_ops_give_the_layouts():
    f = torch.ops.fpx
    with FakeTensorMode():
        pool = torch.empty(4, 2, 16, 146, dtype=torch.uint8, device="cuda")
        k = torch.empty(3, 5, 2, 128, dtype=torch.bfloat16, device="cuda")
        q = torch.empty(3, 5, 6, 128, dtype=torch.bfloat16, device="cuda")
        table, starts = (torch.zeros(*s, dtype=torch.int32, device="cuda") for s in ((3, 4), (3,)))
        assert f.paged_append(k, k, pool, table, starts, None, q, None).shape == q.shape
        assert f.paged_append(k, k, pool, table, starts, starts, None, None).numel() == 0
        gk, gv = f.paged_gather(pool, table, starts, None, 5)
        assert gk.shape == gv.shape == k.shape and gk.dtype == torch.bfloat16
        assert f.paged_decode_attention(q, pool, table, starts, None, 0.1).shape == q.shape


def test_rope_table_is_right_at_far_positions():
    table = paged.rope_table(200001, 128, 1e6, "cpu")
    for p, i in ((0, 0), (7, 3), (200000, 0), (200000, 40), (131071, 63)):
        import math
        angle = p * 1e6 ** (-2 * i / 128)
        assert abs(float(table[p, i]) - math.cos(angle)) < 1e-6 and abs(float(table[p, 64 + i]) - math.sin(angle)) < 1e-6


def test_cache_pages_on_the_host():
    """Pages are handed out once, taken back whole, and refused beyond the pool or a slot's size."""
    cache = paged.PagedKVCache(2, pages=10, kv_heads=2, page_size=16, sequences=3, max_tokens=96, device="cpu")
    assert cache.pools.shape == (2, 10, 2, 16, 146) and cache.page_table.shape == (3, 6)
    cache.reserve(0, 33)
    cache.reserve(0, 40)
    cache.reserve(2, 96)
    assert cache.free_pages == 1
    used = [p for row in cache.page_table.tolist() for p in row if p >= 0]
    assert len(used) == len(set(used)) == 9
    with pytest.raises(_capi.FpxError):
        cache.reserve(1, 17)
    assert cache.free_pages == 1 and cache.page_table[1].tolist() == [-1] * 6
    with pytest.raises(_capi.FpxError):
        cache.reserve(2, 97)
    with pytest.raises(_capi.FpxError):
        cache.set_length(0, 49)
    cache.set_length(0, 48)
    cache.set_length(2, 0)
    cache.advance(2)
    assert cache.lengths == [50, -1, 2] and cache.starts.tolist() == [48, -1, 0]
    cache.release(0)
    assert cache.free_pages == 4 and cache.lengths[0] == -1 and cache.starts.tolist() == [-1, -1, 0]
    cache.reserve(1, 64)
    assert cache.free_pages == 0
    for bad in (dict(layers=0), dict(sequences=0)):
        with pytest.raises(ValueError):
            paged.PagedKVCache(**{**dict(layers=1, pages=2, kv_heads=1, device="cpu"), **bad})
