"""Refusals of the paged calls' binding and of the cache's host side (no GPU)."""

import pytest
import torch

from exp3_b200 import _capi, paged


def decode(**change):
    a = dict(q=torch.zeros(1, 1, 4, 128, dtype=torch.bfloat16), pool=paged.new_pool(4, 2, 128, 16, "int4", "cpu"),
             page_table=torch.zeros(1, 4, dtype=torch.int32), starts=torch.zeros(1, dtype=torch.int32), scale=0.1)
    a.update(change)
    return paged.paged_decode_attention(**a)


@pytest.mark.parametrize("ws", [torch.empty(1, dtype=torch.uint8).expand(1 << 20), torch.empty(1 << 12, 2, dtype=torch.uint8)[:, 0],
                                torch.empty(64, 64, dtype=torch.uint8).t()])
def test_a_workspace_that_is_not_contiguous_is_refused(ws):
    """Its count of bytes is not what may be written from its address on."""
    with pytest.raises(_capi.FpxError, match="ws must be contiguous"):
        decode(ws=ws)
    with pytest.raises(_capi.FpxError, match="CUDA"):
        decode(ws=ws.contiguous())


def test_a_slot_holds_no_more_than_its_tokens():
    """Its last page has room behind max_tokens, where the model's rotation table ends."""
    cache = paged.PagedKVCache(1, pages=8, kv_heads=1, page_size=64, sequences=1, max_tokens=100, device="cpu")
    cache.reserve(0, 100)
    cache.set_length(0, 100)
    with pytest.raises(_capi.FpxError, match="100"):
        cache.set_length(0, 101)
    assert cache.lengths == [100] and cache.starts.tolist() == [100]


def test_more_query_rows_than_a_call_takes_are_refused_by_name():
    for rows, match in ((paged.MAX_ROWS, "CUDA"), (paged.MAX_ROWS + 1, "65 query rows")):
        with pytest.raises(_capi.FpxError, match=match):
            decode(q=torch.zeros(1, rows, 4, 128, dtype=torch.bfloat16))
