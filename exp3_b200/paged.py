"""The paged KV cache on libfpx: append with rotation, decode attention, gather.

The reference keeps HF's dynamic cache, one dense bf16 tensor a layer (``evaluate.py:357-405``);
a cache in pages lets sequences of any lengths share one pool, and the 4-bit form (146 bytes a token
and head of 128 dims against 512) holds 3.5 times the tokens, with as many fewer bytes to read in a
decode step at long context.

A pool is a tensor ``[pages, Hkv, page_size, row]``: bf16 with ``row = 2 d``, or uint8 with
``row = 9 d / 8 + 2`` for the 4-bit form (groups of 32 dims; the bytes' order is the kernels' own,
``paged_gather`` reads them back). ``new_pool`` makes one; ``PagedKVCache`` keeps the pools of a
model's layers with their page table.

Every call takes ``page_table`` [B, max_pages] int32 (a sequence's pages in order) and ``starts``
[B] int32: row i of sequence b stands at position ``starts[b] + i``. ``counts`` [B] int32 says how
many of the call's rows are rows; those behind are padding. A negative start makes a sequence
inactive. All three are read on the device, so a captured step follows them. An index that
names nothing (a page outside the pool, a position past the table) is skipped, and sets
``_capi.device_error`` to 2.
"""

from __future__ import annotations

import ctypes
import functools
from pathlib import Path
from typing import Optional

import torch

from ._capi import FpxError, lib

FORMATS = {"bf16": 0, "int4": 1}
BINDING_PATH = Path(__file__).resolve().parent / "_paged.so"
MAX_ROWS = 64  # query rows of a sequence in one paged_decode_attention (FPX_PAGED_MAX_ROWS)


def row_elements(format: str, head_dim: int) -> int:
    """Pool elements (bf16, or bytes of int4) of one token and KV head."""
    if format not in FORMATS:
        raise ValueError(f"unknown page format {format!r}; choose from {tuple(FORMATS)}")
    if head_dim not in (128, 256):
        raise FpxError(f"head dim {head_dim} is not compiled (128 or 256)")
    return 2 * head_dim if format == "bf16" else 9 * head_dim // 8 + 2


def new_pool(pages: int, kv_heads: int, head_dim: int = 128, page_size: int = 64, format: str = "int4",
             device="cuda", layers: int | None = None) -> torch.Tensor:
    """An unwritten pool [pages, Hkv, page_size, row], with ``layers`` a stack of them."""
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise FpxError("page_size must be a power of two, 16 .. 1024")
    if pages <= 0 or kv_heads <= 0:
        raise ValueError("a pool needs pages and KV heads")
    shape = (pages, kv_heads, page_size, row_elements(format, head_dim))
    return torch.empty(shape if layers is None else (layers, *shape),
                       dtype=torch.bfloat16 if format == "bf16" else torch.uint8, device=device)


def rope_table(positions: int, rotary: int = 128, theta: float = 1e6, device="cuda") -> torch.Tensor:
    """[positions, rotary] fp32: cosines, then sines, of position * theta^(-2 i / rotary). Angles are
    taken in 64 bits: in 32 a far position's angle is off by more than bf16 rounds."""
    inv = theta ** (-torch.arange(0, rotary, 2, device=device, dtype=torch.float64) / rotary)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * inv
    return torch.cat((angle.cos(), angle.sin()), 1).float()


@functools.lru_cache(maxsize=None)
def _binding():
    """The module that checks a call's tensors and makes the C call on their device's current stream."""
    if not BINDING_PATH.exists():
        raise FpxError(f"{BINDING_PATH} is missing: build it with `python -m exp3_b200.build`")
    try:
        from . import _paged
    except ImportError as e:
        raise FpxError(f"{BINDING_PATH} does not load ({e}): build it again with `python -m exp3_b200.build`") from e
    if _paged.TORCH_VERSION != torch.__version__:
        raise FpxError(f"{BINDING_PATH} was built for torch {_paged.TORCH_VERSION}, this is {torch.__version__}: build it again with "
                       "`python -m exp3_b200.build`")
    names = ("fpx_paged_append", "fpx_paged_gather", "fpx_paged_decode_attention", "fpx_paged_decode_workspace_bytes",
             "fpx_status_string")
    _paged.bind(*(ctypes.cast(getattr(lib(), name), ctypes.c_void_p).value for name in names), FpxError)
    return _paged


def paged_append(k, v, pool, page_table, starts, counts=None, q=None, rope=None, q_out=None, k_out=None):
    """Stores new rows k, v [B, L, Hkv, d] bf16 in the pages, keys rotated by ``rope``.

    ``rope`` is a table like ``rope_table``'s, [positions, rotary] fp32 (NeoX pairs (i, i + rotary / 2) of
    the first ``rotary`` dims), or None: no rotation. ``q`` [B, L, H, d]: queries, rotated into ``q_out``
    (may be q), which is returned; without ``q_out`` into a new tensor, whose padding rows are zero.
    ``k_out`` [B, L, Hkv, d] (may be k) also takes the rotated keys in bf16. With ``q_out`` given (or no q),
    padding rows are left as they are.
    Rotation is in fp32 and rounds once, to bf16 or to the 4-bit codes. Sequences of one call must not
    write the same page."""
    return _binding().paged_append(k, v, pool, page_table, starts, counts, q, rope, q_out, k_out)


def paged_gather(pool, page_table, starts, counts, length: int, k_out=None, v_out=None):
    """Rows back as bf16: (k, v) [B, length, Hkv, d], for a prefill over a cached prefix. Rows behind
    ``counts`` (None: every row counts) are left as they are in given outputs, and zero in new ones."""
    return _binding().paged_gather(pool, page_table, starts, counts, length, k_out, v_out)


def paged_decode_attention(q, pool, page_table, starts, scale: float, counts=None, out=None, lse=None, ws=None):
    """Attention of q [B, Lq, H, d] bf16 to the cached tokens, causal by position: row i of sequence b
    sees positions 0 .. starts[b] + i, its own with them (append first). Returns bf16 [B, Lq, H, d]
    (``out`` if given); ``lse`` fp32 [B, Lq, H] takes the natural-log sums. Padding rows give 0 and -inf. An infinity or NaN in
    a value spoils its dim (4-bit pages: its group of 32) of the rows that see it, and nothing else.

    For the few rows of a decode or verification step: Lq <= MAX_ROWS. A longer continuation reads its
    prefix with ``paged_gather`` and runs ``prefill_attention``. ``ws`` is a contiguous uint8 workspace of
    ``paged_decode_workspace_bytes``; without it each call takes its own from torch's allocator, so calls on
    several streams or in several graphs share nothing."""
    return _binding().paged_decode_attention(q, pool, page_table, starts, scale, counts, out, lse, ws)


def _head_dim(pool) -> int:
    return {256: 128, 512: 256, 146: 128, 290: 256}.get(pool.shape[-1], 0)


def paged_decode_workspace_bytes(pool, batch: int, rows: int, heads: int) -> int:
    """Bytes of ``paged_decode_attention``'s workspace, whatever the sequences' lengths."""
    none = torch.empty(0, dtype=torch.int32)
    form = _binding().check_where(pool, none[None, :0][:0], none, None, 0, pool.shape[1], _head_dim(pool))
    return int(lib().fpx_paged_decode_workspace_bytes(form, batch, rows, heads, pool.shape[1], _head_dim(pool)))


class PagedKVCache:
    """The pools of a model's layers, the page table that they share, and which pages are free.

    ``sequences`` slots of up to ``max_tokens`` tokens share ``pages`` pages. ``starts`` (device) is the
    position of a slot's next token, negative for an inactive slot; ``lengths`` is the same on the host. Pages are
    handed out by ``reserve`` and taken back by ``release``, on the host, before the calls that use them."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int = 128, page_size: int = 64,
                 format: str = "int4", sequences: int = 1, max_tokens: int | None = None, device="cuda"):
        if layers <= 0 or sequences <= 0:
            raise ValueError("a cache needs layers and sequences")
        self.pools = new_pool(pages, kv_heads, head_dim, page_size, format, device, layers)
        self.page_size, self.format, self.sequences = page_size, format, sequences
        self.max_tokens = pages * page_size if max_tokens is None else max_tokens
        self.page_table = torch.full((sequences, -(-self.max_tokens // page_size)), -1, dtype=torch.int32, device=device)
        self.starts = torch.full((sequences,), -1, dtype=torch.int32, device=device)
        self.lengths = [-1] * sequences
        self._free = list(range(pages - 1, -1, -1))
        self._held: list[list[int]] = [[] for _ in range(sequences)]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, sequence: int, tokens: int) -> None:
        """Pages for ``tokens`` tokens of a slot in all (those that it holds count)."""
        if tokens > self.max_tokens:
            raise FpxError(f"{tokens} tokens: a slot holds {self.max_tokens}")
        held = self._held[sequence]
        more = -(-tokens // self.page_size) - len(held)
        if more <= 0:
            return
        if more > len(self._free):
            raise FpxError(f"{more} pages are needed, {len(self._free)} are free")
        new = [self._free.pop() for _ in range(more)]
        self.page_table[sequence, len(held):len(held) + more] = torch.tensor(new, dtype=torch.int32).to(self.page_table.device)
        held.extend(new)

    def release(self, sequence: int) -> None:
        """Takes a slot's pages back and makes it inactive. Its calls must be in the stream already."""
        self._free.extend(reversed(self._held[sequence]))
        self._held[sequence] = []
        self.page_table[sequence] = -1
        self.set_length(sequence, -1)

    def set_length(self, sequence: int, tokens: int) -> None:
        """The slot's next token stands at position ``tokens`` (negative: inactive)."""
        if tokens > self.max_tokens:
            raise FpxError(f"{tokens} tokens: a slot holds {self.max_tokens}")
        if tokens > len(self._held[sequence]) * self.page_size:
            raise FpxError(f"the slot's {len(self._held[sequence])} pages hold fewer than {tokens} tokens")
        self.lengths[sequence] = tokens
        self.starts[sequence] = tokens

    def advance(self, tokens: int = 1) -> None:
        """Host side of a step that appended ``tokens`` tokens to every active slot and moved ``starts`` itself."""
        self.lengths = [n + tokens if n >= 0 else n for n in self.lengths]


# The same calls as PyTorch custom ops, for torch.compile and fake tensors.


@torch.library.custom_op("fpx::paged_append", mutates_args=("pool",))
def _append_op(k: torch.Tensor, v: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
               counts: Optional[torch.Tensor], q: Optional[torch.Tensor],
               rope: Optional[torch.Tensor]) -> torch.Tensor:
    out = paged_append(k, v, pool, page_table, starts, counts, q, rope)
    return k.new_empty(0) if out is None else out


@_append_op.register_fake
def _(k, v, pool, page_table, starts, counts, q, rope):
    return k.new_empty(0 if q is None else q.shape)


@torch.library.custom_op("fpx::paged_gather", mutates_args=())
def _gather_op(pool: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor, counts: Optional[torch.Tensor],
               length: int) -> tuple[torch.Tensor, torch.Tensor]:
    return paged_gather(pool, page_table, starts, counts, length)


@_gather_op.register_fake
def _(pool, page_table, starts, counts, length):
    shape = (starts.shape[0], length, pool.shape[1], _head_dim(pool))
    return pool.new_empty(shape, dtype=torch.bfloat16), pool.new_empty(shape, dtype=torch.bfloat16)


@torch.library.custom_op("fpx::paged_decode_attention", mutates_args=())
def _decode_op(q: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
               counts: Optional[torch.Tensor], scale: float) -> torch.Tensor:
    return paged_decode_attention(q, pool, page_table, starts, scale, counts)


@_decode_op.register_fake
def _(q, pool, page_table, starts, counts, scale):
    return q.new_empty(q.shape)


__all__ = ["FORMATS", "PagedKVCache", "new_pool", "rope_table", "row_elements", "paged_append", "paged_gather",
           "paged_decode_attention", "paged_decode_workspace_bytes", "FpxError"]
