"""Paged key/value cache: append, read back, and attention over it.

Serving next to ``flash_attn``: a prompt's attention runs in flash_attn while
``kv_cache_append`` stores its keys and values; then each new token is appended
(rotated on the way) and ``flash_attn_decode`` attends to everything cached.
A prompt that arrives in chunks, where the chunk ends at the same length in every
sequence of the call, reads its prefix back with ``kv_cache_read`` up to that length
and calls flash_attn(q_chunk, k_all, v_all, causal=True); flash_attn knows no lengths,
so the zeros behind a shorter sequence would count as keys and the mask would stand
at the longest one's end.  Chunks of different starts or counts go through
flash_attn_decode(..., starts=starts), or through read and flash_attn one sequence
at a time.

A page holds ``page_size`` tokens of one sequence; ``page_table`` (B, W) int32 names
the page of tokens i * page_size .. of each sequence in column i (entries behind
a sequence's length are not read).  Lengths and starts are (B,) int32 tensors on
the device and are never copied to the host, so the calls can be captured in CUDA
graphs and replayed with other lengths, tables and tokens.  A page id outside the
cache, or a length beyond the table, sets bit 2 of the status word
(``check_status``); those tokens are not written, and take no part in reads.

16-bit pages are ordinary tensors (pages, kv heads, page, head_dim).  4-bit pages
hold groups of 32 dims of a token as 4-bit codes with an fp16 scale and minimum
(5 bits a value; include/fa_sm100.h, csrc/fa_kv_cache.cuh); the attention
kernel multiplies the codes themselves.

The reference has no cache (its patched models decode in their own code).
"""
from __future__ import annotations

import math

import torch

from . import _lib, ops
from .rotary import Rotary, _NO_GRADIENT

BLOCK_TOKENS = 16


class PagedKVCache:
    """Pages of one attention layer, 16-bit (``k_pages``, ``v_pages``) or 4-bit
    (``PagedKVCache.of_blocks``); ``PagedKVCache.allocate`` makes them."""
    __slots__ = ("k_pages", "v_pages", "num_pages", "page_size", "n_heads", "head_dim", "dtype",
                 "bits", "device")

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor):
        shape, dtype = k_pages.shape, k_pages.dtype
        assert len(shape) == 4 and v_pages.shape == shape, \
            "k_pages and v_pages must be (pages, kv heads, page_size, head_dim)"
        assert dtype in (torch.float16, torch.bfloat16) and v_pages.dtype == dtype, \
            "fp16 (or bf16) pages only"
        assert k_pages.device == v_pages.device, "k_pages and v_pages must be on one device"
        assert shape[3] in (16, 32, 64, 128), \
            f"unsupported head_dim {shape[3]} (allowed: 16,32,64,128)"
        assert v_pages.is_contiguous(), "pages must be contiguous"
        self._set(k_pages, v_pages, shape, shape[2], shape[3], dtype, 16)

    def _set(self, k_pages, v_pages, shape, page_size, head_dim, dtype, bits):
        assert k_pages.is_contiguous(), "pages must be contiguous"
        assert 16 <= page_size <= 1024 and page_size & (page_size - 1) == 0, \
            f"page_size {page_size} is not a power of two from 16 to 1024"
        num_pages, n_heads = shape[0], shape[1]
        assert num_pages > 0 and n_heads > 0, "a cache needs pages and heads"
        assert num_pages * n_heads * page_size < 2 ** 31, \
            "pages * heads * page_size must be below 2^31"
        self.k_pages, self.v_pages = k_pages, v_pages
        self.num_pages, self.n_heads = num_pages, n_heads
        self.page_size, self.head_dim = page_size, head_dim
        self.dtype, self.bits, self.device = dtype, bits, k_pages.device

    @classmethod
    def of_blocks(cls, blocks: torch.Tensor, head_dim: int,
                  dtype: torch.dtype = torch.float16) -> "PagedKVCache":
        """4-bit pages: uint8 (pages, kv heads, page_size / 16, 20 * head_dim);
        ``dtype`` is that of the keys, values and queries in the calls."""
        assert head_dim in (32, 64, 128), f"unsupported head_dim {head_dim} at 4 bits (32,64,128)"
        assert dtype in (torch.float16, torch.bfloat16), "fp16 (or bf16) only"
        shape = blocks.shape
        assert blocks.dtype == torch.uint8 and len(shape) == 4 and shape[3] == 20 * head_dim, \
            "blocks must be uint8 (pages, kv heads, page_size / 16, 20 * head_dim)"
        c = cls.__new__(cls)
        c._set(blocks, None, shape, shape[2] * BLOCK_TOKENS, head_dim, dtype, 4)
        return c

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, n_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, bits: int = 16,
                 device="cuda") -> "PagedKVCache":
        """A new cache; what its pages hold is undefined until it is appended."""
        assert bits in (4, 16), "bits must be 4 or 16"
        if bits == 4:
            assert page_size % BLOCK_TOKENS == 0, "page_size must be a multiple of 16"
            return cls.of_blocks(torch.empty((num_pages, n_heads, page_size // BLOCK_TOKENS,
                                              20 * head_dim), dtype=torch.uint8, device=device),
                                 head_dim, dtype)
        shape = (num_pages, n_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device),
                   torch.empty(shape, dtype=dtype, device=device))


_INFERENCE = "the cache operators are for inference: call them under torch.no_grad()"


# The operators check their arguments themselves; the assertions, which say what
# is wrong in this module's terms, run when one refuses (they cost as much host
# time as a small call's launch).
def _check_ints(cache, batch, page_table, **vectors):
    dev = cache.device
    assert dev.type == "cuda", "the cache must be on CUDA"
    shape = page_table.shape
    assert len(shape) == 2 and shape[0] == batch and shape[1] > 0 \
        and page_table.dtype == torch.int32 and page_table.device == dev, \
        "page_table must be (batch, pages) int32 on the cache's device"
    for name, t in vectors.items():
        assert t is None or (t.shape == (batch,) and t.dtype == torch.int32 and t.device == dev), \
            f"{name} must be (batch,) int32 on the cache's device"


def _check_append(cache, k, v, page_table, starts, counts, q, rotary):
    shape = k.shape
    assert len(shape) == 4 and v.shape == shape, f"kv shape mismatch {shape} {v.shape}"
    B, S, Hkv, D = shape
    assert Hkv == cache.n_heads and D == cache.head_dim, \
        f"k {tuple(shape)} does not fit a cache of {cache.n_heads} heads of {cache.head_dim}"
    assert v.dtype == cache.dtype, f"k and v must have the cache's dtype {cache.dtype}"
    assert k.device == v.device == cache.device, "k and v must be on the cache's device"
    _check_ints(cache, B, page_table, starts=starts, counts=counts)
    if q is not None:
        assert q.dim() == 4 and q.shape[:2] == (B, S) and q.shape[3] == D and q.dtype == k.dtype \
            and q.device == cache.device, f"q {tuple(q.shape)} does not fit k {tuple(shape)}"
    if rotary is not None:
        assert rotary.dim <= D, f"rotary dim {rotary.dim} does not fit head_dim {D}"
        assert rotary.inv_freq.device == cache.device, "inv_freq must be on the cache's device"
        assert not (rotary.inv_freq.requires_grad and torch.is_grad_enabled()), _NO_GRADIENT


def _check_decode(q, cache, page_table, lengths, starts, sm_scale):
    assert math.isfinite(sm_scale), f"sm_scale {sm_scale} is not finite"
    shape, H = q.shape, cache.n_heads
    assert len(shape) == 4 and shape[3] == cache.head_dim and shape[2] > 0 and shape[2] % H == 0, \
        f"q {tuple(shape)} does not fit a cache of {H} heads of {cache.head_dim}"
    assert q.device == cache.device, "q must be on the cache's device"
    _check_ints(cache, shape[0], page_table, lengths=lengths, starts=starts)


def kv_cache_append(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor,
                    page_table: torch.Tensor, starts: torch.Tensor,
                    counts: torch.Tensor | None = None, *, q: torch.Tensor | None = None,
                    rotary: Rotary | None = None) -> torch.Tensor | None:
    """Store new tokens: token s of sequence b at position starts[b] + s.

    Args:
        k, v: (B, S, H_kv, D) of the cache's dtype, any strides.
        counts: (B,) tokens of each sequence that are new (the rows behind are
            padding and are not stored); None: all S.
        rotary: rotates k (and q) at those positions before k is stored.
        q: (B, S, H, D) queries of the same tokens; returned rotated (copied
            without ``rotary``), contiguous, padding rows included.
    No two tokens of one call may go to the same place of the cache.
    """
    dtype, dev = cache.dtype, cache.device
    assert k.dtype == dtype, f"k and v must have the cache's dtype {dtype}"
    assert not ((k.requires_grad or v.requires_grad or (q is not None and q.requires_grad))
                and torch.is_grad_enabled()), _INFERENCE
    if rotary is None:
        freq, interleaved, magnitude = None, False, 1.0
    else:
        freq, interleaved, magnitude = rotary.inv_freq, rotary.interleaved, rotary.magnitude
    ops.load()
    try:
        out = torch.ops.fav.kv_append(cache.k_pages, cache.v_pages, k, v, q, page_table, starts,
                                      counts, freq, interleaved, magnitude)
    except RuntimeError:
        _check_append(cache, k, v, page_table, starts, counts, q, rotary)
        raise
    ops.note_device(dev.index)
    if _lib.debug_sync():
        _lib.check_status(dev)
    return out if q is not None else None


def kv_cache_read(cache: PagedKVCache, page_table: torch.Tensor, lengths: torch.Tensor,
                  max_len: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The first lengths[b] cached tokens of each sequence as contiguous k and v
    (B, max_len, H_kv, D) of the cache's dtype; rows behind a length are zero (not
    masked: an attention over them needs the lengths).
    max_len: default the table's room; longer sequences are cut there."""
    if max_len is None:
        max_len = page_table.shape[-1] * cache.page_size
    assert max_len >= 0, "max_len must not be negative"
    dev = cache.device
    _check_ints(cache, lengths.shape[0], page_table, lengths=lengths)
    ops.load()
    ops.note_device(dev.index)
    k, v = torch.ops.fav.kv_read(cache.k_pages, cache.v_pages, cache.dtype, page_table, lengths,
                                 max_len)
    if _lib.debug_sync():
        _lib.check_status(dev)
    return k, v


def flash_attn_decode(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor,
                      lengths: torch.Tensor, causal: bool = True, sm_scale: float | None = None,
                      return_softmax_lse: bool = False, *, starts: torch.Tensor | None = None):
    """Attention of one or a few new tokens per sequence over the cache.

    Args:
        q: (B, S, H, D) of the cache's dtype, H % H_kv == 0 (query head h reads
            K/V head h // (H // H_kv)).  Any S; built for S * H / H_kv up to a
            few tens of rows (the cache is read once per 16 of them, 32 for
            head_dim up to 64).
        lengths: (B,) int32 cached tokens of each sequence, the new ones included.
        causal: query i of sequence b sees tokens j <= starts[b] + i.
        starts: (B,) int32 position of each sequence's first query (default
            lengths - S); for a batch whose sequences have different counts of
            new tokens, pass what kv_cache_append got (rows behind a count are
            padding: what they give means nothing).
        sm_scale, return_softmax_lse: as in flash_attn_forward (a scale that is not
            finite is refused).

    Returns:
        out (B, S, H, D), with return_softmax_lse also lse (B, H, S) fp32.  A row
        that sees no token gets out 0 and lse +inf.
    """
    assert q.dtype == cache.dtype, f"q must have the cache's dtype {cache.dtype}"
    assert not (q.requires_grad and torch.is_grad_enabled()), _INFERENCE
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(cache.head_dim)
    ops.load()
    fn = torch.ops.fav.decode_lse if return_softmax_lse else torch.ops.fav.decode
    try:
        out = fn(q, cache.k_pages, cache.v_pages, page_table, lengths, starts, causal, sm_scale)
    except RuntimeError:
        _check_decode(q, cache, page_table, lengths, starts, sm_scale)
        raise
    dev = cache.device
    ops.note_device(dev.index)
    if _lib.debug_sync():
        _lib.check_status(dev)
    return out
