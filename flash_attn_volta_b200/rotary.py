"""Rotary positions for q and k: fav::rotary / fav::rotary_qk (csrc/fa_rotary.cu).

With a = position * inv_freq[i] (in 64 bits, so far positions keep their
angle) each pair (x1, x2) of the first 2 * len(inv_freq) dims of a head becomes
(M (x1 cos a - x2 sin a), M (x2 cos a + x1 sin a)); the dims behind are kept.
Pairs are dims (i, i + R/2), or (2 i, 2 i + 1) with ``interleaved``.  Scaling for
long contexts changes inv_freq and the magnitude M only (``Rotary.build``).
``flash_attn(..., rotary=...)`` and ``ring.ring_flash_attn(..., rotary=...)`` apply
it to their q and k, ``kv_cache.kv_cache_append`` on the way into a cache.

The reference has no rotary operator (its patched models rotate q and k in
their own code).
"""
from __future__ import annotations

import math

import torch

from . import ops


class Rotary:
    """Frequencies and pairing of a rotary embedding.

    Args:
        inv_freq: 1-D tensor of R/2 angular frequencies (radians per position)
            on the device of the tensors to rotate; used in fp64 (any other
            floating type is converted here, once).  Gets no gradient: one that
            requires it is refused.
        interleaved: pairs (2 i, 2 i + 1) instead of (i, i + R/2).
        magnitude: factor on cos and sin (1 but for some long-context scalings).
    """
    __slots__ = ("inv_freq", "interleaved", "magnitude")

    def __init__(self, inv_freq: torch.Tensor, interleaved: bool = False, magnitude: float = 1.0):
        assert inv_freq.dim() == 1 and inv_freq.shape[0] > 0 and inv_freq.is_floating_point(), \
            "inv_freq must be a 1-D floating-point tensor of R/2 frequencies"
        self.inv_freq = inv_freq if inv_freq.dtype == torch.float64 else inv_freq.double()
        self.interleaved = bool(interleaved)
        self.magnitude = float(magnitude)

    @property
    def dim(self) -> int:
        """Rotated dims of a head."""
        return 2 * self.inv_freq.shape[0]

    @classmethod
    def build(cls, dim: int, base: float = 10000.0, *, interleaved: bool = False,
              scaling: str | None = None, factor: float = 1.0,
              trained_length: int | None = None, device="cuda") -> "Rotary":
        """inv_freq[i] = base ** (-2 i / dim), i < dim / 2, scaled for contexts
        ``factor`` times as long as the ``trained_length``:

        * None: as it is.
        * "linear": positions interpolated, inv_freq / factor.
        * "ntk": base * factor ** (dim / (dim - 2)), which divides the lowest
          frequency by ``factor`` and keeps the highest.
        * "yarn": frequencies that make r = trained_length * inv_freq / (2 pi)
          turns over the trained length are kept for r >= 32, divided by
          ``factor`` for r <= 1 and mixed linearly in r between; the magnitude
          is 0.1 ln(factor) + 1.
        """
        assert dim >= 2 and dim % 2 == 0, f"rotary dim {dim} must be even"
        assert scaling in (None, "linear", "ntk", "yarn"), f"unknown scaling {scaling!r}"
        assert factor >= 1.0, "factor must be at least 1"
        i = torch.arange(dim // 2, dtype=torch.float64)
        if scaling == "ntk":
            assert dim > 2, "ntk scaling needs more than one frequency"
            base = base * factor ** (dim / (dim - 2))
        inv = base ** (-2.0 * i / dim)
        magnitude = 1.0
        if scaling == "linear":
            inv = inv / factor
        elif scaling == "yarn":
            assert trained_length is not None and trained_length > 0, "yarn needs trained_length"
            keep = ((trained_length * inv / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
            inv = inv / factor * (1.0 - keep) + inv * keep
            magnitude = 0.1 * math.log(factor) + 1.0
        return cls(inv.to(device), interleaved, magnitude)


_NO_GRADIENT = "inv_freq gets no gradient: detach it"


def _check(x: torch.Tensor, rotary: Rotary, positions, k=None) -> None:
    """Raise AssertionError for a call the operators refuse."""
    shape, dev = x.shape, x.device
    assert dev.type == "cuda", "tensors must be on CUDA"
    assert x.dtype in (torch.float16, torch.bfloat16), "fp16 (or bf16) only"
    assert len(shape) == 4, "expected (batch, seqlen, heads, head_dim)"
    assert shape[3] % 2 == 0 and rotary.dim <= shape[3], \
        f"rotary dim {rotary.dim} does not fit head_dim {shape[3]}"
    assert rotary.inv_freq.device == dev, "inv_freq must be on the tensors' device"
    assert not (rotary.inv_freq.requires_grad and torch.is_grad_enabled()), _NO_GRADIENT
    if positions is not None:
        assert positions.device == dev, "positions must be on the tensors' device"
        assert positions.dtype in (torch.int32, torch.int64), "positions must be int32 or int64"
        assert positions.shape in (shape[:2], shape[1:2]), \
            f"positions must be (seqlen,) or (batch, seqlen), got {tuple(positions.shape)}"
    if k is not None:
        ks = k.shape
        assert len(ks) == 4 and shape[:2] == ks[:2] and shape[3] == ks[3], \
            f"qk shape mismatch {shape} {ks}"
        assert k.dtype == x.dtype and k.device == dev, "q and k must have one dtype and device"


# The operators check their arguments themselves; the assertions, which say what
# is wrong in this module's terms, run when one refuses (they cost as much host
# time as a small call's launch).
def rotary_embed(x: torch.Tensor, rotary: Rotary, positions: torch.Tensor | None = None,
                 first: int = 0) -> torch.Tensor:
    """x (B, S, H, D), fp16 or bf16, any strides, rotated; autograd-aware.

    positions: (S,) or (B, S) int32 / int64; None: first, first + 1, ...
    The result is contiguous, in x's dtype; sums are in fp32, rounded once.
    Reverse-mode derivatives only: a forward-mode tangent is refused.
    """
    ops.load()
    try:
        return torch.ops.fav.rotary(x, rotary.inv_freq, positions, first, rotary.interleaved,
                                    rotary.magnitude, False)
    except RuntimeError:
        _check(x, rotary, positions)
        raise


def rotary_embed_qk(q: torch.Tensor, k: torch.Tensor, rotary: Rotary,
                    positions: torch.Tensor | None = None,
                    first: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """rotary_embed of q (B, S, H, D) and k (B, S, H_kv, D) at the same
    positions, in one launch (and one for both gradients)."""
    ops.load()
    try:
        return torch.ops.fav.rotary_qk(q, k, rotary.inv_freq, positions, first,
                                       rotary.interleaved, rotary.magnitude, False)
    except RuntimeError:
        _check(q, rotary, positions, k)
        raise


def rotate_for_attention(q, k, rotary: Rotary, positions=None):
    """q (B, N, H, D) and k (B, N_k, H_kv, D) of one attention call rotated.
    ``positions`` are the keys' ((N_k,) or (B, N_k), default 0 ..); the queries
    are the last N of them, as in the causal mask's alignment."""
    N, Nk = q.shape[1], k.shape[1]
    if N == Nk:
        return rotary_embed_qk(q, k, rotary, positions)
    if positions is None:
        return rotary_embed(q, rotary, first=Nk - N), rotary_embed(k, rotary)
    assert N <= Nk, "positions of more queries than keys: rotate q and k with rotary_embed"
    return (rotary_embed(q, rotary, positions[..., Nk - N:]), rotary_embed(k, rotary, positions))
