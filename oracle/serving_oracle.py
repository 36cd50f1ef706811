"""CPU oracle of the rotary positions and of the paged key/value cache — TEST
INFRASTRUCTURE ONLY, in float64, written from the operators' formulas.

* `rotate`  — pairs as complex numbers times M exp(i position inv_freq).
* `four_bit` — the values, minima and scales of 4-bit groups of 32.
* `blocks`  — a 4-bit cache's bytes of given codes, one token and dim at a time
  (the layout of csrc/fa_kv_cache.cuh).
* `decode`  — attention of a sequence's query rows over its keys and values,
  with the sums that bound a kernel's rounding.
"""
from __future__ import annotations

import math

import numpy as np
import torch


def rotate(x, positions, inv_freq, interleaved=False, magnitude=1.0, inverse=False):
    """x (B, S, H, D) in any type -> float64; positions (B, S) or (S,)."""
    x = x.double()
    R = 2 * len(inv_freq)
    pos = torch.as_tensor(positions).double()
    if pos.dim() == 1:
        pos = pos.expand(x.shape[0], -1)
    a = pos[:, :, None, None] * inv_freq.double()
    if inverse:
        a = -a
    lo = slice(0, R, 2) if interleaved else slice(0, R // 2)
    hi = slice(1, R, 2) if interleaved else slice(R // 2, R)
    y = x.clone()
    y[..., lo] = magnitude * (x[..., lo] * a.cos() - x[..., hi] * a.sin())
    y[..., hi] = magnitude * (x[..., hi] * a.cos() + x[..., lo] * a.sin())
    return y


def _directed(x, up):
    """float64 array -> the nearest fp16 not below (up) or not above it."""
    h = x.astype(np.float16)
    wrong = h.astype(np.float64) < x if up else h.astype(np.float64) > x
    return np.where(wrong, np.nextafter(h, np.float16(np.inf if up else -np.inf)), h).astype(np.float64)


def four_bit(x):
    """x (..., D) -> (codes (..., D), m, s (..., D/32)) of its 4-bit groups."""
    g = x.double().numpy().reshape(*x.shape[:-1], -1, 32)
    g = np.clip(g, -65504.0, 65504.0)
    m = _directed(g.min(-1), up=False)
    s = _directed((g.max(-1) - m) / 15.0, up=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s[..., None] > 0, np.rint((g - m[..., None]) / s[..., None]), 0.0)
    return (torch.from_numpy(c).reshape(x.shape), torch.from_numpy(m), torch.from_numpy(s))


def values(codes, m, s):
    return (codes.unflatten(-1, (-1, 32)) * s[..., None] + m[..., None]).flatten(-2)


def block_bytes(kc, km, ks, vc, vm, vs):
    """One block (16 tokens of a head) from codes (16, D) and (16, D/32) minima and
    scales: uint8 array of 20 D bytes."""
    D = kc.shape[1]
    NG = D // 32
    kc, vc = kc.numpy().astype(np.uint64), vc.numpy().astype(np.uint64)
    kw = np.zeros(16 * 4 * NG, dtype=np.uint64)
    vw = np.zeros(2 * 8 * 4 * NG, dtype=np.uint64)
    kp = np.zeros((16 * NG, 2), dtype=np.float16)
    vp = np.zeros((2, NG * 16), dtype=np.float16)
    for r in range(16):
        tp, t, hi = r // 8, r % 8 // 2, r % 2
        for d in range(D):
            grp, e = d // 32, d % 32
            bit = (e % 8 // 2) * 4 + (e % 2) * 16
            kw[(r * 4 + e // 8) * NG + grp] |= kc[r, d] << np.uint64(bit)
            bit = (e % 4) * 4 + hi * 16
            vw[((tp * 8 + e // 4) * 4 + t) * NG + grp] |= vc[r, d] << np.uint64(bit)
        for grp in range(NG):
            kp[r * NG + grp] = ks[r, grp], km[r, grp]
            at = (grp * 4 + t) * 4 + tp * 2 + hi
            vp[0, at], vp[1, at] = vs[r, grp], vm[r, grp]
    parts = (kw.astype(np.uint32), kp, vw.astype(np.uint32), vp)
    return np.concatenate([np.ascontiguousarray(x).reshape(-1).view(np.uint8) for x in parts])


def decode(q, k, v, sizes, limits, scale):
    """q (R, D) query rows, k, v (n, D) and |v|'s bound `sizes` (n, D) in float64;
    row r sees keys j < limits[r].  Returns out (R, D), lse (R,), and per row
    sum_j p_j sizes_j (R, D) and max_j |scale| sum_d |q_d k_jd|."""
    R, D = q.shape
    out, lse = torch.zeros(R, D, dtype=torch.float64), torch.full((R,), math.inf, dtype=torch.float64)
    mass, reach = torch.zeros(R, D, dtype=torch.float64), torch.zeros(R, dtype=torch.float64)
    for r in range(R):
        n = max(0, min(int(limits[r]), k.shape[0]))
        if n == 0:
            continue
        sc = (k[:n] @ q[r]) * scale
        lse[r] = torch.logsumexp(sc, 0)
        p = torch.softmax(sc, 0)
        out[r], mass[r] = p @ v[:n], p @ sizes[:n]
        reach[r] = ((k[:n].abs() @ q[r].abs()) * abs(scale)).max()
    return out, lse, mass, reach
