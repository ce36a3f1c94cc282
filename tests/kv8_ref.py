"""64-bit plain forms of the 8-bit paged cache and of normed and rotated heads, on the CPU from
the definitions, with their tolerances (roundings counted as in serving_ref)."""
from __future__ import annotations

import math

import numpy as np
import torch

from tests import serving_ref as ref

LOWEST, HIGHEST, LARGEST = -40, 40, 448.0

#: The 256 values of e4m3: sign, four bits of exponent (bias 7), three of mantissa; 0x7f is NaN.
VALUES = np.array([(-1.0) ** (b >> 7) * (math.nan if b & 127 == 127 else (b & 7) * 2.0 ** -9 if b & 120 == 0
                                         else (8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10)) for b in range(256)])


def encode(x):
    """The codes of the values nearest to x (ties to even codes, ends at +-448, NaN for what is not finite)."""
    x = np.asarray(x, dtype=np.float64)
    grid = VALUES[:127]
    size = np.minimum(np.abs(np.where(np.isfinite(x), x, 0.0)), LARGEST)
    hi = np.minimum(np.searchsorted(grid, size, side="left"), 126)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - size, size - grid[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(grid[hi] == size, hi, code) | np.where(np.signbit(x), 128, 0)
    return np.where(np.isfinite(x), code, 127).astype(np.uint8)


def exponent(amax):
    """ceil(log2(amax / 448)) within the bounds, exactly."""
    if amax == 0:
        return LOWEST
    m, e = math.frexp(amax)
    return min(max(e - 9 if m <= 0.875 else e - 8, LOWEST), HIGHEST)


def half_step(x, e):
    """Half a step of e4m3 at x under scale 2^e."""
    size = np.maximum(np.abs(x) * 2.0 ** -e, 2.0 ** -6)
    return 2.0 ** (np.floor(np.log2(size)) - 4 + e)


class Cache:
    """Codes and scales' exponents of K and V, [pages][heads][page or page / block]([hd])."""

    def __init__(self, pages, hkv, page, hd, block):
        self.codes = [np.full((pages, hkv, page, hd), 127, dtype=np.uint8) for _ in range(2)]
        self.scales = [np.full((pages, hkv, page // block), 255, dtype=np.uint8) for _ in range(2)]
        self.page, self.block = page, block

    def append(self, which, table, ctx, new, errors):
        """`new` [n][heads][hd] in 64 bits to the slots from ctx on of a sequence with this page
        table, from values that are off by at most `errors`; returns [n][heads] of whether a
        rounding's direction cannot be told (the scale's own border is met by an error)."""
        n, block, codes, scales = len(new), self.block, self.codes[which], self.scales[which]
        unsure = np.zeros(new.shape[:2], dtype=bool)
        if n == 0:
            return unsure
        for first in range(ctx // block * block, ctx + n, block):
            p, off = table[first // self.page], first % self.page
            lo, hi = max(first, ctx), min(first + block, ctx + n)
            for h in range(new.shape[1]):
                x, dx = new[lo - ctx:hi - ctx, h], errors[lo - ctx:hi - ctx, h]
                size = np.where(np.isfinite(x), np.abs(x), 0.0)
                e = exponent(size.max())
                unsure[lo - ctx:hi - ctx, h] = exponent((size + dx).max()) != exponent(max((size - dx).max(), 0.0))
                if first < ctx:
                    before = min(max(int(scales[p, h, off // block]) - 127, LOWEST), HIGHEST)
                    e = max(e, before)
                    if e > before:
                        kept = codes[p, h, off:off + ctx - first]
                        codes[p, h, off:off + ctx - first] = encode(VALUES[kept] * 2.0 ** (before - e))
                codes[p, h, lo % self.page:lo % self.page + hi - lo] = encode(x * 2.0 ** -e)
                scales[p, h, off // block] = e + 127
        return unsure

    def tensors(self, device):
        k, v = (torch.from_numpy(c.copy()).to(device).view(torch.float8_e4m3fn) for c in self.codes)
        ks, vs = (torch.from_numpy(c.copy()).to(device).view(torch.float8_e8m0fnu) for c in self.scales)
        return k, v, ks, vs

    def values(self, which):
        e = np.clip(self.scales[which].astype(np.int64) - 127, LOWEST, HIGHEST)
        return VALUES[self.codes[which]] * np.repeat(2.0 ** e, self.block, axis=2)[..., None]


def normed(x, weight, eps):
    """(x rsqrt(mean(x^2) + eps) w in 64 bits, its relative error in fp32): a sum of hd squares is
    off by at most hd 2^-24 of itself, half of that behind the root; rsqrtf by 2 steps; the
    division, the sum with eps and two products by half a step each."""
    x = x.detach().cpu().double().numpy()
    if weight is None:
        return x, 0.0
    hd = x.shape[-1]
    w = weight.detach().cpu().double().numpy()
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w, (hd / 2 + 8) * 2.0 ** -24


def turned(x, weight, eps, positions, freq, interleaved):
    """(normed and rotated x in 64 bits, bound of an fp32 computation's error before any rounding
    to the storage type); freq None: not rotated."""
    y, rel = normed(x, weight, eps)
    if freq is None:
        return y, rel * np.abs(y) if rel else np.zeros_like(y)
    out, pair = ref.rotated(torch.from_numpy(y), positions, freq, 1.0, interleaved)
    moved = pair > 0
    return out, np.where(moved, (rel + 4 * 2.0 ** -24) * pair + 2.0 ** -32, rel * np.abs(y))
