"""The 8-bit cache from its definition, slowly, on the CPU: what a page holds after a step's rows have come, and attention
over it in 64 bits."""
import math

import numpy as np
import torch

PAGE = 64
E_MIN, E_MAX = -60, 40

# the e4m3 numbers by their bytes: 4 bits of exponent (bias 7), 3 of mantissa, 0x7f and 0xff NaN
VALUES = torch.tensor([(-1.0 if b >> 7 else 1.0) * (math.nan if b & 0x7f == 0x7f else
                       (b & 7) * 2.0 ** -9 if (b >> 3) & 15 == 0 else (1 + (b & 7) / 8) * 2.0 ** (((b >> 3) & 15) - 7))
                       for b in range(256)], dtype=torch.float64)
_POSITIVE = VALUES[:0x7f].numpy()                                     # 0 .. 448, ascending


def to_bytes(x):
    """The nearest e4m3 numbers of float64 values, ties to the even byte, magnitudes above 448 held there, NaN for what is not finite."""
    a = x.abs().double().numpy()
    finite = np.isfinite(a)
    a = np.minimum(np.where(finite, a, 0.0), 448.0)
    hi = np.clip(np.searchsorted(_POSITIVE, a), 1, len(_POSITIVE) - 1)
    lo = hi - 1
    d_lo, d_hi = a - _POSITIVE[lo], _POSITIVE[hi] - a
    byte = np.where((d_lo < d_hi) | ((d_lo == d_hi) & (lo % 2 == 0)), lo, hi)
    byte = np.where(finite, byte, 0x7f) | (np.signbit(x.double().numpy()) << 7)
    return torch.from_numpy(byte.astype(np.uint8))


def exponent(most: float) -> int:
    if most == 0:
        return E_MIN
    e = math.frexp(most)[1] - 9                                       # 448 * 2^e = 0.875 * 2^(9 + e)
    while 448.0 * 2.0 ** e < most:
        e += 1
    while 448.0 * 2.0 ** (e - 1) >= most:
        e -= 1
    return min(max(e, E_MIN), E_MAX)


def rotate(x, pos, cos, sin, rot, pairing):
    """x float32 [heads, hd] at `pos`: products and sums rounded one by one, as the cache's writer has them."""
    y = x.clone()
    if cos is None:
        return y
    c, s = cos[pos], sin[pos]
    if pairing == "half":
        ia, ib = slice(0, rot // 2), slice(rot // 2, rot)
    else:
        ia, ib = slice(0, rot, 2), slice(1, rot, 2)
    a, b = x[:, ia], x[:, ib]
    y[:, ia], y[:, ib] = a * c - b * s, a * s + b * c
    return y


class PlainCache:
    """bytes [pages, G, 64, hd] and exponents [pages, G] of keys and of values."""

    def __init__(self, k_bytes, v_bytes, k_scale, v_scale):
        self.bytes = [k_bytes.clone(), v_bytes.clone()]
        self.scale = [k_scale.double().clone(), v_scale.double().clone()]

    def append(self, rows, which, pages, pos0):
        """rows float32 [n, G, hd] at positions pos0 .. of the sequence whose pages are `pages`."""
        held, scale = self.bytes[which], self.scale[which]
        n, G, _ = rows.shape
        for first in range(0, n):
            p = pos0 + first
            if first and p % PAGE:
                continue
            count = min(n - first, PAGE - p % PAGE)
            page, place = int(pages[p // PAGE]), p % PAGE
            if page == 0:
                continue
            for g in range(G):
                x = rows[first:first + count, g].double()
                fin = x[torch.isfinite(x)].abs()
                e = exponent(float(fin.max()) if fin.numel() else 0.0)
                if place:
                    e = max(e, int(math.log2(float(scale[page, g]))))
                    held[page, g, :place] = to_bytes(VALUES[held[page, g, :place].long()] * float(scale[page, g]) / 2.0 ** e)
                held[page, g, place:place + count] = to_bytes(x / 2.0 ** e)
                scale[page, g] = 2.0 ** e

    def read(self, which, pages, g, length):
        pages = torch.as_tensor(pages)[:(length + PAGE - 1) // PAGE].long()
        x = VALUES[self.bytes[which][pages, g].long()] * self.scale[which][pages, g][:, None, None]
        return x.reshape(-1, x.shape[-1])[:length]


def visible(p, length, window, keep_first):
    j = torch.arange(length)
    seen = j <= p
    if window and window > 0:
        seen &= (j > p - window) | (j < keep_first)
    elif window and window < 0:
        seen &= j >= p - p % -window
    return seen


def attend(q, p, cache, pages, G, scale, window=None, sink=None, keep_first=0, slopes=None):
    """One query token, q [H, hd] float64 at position p: (out [H, hd], sum_j w_j |v_j| [H, hd], max_j sum_i |q_i k_ji| scale [H]);
    keys that it does not see are not looked at."""
    H, hd = q.shape
    out, weight, size = torch.zeros(H, hd, dtype=torch.float64), torch.zeros(H, hd, dtype=torch.float64), torch.zeros(H, dtype=torch.float64)
    seen = visible(p, p + 1, window, keep_first)
    j = torch.arange(p + 1)[seen]
    for h in range(H):
        g = h // (H // G)
        k, v = cache.read(0, pages, g, p + 1)[seen], cache.read(1, pages, g, p + 1)[seen]
        s = k @ q[h] * scale
        if slopes is not None:
            s = s - float(slopes[h]) * (p - j)
        top = s.max() if sink is None else torch.maximum(s.max(), sink[h].double())
        w = torch.exp(s - top)
        total = w.sum() + (0 if sink is None else torch.exp(sink[h].double() - top))
        out[h], weight[h] = (w / total) @ v, (w / total) @ v.abs()
        size[h] = (k.abs() @ q[h].abs()).max() * scale
    return out, weight, size
