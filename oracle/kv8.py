"""CPU oracle (test infra) of the 8-bit decode cache: the ring of
msq_relattn_decode with e4m3 codes and a power-of-two scale for each (block of
slots, head), written position by position, and the decode attention over it,
all in 64 bits."""
import math

import numpy as np


def e4m3_value(code):
    """The value of e4m3 codes (uint8 array): 4 exponent bits (bias 7), 3 mantissa bits, no infinity."""
    c = np.asarray(code).astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


_GRID = e4m3_value(np.arange(127))  # 0 .. 448, ascending


def e4m3_round(y):
    """y (|y| <= 448 or NaN) to the nearest e4m3 value, ties to the even code."""
    a = np.abs(np.nan_to_num(y))
    hi = np.clip(np.searchsorted(_GRID, a), 1, 126)
    lo = hi - 1
    dl, dh = a - _GRID[lo], _GRID[hi] - a
    pick = np.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, lo)
    return np.where(np.isnan(y), np.nan, np.copysign(_GRID[pick], y))


def scale_of(amax):
    """The smallest power of two 2^e, e >= -126, with amax <= 448 * 2^e."""
    e = -126
    while amax > math.ldexp(448.0, e):
        e += 1
    return math.ldexp(1.0, e)


class Ring:
    """One of the two tensors (keys or values) of one row of the batch: [H, S_ring, hs]."""

    def __init__(self, H, S_ring, hs, n_meta, block):
        self.n_meta, self.ctx, self.block = n_meta, S_ring - n_meta, block
        self.val = np.zeros((H, S_ring, hs))                      # codes' values, without the scale
        self.scale = np.ones((H, -(-S_ring // block)))
        self.last = -n_meta - 1

    def slot(self, p):
        return p + self.n_meta if p < 0 else self.n_meta + p % self.ctx

    def window(self, last=None):
        """Slots of the window, oldest first."""
        last = self.last if last is None else last
        return ([self.slot(p) for p in range(-self.n_meta, min(0, last + 1))] +
                [self.slot(p) for p in range(max(0, last + 1 - self.ctx), last + 1)])

    def write(self, x, p0):
        """x [T, H, hs] (64-bit) at positions p0 ..: the whole call's rows are taken before a scale is set."""
        if p0 < -self.n_meta:
            return
        old = set(self.window(p0 - 1))
        new = {}
        for t in range(len(x)):
            new[self.slot(p0 + t)] = x[t]
        for g in sorted({s // self.block for s in new}):
            slots = [s for s in range(g * self.block, min((g + 1) * self.block, self.val.shape[1]))
                     if s in new or s in old]
            for h in range(self.val.shape[0]):
                c = np.stack([new[s][h] if s in new else self.val[h, s] * self.scale[h, g] for s in slots])
                fin = np.abs(c[np.isfinite(c)])
                sc = scale_of(fin.max() if fin.size else 0.0)
                y = c / sc
                top = 448.0 if sc < 2.0 ** 120 else 240.0             # 256 * 2^120 is no fp32 number
                self.val[h, slots] = e4m3_round(np.where(np.isnan(y), y, np.clip(y, -top, top)))
                self.scale[h, g] = sc
        self.last = p0 + len(x) - 1

    def rows(self, last=None):
        """The window's rows [H, S, hs], oldest first."""
        w = self.window(last)
        return self.val[:, w] * self.scale[:, [s // self.block for s in w]][..., None]


def attend(q, k, v, R, scale):
    """q [H, hs], k / v [H, S, hs] oldest first, R [H, >= S, hs] -> [H, hs] (zeros for S = 0)."""
    S = k.shape[1]
    if S == 0:
        return np.zeros_like(q)
    s = np.einsum("hjd,hd->hj", k + R[:, :S], q) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    return np.einsum("hj,hjd->hd", p / p.sum(-1, keepdims=True), v)
