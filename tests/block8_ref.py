"""Plain 64-bit forms of the 8-bit page operators: page tables as lists, codes and
attention in float64 on the host."""
from __future__ import annotations

import numpy as np
import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
BAD, NO_PAGES, NOT_FINITE = 1, 2, 4


class Tables:
    """Page tables kept as lists; ``free`` is a stack."""

    def __init__(self, n, max_pages, pool_pages, block):
        self.pages = [[] for _ in range(n)]
        self.max_pages, self.block = max_pages, block
        self.free = list(range(pool_pages - 1, -1, -1))

    def update(self, lengths, new, rows):
        """(starts, slot_map, lengths, granted, status bits) after keeping and adding rows."""
        b, status, asks, start = self.block, 0, [], 0
        starts = []
        for pages, keep, add in zip(self.pages, lengths, new):
            starts.append(min(start, rows))
            fits = (keep >= 0 and add >= 0 and keep <= len(pages) * b and keep + add <= self.max_pages * b
                    and start + add <= rows)
            start += max(add, 0)
            asks.append((keep, add, fits, -(-(keep + add) // b)))
        starts.append(min(start, rows))
        released = []
        for pages, (_, _, fits, need) in zip(self.pages, asks):
            if fits:  # a request's pages are released in order
                released += pages[need:]
                del pages[need:]
        self.free.extend(reversed(released))  # the first released page is on top
        top, asked = len(self.free), 0
        slots, lens, granted = [-1] * rows, [], []
        for i, (pages, (keep, add, fits, need)) in enumerate(zip(self.pages, asks)):
            want = max(0, need - len(pages)) if fits else 0
            asked += want
            ok = fits and (want == 0 or asked <= top)
            status |= 0 if fits else BAD
            status |= NO_PAGES if fits and not ok else 0
            if ok:
                pages.extend(self.free.pop() for _ in range(want))
                for r in range(add):
                    p = keep + r
                    slots[starts[i] + r] = pages[p // b] * b + p % b
            granted.append(add if ok else 0)
            lens.append(min(max(keep, 0), len(pages) * b) + granted[-1] if not ok else keep + add)
        return starts, slots, lens, granted, status


def step_of(dtype, x):
    """Distance of neighbouring codes at magnitudes |x| (codes' units)."""
    if dtype == torch.int8:
        return np.ones_like(x)
    e = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6)))
    return 2.0 ** (e - 3)


def dequant(codes, scale):
    """float64 values of pages [pages, H, b, D]."""
    s = scale.double().cpu().numpy().clip(2.0 ** -64, 2.0 ** 32)
    return codes.cpu().float().double().numpy() * s[:, :, None, None]


def rows_of(values, table, length, block):
    """[H, length, D] of one request from dequantised pages."""
    pages = values[np.asarray(table[:-(-length // block)], dtype=np.int64)] if length else values[:0]
    h, d = values.shape[1], values.shape[3]
    return pages.transpose(1, 0, 2, 3).reshape(h, -1, d)[:, :length]


def attend(q, k, v, length, scale, window):
    """q [m, Hq, D] float64 over k, v [H, length, D]: out and a bound of its error.

    The bound counts the roundings: bf16 output 2^-8 of the value; each weight to
    fp16 (2^-11) and from its score's error, which is fp32 sums over D products
    (each 2^-24 of the sum of magnitudes) and the terms of the exponent; twice, for
    numerator and denominator. Weights below 2^-21 of the largest are fp16
    subnormals: 2^-32 of it each (2^-30 where V scales differ by up to 4)."""
    m, hq, d = q.shape
    g = hq // k.shape[0]
    out, tol = np.zeros((m, hq, d)), np.zeros((m, hq, d))
    for r in range(m):
        p = length - m + r
        lo, hi = (max(0, p - window + 1) if window else 0), p + 1
        if hi <= lo or hi <= 0:
            continue
        for h in range(hq):
            kk, vv = k[h // g, lo:hi], v[h // g, lo:hi]
            s = kk @ q[r, h] * scale
            mag = float((np.abs(kk) @ np.abs(q[r, h])).max() * abs(scale))
            w = np.exp(s - s.max())
            w /= w.sum()
            out[r, h] = w @ vv
            delta = 2.0 ** -24 * ((d + 8) * mag + 4 * (np.abs(s).max() + 128))
            tol[r, h] = (2.0 ** -8 * np.abs(out[r, h]) + 2 * (2.0 ** -11 + 2 * delta) * (w @ np.abs(vv))
                         + len(w) * 2.0 ** -30 * w.max() * np.abs(vv).max() + 1e-30)
    return out, tol
