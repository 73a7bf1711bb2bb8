"""Reference of shared-prefix attention in 64 bits, and what its result may be off by."""
from __future__ import annotations

import torch

BF16 = torch.bfloat16


def attend(q, keys, values, pos, scale, *, window=0, cap=0.0, slopes=None, visible=None):
    """(answer, allowed error) for one session, float64: q [Hq, Q, D] at positions pos [Q] over
    keys, values [Hkv, T, D], key j at position j; visible [T] bool: a mask on top.

    Allowed: the answer's rounding (2^-8 relative) and weights that are off by a factor of
    1 + e. A product's sum of D exact terms errs by at most 2^-24 per addition of its running
    value, below the sum of magnitudes (D / 8 additions deep at most: a matrix instruction adds
    8 terms and more at once); a score's own operations (scale, tanh by 1 - 2 / (exp + 1) or
    its series, bias, max) by 2^-19 of it (2^-22 without a cap); exponential and two-term
    weights by 2^-16. e is twice that, since sum and products both carry it; it weighs the
    answer's sum of magnitudes."""
    hq, n, d = q.shape
    g = hq // keys.shape[0]
    q, keys, values = q.double(), keys.double(), values.double()
    k, v = keys.repeat_interleave(g, 0), values.repeat_interleave(g, 0)
    at = torch.arange(k.shape[1], device=q.device)
    pos = torch.as_tensor(pos, device=q.device)
    seen = at[None] <= pos[:, None]
    if window:
        seen = seen & (at[None] > pos[:, None] - window)
    if visible is not None:
        seen = seen & visible[None]
    hide = ~seen[None]
    clean_k, clean_v = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
    used = seen.any(0)  # rows that nobody sees may hold anything
    k = torch.where(used[None, :, None], k, clean_k)
    w = torch.matmul(q, k.transpose(1, 2)) * scale
    mag = (torch.matmul(q.abs(), clean_k.abs().transpose(1, 2)) * abs(scale)).masked_fill(hide, 0)
    if cap:
        w = cap * torch.tanh(w / cap)
    if slopes is not None:
        w = w + slopes.double()[:, None, None] * (at[None] - pos[:, None])[None]
    big = w.abs().masked_fill(hide, 0).nan_to_num(0, 0, 0).amax(-1, keepdim=True)
    slack = 2.0 ** -24 * (d / 8) * mag.amax(-1, keepdim=True) + 2.0 ** (-19 if cap else -22) * (big + 1) + 2.0 ** -16
    w = w.masked_fill(hide, float("-inf"))
    none = ~seen.any(1)
    p = torch.softmax(w.masked_fill(none[None, :, None], 0.0), -1) * (~none)[None, :, None]
    o = torch.empty((hq, n, d), dtype=torch.float64, device=q.device)
    for i in range(n):  # a row's products take only what it sees
        o[:, i] = torch.matmul(p[:, i:i + 1], torch.where(seen[i][None, :, None], v, torch.zeros_like(v)))[:, 0]
    total = torch.matmul(p.nan_to_num(0), clean_v.abs())
    return o, 2.0 ** -8 * o.abs() + 2 * torch.expm1(2 * slack) * total + 1e-30


class Sessions:
    """A runtime of one layer whose sessions (slots 0 ..) stand behind a prefix (the last slot)."""

    def __init__(self, gen, lens, prefix, *, hkv, d, layout="contig", window=0, q=1, block=16, spare=8, ring=None,
                 poison=True, capacity=None):
        from kvrt import KVRuntime, LayerSpec

        n = len(lens)
        ring_rows = (ring or window + max(q, 2) - 1) if layout == "ring" else 0
        spec = LayerSpec(kv_heads=hkv, head_dim=d, layout=layout, window=window, ring_rows=ring_rows)
        cap = capacity or max([*lens, prefix, 1]) + spare
        pages = sum(-(-(x + spare) // block) for x in [*lens, prefix]) + 2
        self.rt = KVRuntime([spec], n_slots=n + 1, capacity=cap, max_q=2, block_size=block,
                            pool_pages=pages if layout == "paged" else 0, pool_seed=7)
        if poison:  # rows that hold nothing yet
            for t in self.rt.storage(0)[:2]:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        self.n, self.prefix, self.lens, self.window, self.hkv, self.d = n, prefix, list(lens), window, hkv, d
        self.gen = gen
        self.k, self.v = [], []
        for i, rows in enumerate([*lens, prefix]):
            k, v = (torch.randn(hkv, rows, d, generator=gen, device="cuda").to(BF16) for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            self.load(i)

    def load(self, slot):
        """(Again) the rows of a slot, as self.k and self.v hold them."""
        self.rt.truncate(slot, 0)
        if self.k[slot].shape[1]:
            self.rt.import_(slot, 0, self.k[slot][None].contiguous(), self.v[slot][None].contiguous())

    def append(self, k, v):
        """k, v [n, Hkv, Q, D] to every session."""
        self.rt.append(0, k, v, range(self.n))
        for i in range(self.n):
            self.k[i], self.v[i] = torch.cat((self.k[i], k[i]), 1), torch.cat((self.v[i], v[i]), 1)
            self.lens[i] += k.shape[2]

    def check(self, got, q, scale, *, shared=True, cap=0.0, slopes=None, masks=None):
        """got against the reference; masks: per slot a bool [P] or None."""
        qn = q.shape[2]
        for i in range(self.n):
            parts = ([self.n] if shared else []) + [i]
            keys, values = (torch.cat([x[j] for j in parts], 1) for x in (self.k, self.v))
            visible = None
            if masks is not None:
                flat = []
                for j in parts:
                    m = torch.ones(self.k[j].shape[1], dtype=torch.bool, device="cuda")
                    if masks[j] is not None:
                        m[:masks[j].numel()] = masks[j][:m.numel()]
                    flat.append(m)
                visible = torch.cat(flat)
            total = keys.shape[1]
            want, tol = attend(q[i], keys, values, list(range(total - qn, total)), scale, window=self.window, cap=cap,
                               slopes=slopes, visible=visible)
            off = (got[i].double() - want).abs()
            # (an infinity times a weight of two terms may be NaN)
            ok = (off <= tol) | (~want.isfinite() & ~got[i].isfinite())
            assert bool(ok.all()), (i, int((~ok).sum()), float((off - tol).nan_to_num(9e9).max()))
