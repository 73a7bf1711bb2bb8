"""The codes of 8-bit pages, bit for bit, against a replay of every append on the host.

The arithmetic is fixed: amax / top, 1 / scale and old / scale are single fp32 divisions,
a code is one fp32 product rounded to the nearest code (ties to even). So the codes
of a whole run of updates, appends, rollbacks and growing scales are known exactly, and
a row that is lost, shifted or left out by a recoding shows."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import block8_ref as R
from tests.helpers import randn_bf16

pytestmark = pytest.mark.gpu

I8, F8 = torch.int8, torch.float8_e4m3fn
LOW, HIGH = np.float32(2.0 ** -64), np.float32(2.0 ** 32)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Codes:
    """One tensor of a pool on the host: raw codes [pages, H, b, D] and fp32 scales."""

    def __init__(self, pages, heads, block, dim, dtype):
        self.dtype, self.block, self.top = dtype, block, np.float32(R.TOP[dtype])
        self.raw = np.zeros((pages, heads, block, dim), np.uint8)
        self.scale = np.zeros((pages, heads), np.float32)

    def floats(self, raw):
        return torch.from_numpy(raw.copy()).view(self.dtype).float().numpy()

    def code(self, x):
        """fp32 values in units of the scale to raw codes."""
        x = np.clip(x, -self.top, self.top)
        t = torch.from_numpy(np.rint(x).astype(np.int8)) if self.dtype == I8 else torch.from_numpy(x).to(F8)
        return t.view(torch.uint8).numpy()

    def append(self, x, slots):
        """Rows x [T, H, D] (finite fp32) into slots, run by run."""
        runs = []
        for t, s in enumerate(slots):
            if s < 0:
                continue
            if runs and runs[-1][0] + len(runs[-1][1]) == s and s % self.block and runs[-1][1][-1] == t - 1:
                runs[-1][1].append(t)
            else:
                runs.append((s, [t]))
        for first, rows in runs:
            p, off, m = first // self.block, first % self.block, len(rows)
            for h in range(x.shape[1]):
                v = x[rows, h]
                s = np.clip(np.abs(v).max() / self.top, LOW, HIGH)
                if off:
                    old = np.clip(self.scale[p, h], LOW, HIGH)
                    s = np.maximum(s, old)
                    if s > old:
                        before = self.floats(self.raw[p, h, :off])
                        self.raw[p, h, :off] = self.code(before * (old / s))
                self.scale[p, h] = s
                self.raw[p, h, off:off + m] = self.code(v * (np.float32(1) / s))


def _equal(host, codes, scale):
    return np.array_equal(host.raw, codes.cpu().contiguous().view(torch.uint8).numpy()) and \
        np.array_equal(host.scale, scale.cpu().numpy())


@pytest.mark.parametrize("name", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,dim,block", [(8, 128, 16), (1, 256, 32), (2, 64, 64), (1, 512, 16)])
def test_every_code_of_a_serving_run(name, heads, dim, block):
    from kvrt import Block8Pool, BlockTables

    gen = torch.Generator().manual_seed(dim + block)
    n, pages, dtype = 4, 60, {"int8": I8, "e4m3": F8}[name]
    tables, ref = BlockTables(n, 16, pages, block_size=block), R.Tables(n, 16, pages, block)
    pool = Block8Pool.zeros(pages, heads, dim, block_size=block, dtype=name)
    host = [Codes(pages, heads, block, dim, dtype) for _ in range(2)]
    lens, grown = [0] * n, 0
    steps = [([0] * n, [40, 7, 100, 0])] + [(None, [1, 1, 1, 0])] * 4
    steps += [([38, 9, 90, 0], [1, 2, 30, 60]), (None, [1, 1, 1, 1]), ([0, 5, 100, 50], [0, 3, 1, 9]), (None, [21, 1, 1, 1])]
    steps += [(None, [1, 1, 1, 1])] * 3 + [([7, 0, 33, 58], [2, 90, 1, 1])]
    for step, (keep, new) in enumerate(steps):
        keep = lens if keep is None else [min(a, b) for a, b in zip(keep, lens)]
        rows = sum(new) + step % 3
        want = ref.update(keep, new, rows)
        plan = tables.update(_i32(keep), _i32(new), rows=rows)
        assert plan.slot_map.tolist() == want[1], step
        lens = want[2]
        # magnitudes that grow and shrink: scales of opened pages grow in some steps, stay in others
        x = [randn_bf16(gen, (rows, heads, dim), s) for s in (1.0 + step % 4, 2.0 ** (step % 5 - 2))]
        before = [h.scale.copy() for h in host]
        pool.append(x[0].cuda(), x[1].cuda(), plan.slot_map)
        for h, v in zip(host, x):
            h.append(v.float().numpy(), want[1])
        grown += sum(int(((b > 0) & (h.scale > b)).sum()) for b, h in zip(before, host))
        assert _equal(host[0], pool.k, pool.k_scale) and _equal(host[1], pool.v, pool.v_scale), step
        k, v, mask = pool.gather(tables.table, plan.lengths, max(lens), dtype=torch.float32)
        for got, h in ((k, host[0]), (v, host[1])):
            values = h.floats(h.raw) * np.clip(h.scale, LOW, HIGH)[:, :, None, None]
            for i, length in enumerate(lens):
                assert np.array_equal(got[i, :, :length].cpu().numpy(), R.rows_of(values, ref.pages[i], length, block)), (step, i)
    assert grown > 8  # recodings took place
    assert pool.status() == 0 and tables.status() == 0


@pytest.mark.parametrize("name", ["int8", "e4m3"])
def test_the_replay_tells_lost_and_shifted_rows(name):
    """The comparison itself: a zeroed, a shifted and a not recoded row differ."""
    dtype = {"int8": I8, "e4m3": F8}[name]
    gen = torch.Generator().manual_seed(1)
    x = randn_bf16(gen, (9, 2, 64)).float().numpy()
    x[8] *= 4  # the last row makes the scale grow
    host, stale = Codes(3, 2, 16, 64, dtype), Codes(3, 2, 16, 64, dtype)
    for h in (host, stale):
        h.append(x[:8], [*range(16, 24)])
    before = stale.raw.copy()
    host.append(x[8:], [24])
    stale.append(x[8:], [24])
    codes, scale = torch.from_numpy(host.raw.copy()), torch.from_numpy(host.scale.copy())
    assert _equal(stale, codes, scale)
    stale.raw[1, :, :8] = before[1, :, :8]
    assert not _equal(stale, codes, scale)
    for change in (lambda c: c[1, 0, 3].zero_(), lambda c: c[1].copy_(c[1].roll(1, 1)), lambda c: c[1, 1, 8].copy_(c[1, 1, 7])):
        bad = codes.clone()
        change(bad)
        assert not _equal(host, bad, scale)
