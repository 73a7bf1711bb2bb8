"""8-bit pages with one scale per page and head, against plain 64-bit forms: the
page tables, the codes appended rows become, the padded batch, attention of few
and of many query rows, and steps of all of them together, captured too."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import block8_ref as R
from tests.helpers import bits, randn_bf16

pytestmark = pytest.mark.gpu

I8, F8 = torch.int8, torch.float8_e4m3fn
NAMES = {"int8": I8, "e4m3": F8}


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _codes_bits(t):
    return t.cpu().contiguous().view(torch.uint8).numpy()


# ---- page tables ---------------------------------------------------------------------------


def _compare_tables(t, ref, plan, want, where):
    starts, slots, lens, granted, status = want
    assert plan.starts.tolist() == starts, where
    assert plan.granted.tolist() == granted, where
    assert plan.lengths.tolist() == lens, where
    assert plan.slot_map.tolist() == slots, where
    table = t.table.cpu().numpy()
    for i, pages in enumerate(ref.pages):
        assert table[i, :len(pages)].tolist() == pages, (where, i)
        assert (table[i, len(pages):] == -1).all(), (where, i)
    assert t.mapped.tolist() == [len(p) for p in ref.pages], where
    assert t.free_count.item() == len(ref.free), where
    assert t.free[:len(ref.free)].tolist() == ref.free, where
    assert t.status() == status and t.status() == 0, where


@pytest.mark.parametrize("n,max_pages,pool,block,longest,steps", [
    (1, 4, 4, 16, 40, 30), (3, 20, 24, 16, 200, 40), (7, 9, 40, 64, 400, 30), (64, 12, 300, 32, 250, 12),
    (65, 12, 330, 32, 250, 12), (300, 40, 4000, 16, 500, 6), (1030, 8, 3000, 16, 90, 5),
])
def test_tables_follow_lengths(n, max_pages, pool, block, longest, steps):
    """Growth, rollback, release and refusals, step by step, all outputs equal."""
    from kvrt import BlockTables

    rng = np.random.default_rng(n * 1000 + block)
    t, ref = BlockTables(n, max_pages, pool, block_size=block), R.Tables(n, max_pages, pool, block)
    held = [0] * n
    for step in range(steps):
        keep = [int(h if rng.random() < 0.6 else rng.integers(0, h + 1) if rng.random() < 0.7 else 0) for h in held]
        new = [int(rng.integers(0, longest) if rng.random() < 0.3 else rng.integers(0, 3)) for _ in range(n)]
        if step % 5 == 4:  # numbers that are not possible
            i = int(rng.integers(0, n))
            keep[i], new[i] = [(-1, 2), (3, -2), (keep[i], max_pages * block + 1), (10 ** 9, 1)][step // 5 % 4]
        rows = max(0, sum(max(x, 0) for x in new) + int(rng.integers(-3, 9)))
        if step % 3 == 0:
            rows = sum(max(x, 0) for x in new)
        want = ref.update(keep, new, rows)
        plan = t.update(_i32(keep), _i32(new), rows=rows)
        _compare_tables(t, ref, plan, want, (n, step))
        held = want[2]


def test_tables_of_many_rows_take_two_launches():
    from kvrt import BlockTables

    n, block, width, pool = 37, 16, 600, 12000
    rng = np.random.default_rng(5)
    t, ref = BlockTables(n, width, pool, block_size=block), R.Tables(n, width, pool, block)
    held = [0] * n
    for step in range(4):
        keep = [int(rng.integers(0, h + 1)) for h in held]
        new = [int(rng.integers(0, 900)) if i % 3 else 1 for i in range(n)]
        rows = sum(new) + 700 * (step % 2)
        want = ref.update(keep, new, rows)
        _compare_tables(t, ref, t.update(_i32(keep), _i32(new), rows=rows), want, step)
        held = want[2]
    want = ref.update([0] * n, [0] * n, 0)  # everything released, long tables among them
    _compare_tables(t, ref, t.update(_i32([0] * n), _i32([0] * n), rows=0), want, "end")


def test_lengths_may_be_the_plans_own_and_a_captured_update_replays():
    """A captured decode step: lengths advance in place, pages come as needed."""
    from kvrt import BlockTables

    n, block, pool = 5, 16, 40
    t, ref = BlockTables(n, 8, pool, block_size=block), R.Tables(n, 8, pool, block)
    lengths, new = _i32([3, 15, 16, 0, 31]), _i32([1, 2, 1, 1, 1])
    t.update(torch.zeros_like(lengths), lengths, rows=70)
    ref.update([0] * n, [3, 15, 16, 0, 31], 70)
    want = ref.update([3, 15, 16, 0, 31], [1, 2, 1, 1, 1], 6)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        plan = t.update(lengths, new, rows=6)
        lengths.copy_(plan.lengths)
    side.synchronize()
    _compare_tables(t, ref, plan, want, "eager")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan = t.update(lengths, new, rows=6)
        lengths.copy_(plan.lengths)
    for step in range(20):
        want = ref.update(want[2], [1, 2, 1, 1, 1], 6)
        g.replay()
        torch.cuda.synchronize()
        _compare_tables(t, ref, plan, want, step)


# ---- append -----------------------------------------------------------------------------------


def _append_reference(codes, scale, x, slots):
    """(old codes, allowed error) in 64 bits is checked by the caller; here the exact
    scale after, and for every coded row its exact value in codes' units."""
    block = codes.shape[2]
    top = R.TOP[codes.dtype]
    page = [s // block for s in slots if s >= 0]
    out = {}
    for p in dict.fromkeys(page):
        rows = [(t, s % block) for t, s in enumerate(slots) if s >= 0 and s // block == p]
        first = rows[0][1]
        v = x[[t for t, _ in rows]].astype(np.float64)  # [m, H, D]
        fin = np.where(np.isfinite(v), np.abs(v), 0.0).max((0, 2))
        new = np.clip((fin.astype(np.float32) / np.float32(top)).astype(np.float32), np.float32(2.0 ** -64),
                      np.float32(2.0 ** 32))
        old = np.clip(scale[p], 2.0 ** -64, 2.0 ** 32)
        out[p] = (first, len(rows), np.maximum(new, old) if first > 0 else new, old, v)
    return out


def _near(codes, exact, dtype):
    """codes are the nearest ones to `exact` up to fp32 arithmetic: half a step, and
    2^-22 of the value for the reciprocal and the products."""
    top = R.TOP[dtype]
    want = np.clip(np.nan_to_num(exact, nan=0.0, posinf=top, neginf=-top), -top, top)
    near = np.abs(codes - want) <= 0.5 * R.step_of(dtype, want) + 2.0 ** -22 * np.abs(want)
    return near


@pytest.mark.parametrize("name", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,dim,block", [(2, 64, 16), (8, 128, 16), (1, 256, 32), (1, 512, 16), (3, 128, 64),
                                             (1, 64, 128)])
def test_append_codes_rows(name, heads, dim, block):
    """Runs that begin and end inside pages, whole pages, single rows, skipped rows,
    all in one call; rows around them untouched; the scale grows or stays."""
    from kvrt import Block8Pool

    gen = torch.Generator().manual_seed(heads * dim + block)
    pages = 12
    pool = Block8Pool.zeros(pages, heads, dim, block_size=block, dtype=name)
    # what earlier steps left: codes of every value, scales around 1/50
    raw = torch.randint(-126, 127, (2, pages, heads, block, dim), generator=gen, dtype=torch.int8)
    scales = torch.rand((2, pages, heads), generator=gen) * 0.03 + 0.005
    pool.k.view(I8).copy_(raw[0]), pool.v.view(I8).copy_(raw[1])
    pool.k_scale.copy_(scales[0]), pool.v_scale.copy_(scales[1])
    before = [(_codes_bits(t), s.cpu().numpy().copy()) for t, s in ((pool.k, pool.k_scale), (pool.v, pool.v_scale))]
    vals = [pool.k.float().cpu().double().numpy(), pool.v.float().cpu().double().numpy()]
    slots = [5 * block + 3, -1]                                             # one row, and a skipped one
    slots += list(range(7 * block + block - 5, 7 * block + block))          # up to a page's end ...
    slots += list(range(2 * block, 3 * block))                              # ... on another whole page ...
    slots += list(range(3 * block, 3 * block + 7)) + [-1, -1]               # ... and its neighbour's start
    slots += [0, 9 * block + 1, 9 * block + 2, pages * block - 1, -7]
    x = [randn_bf16(gen, (len(slots), heads, dim)) * s for s in (1.0, 3.0)]
    x[0][slots.index(5 * block + 3)] *= 0.01  # smaller than what its page holds: the scale stays
    dev = [t.cuda() for t in x]
    pool.append(dev[0], dev[1], _i32(slots))
    assert pool.status() == 0
    for codes, scale, (b0, s0), old, rows in ((pool.k, pool.k_scale, before[0], vals[0], x[0]),
                                              (pool.v, pool.v_scale, before[1], vals[1], x[1])):
        got = codes.float().cpu().double().numpy()
        after = scale.cpu().numpy()
        ref = _append_reference(codes, s0, rows.float().numpy(), slots)
        b1 = _codes_bits(codes)
        for p in range(pages):
            if p not in ref:
                assert (b1[p] == b0[p]).all() and (after[p] == s0[p]).all(), p
                continue
            first, m, s1, s_old, v = ref[p]
            assert (after[p] == s1).all(), p
            exact = v.transpose(1, 0, 2) / s1.astype(np.float64)[:, None, None]
            assert _near(got[p, :, first:first + m], exact, codes.dtype).all(), p
            exact = old[p, :, :first] * (s_old.astype(np.float64) / s1)[:, None, None]
            stays = s1 == s_old  # such a head's codes are left as they are, e4m3's NaN (0xff here) among them
            assert _near(got[p, ~stays, :first], exact[~stays], codes.dtype).all(), p
            assert (b1[p][stays, :first] == b0[p][stays, :first]).all(), p
            assert (b1[p][:, first + m:] == b0[p][:, first + m:]).all(), p


@pytest.mark.parametrize("name", ["int8", "e4m3"])
def test_append_many_rows(name):
    """Enough rows that a wave looks through sixteen slots at a time."""
    from kvrt import Block8Pool

    gen = torch.Generator().manual_seed(3)
    heads, dim, block, pages = 8, 128, 16, 200
    pool = Block8Pool.zeros(pages, heads, dim, block_size=block, dtype=name)
    order = torch.randperm(pages, generator=gen).tolist()
    slots, at = [], 0
    for length, keep in ((333, 5), (1, 0), (700, 16), (40, 39), (1, 15), (517, 0)):
        pos = range(keep, length + keep)
        slots += [order[at + q // block] * block + q % block for q in pos]
        at += -(-(length + keep) // block)
        slots += [-1] * (length % 3)
    x = [randn_bf16(gen, (len(slots), heads, dim)) for _ in range(2)]
    pool.append(x[0].cuda(), x[1].cuda(), _i32(slots))
    for codes, scale, rows in ((pool.k, pool.k_scale, x[0]), (pool.v, pool.v_scale, x[1])):
        got, after = codes.float().cpu().double().numpy(), scale.cpu().numpy()
        ref = _append_reference(codes, np.zeros((pages, heads), np.float32), rows.float().numpy(), slots)
        for p, (first, m, s1, _, v) in ref.items():
            assert (after[p] == s1).all()
            exact = v.transpose(1, 0, 2) / s1.astype(np.float64)[:, None, None]
            assert _near(got[p, :, first:first + m], exact, codes.dtype).all(), p
            assert (got[p, :, :first] == 0).all() and (got[p, :, first + m:] == 0).all()
        unused = [p for p in range(pages) if p not in ref]
        assert (after[unused] == 0).all()


@pytest.mark.parametrize("name", ["int8", "e4m3"])
def test_append_of_extreme_values(name):
    """All zeros, the smallest and largest bf16, infinities and NaN."""
    from kvrt import Block8Pool

    pool = Block8Pool.zeros(6, 1, 64, dtype=name)
    top = R.TOP[NAMES[name]]
    x = torch.zeros((6, 1, 64), dtype=torch.bfloat16)
    x[1] = 2.0 ** -130
    x[2] = torch.finfo(torch.bfloat16).max
    x[3, 0, :4] = torch.tensor([1.0, -2.0, 0.5, float("inf")])
    x[4, 0, :4] = torch.tensor([float("nan"), 4.0, -float("inf"), 1.0])
    x[5] = float("nan")
    pool.append(x.cuda(), x.cuda(), _i32([16 * i for i in range(6)]))
    assert pool.status() == R.NOT_FINITE and pool.status() == 0
    s, c = pool.k_scale.cpu().numpy()[:, 0], pool.k.float().cpu().numpy()[:, 0, 0]
    assert s[0] == s[1] == s[5] == 2.0 ** -64 and s[2] == 2.0 ** 32
    assert s[3] == np.float32(2.0) / np.float32(top) and s[4] == np.float32(4.0) / np.float32(top)
    assert (c[0] == 0).all() and (c[1] == 0).all() and (c[2] == top).all() and (c[5] == 0).all()
    assert c[3, 1] == -top and c[3, 3] == top and c[4, 0] == 0 and c[4, 1] == top and c[4, 2] == -top
    assert (pool.v_scale == pool.k_scale).all() and (_codes_bits(pool.v) == _codes_bits(pool.k)).all()


def test_append_takes_strided_rows_and_skips_slots_outside_the_pool():
    from kvrt import Block8Pool

    gen = torch.Generator().manual_seed(9)
    heads, dim, rows = 4, 128, 11
    base = randn_bf16(gen, (2, heads, 40, dim)).cuda()  # HF layout [n, H, S, D]
    k, v = base[0, :, 3:3 + rows].transpose(0, 1), base[1, :, 20:20 + rows].transpose(0, 1)
    slots = _i32([*range(18, 18 + rows)])
    a, b = (Block8Pool.zeros(4, heads, dim) for _ in range(2))
    a.append(k, v, slots)
    b.append(k.contiguous(), v.contiguous(), slots)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(a.k_scale, b.k_scale)
    assert a.status() == 0
    want = a.k.clone()
    a.append(k[:3], v[:3], _i32([64, 2 ** 31 - 1, 1 << 20]))  # 4 pages of 16 rows
    assert a.status() == R.BAD and torch.equal(a.k, want)
    a.append(k[:0], v[:0], _i32([]))
    assert a.status() == 0 and torch.equal(a.k, want)


# ---- gather -------------------------------------------------------------------------------------


def _filled(gen, pages, heads, dim, block, name, poison=()):
    """A pool of random codes; pages in `poison` hold NaN scales and, in e4m3, NaN codes."""
    from kvrt import Block8Pool

    pool = Block8Pool.zeros(pages, heads, dim, block_size=block, dtype=name)
    for codes, scale, size in ((pool.k, pool.k_scale, 0.02), (pool.v, pool.v_scale, 0.01)):
        if name == "int8":
            raw = torch.randint(-127, 128, codes.shape, generator=gen, dtype=torch.int8)
        else:
            raw = (torch.randn(codes.shape, generator=gen) * 100).clamp(-448, 448).to(F8).view(I8)
        codes.view(I8).copy_(raw)
        scale.copy_(size * (0.5 + torch.rand(scale.shape, generator=gen)))
        for p in poison:
            codes.view(I8)[p] = 0x7F
            scale[p] = float("nan")
    return pool


def _tables(gen, lengths, width, block, pages):
    """A table of distinct pages per request, -1 past the mapped ones."""
    order = torch.randperm(pages, generator=gen).tolist()
    table, at = torch.full((len(lengths), width), -1, dtype=torch.int32), 0
    for i, length in enumerate(lengths):
        m = -(-length // block)
        table[i, :m] = torch.tensor(order[at:at + m], dtype=torch.int32)
        at += m
    return table, order[at:]


@pytest.mark.parametrize("name", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,dim,block,lengths", [
    (2, 64, 16, [0, 1, 15, 16, 17, 70]), (1, 256, 32, [33, 5]), (1, 512, 16, [40]), (8, 128, 64, [100, 0, 64, 65]),
])
def test_gather_is_the_padded_batch(name, heads, dim, block, lengths):
    gen = torch.Generator().manual_seed(dim + block)
    pages = sum(-(-x // block) for x in lengths) + 3
    pool = _filled(gen, pages, heads, dim, block, name)
    table, _ = _tables(gen, lengths, max(-(-x // block) for x in lengths), block, pages)
    dev, lens = table.cuda(), _i32(lengths)
    for start in (None, [min(7 * i, x) for i, x in enumerate(lengths)]):
        for dtype in (torch.bfloat16, torch.float32):
            lmax = max(lengths) + 5
            k, v, mask = pool.gather(dev, lens, lmax, start_pos=None if start is None else _i32(start), dtype=dtype)
            assert mask.dtype == torch.bool and pool.status() == 0
            for got, codes, scale in ((k, pool.k, pool.k_scale), (v, pool.v, pool.v_scale)):
                x = codes.float() * scale[:, :, None, None]
                for i, length in enumerate(lengths):
                    lo = 0 if start is None else start[i]
                    rows = x[dev[i, :-(-length // block)].long()].transpose(0, 1).reshape(heads, -1, dim)[:, lo:length]
                    assert torch.equal(got[i, :, :length - lo], rows.to(dtype)), (i, dtype)
                    assert (got[i, :, length - lo:] == 0).all()
                    assert mask[i].tolist() == [j < length - lo for j in range(lmax)]


def test_gather_into_strided_destinations_and_masks():
    gen = torch.Generator().manual_seed(2)
    pool = _filled(gen, 8, 2, 128, 16, "e4m3")
    table, _ = _tables(gen, [37, 20], 3, 16, 8)
    dev, lens = table.cuda(), _i32([37, 20])
    k, v, mask = pool.gather(dev, lens, 40)
    big = torch.full((2, 2, 2, 64, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    for dtype, lowest in ((torch.float32, torch.finfo(torch.float32).min), (torch.bfloat16, torch.finfo(torch.bfloat16).min)):
        m = torch.ones((2, 50), dtype=dtype, device="cuda")
        out = pool.gather(dev, lens, out=(big[0, :, :, 4:44], big[1, :, :, 4:44], m[:, :40]))
        assert torch.equal(out[0], k) and torch.equal(out[1], v)
        assert (big[:, :, :, :4] == 7).all() and (big[:, :, :, 44:] == 7).all() and (m[:, 40:] == 1).all()
        assert torch.equal(m[:, :40] == 0, mask) and (m[:, :40][~mask] == lowest).all()
    assert pool.gather(dev, lens, 40, mask_dtype=None)[2] is None
    bad = dev.clone()
    bad[0, 1], bad[1, 0] = 8, -1
    k2, _, mask2 = pool.gather(bad, lens, 40)
    assert pool.status() == R.BAD and torch.equal(mask2, mask)
    assert (k2[0, :, 16:32] == 0).all() and (k2[1, :, :16] == 0).all()
    assert torch.equal(k2[0, :, :16], k[0, :, :16]) and torch.equal(k2[1, :, 16:], k[1, :, 16:])
    pool.gather(dev, _i32([49, 20]), 40)  # three pages hold 48 rows
    assert pool.status() == R.BAD


# ---- attention --------------------------------------------------------------------------------


def _check(pool, q, table, lengths, counts, out, scale, window, sample=None):
    """Rows of out against float64; `sample` limits the rows of a request looked at."""
    block = pool.block_size
    kv = [R.dequant(pool.k, pool.k_scale), R.dequant(pool.v, pool.v_scale)]
    x, got = q.cpu().double().numpy(), out.cpu().double().numpy()
    at = 0
    for i, (length, m) in enumerate(zip(lengths, counts)):
        k, v = (R.rows_of(a, table[i].tolist(), length, block) for a in kv)
        rows = range(m) if sample is None or m <= sample else sorted({0, 1, m // 2, m - 2, m - 1, *range(3, m, m // sample + 1)})
        for r in rows:
            n = length - m + 1 + r
            want, tol = R.attend(x[at + r][None], k[:, :max(n, 0)], v[:, :max(n, 0)], n, scale, window)
            err = np.abs(got[at + r] - want[0])
            assert (err <= tol[0]).all(), (i, r, float((err / tol[0]).max()))
        at += m


def _starts(counts):
    return _i32(np.concatenate([[0], np.cumsum(counts)]).tolist())


def _attend_case(name, hq, heads, dim, block, lengths, counts, window=0, scale=None, seed=0, poison=True, sample=None):
    gen = torch.Generator().manual_seed(seed + dim + block + hq)
    pages = sum(-(-x // block) for x in lengths) + 4
    table, spare = _tables(gen, lengths, max(1, max(-(-x // block) for x in lengths)) + 1, block, pages)
    pool = _filled(gen, pages, heads, dim, block, name, poison=spare if poison else ())
    if poison:  # rows behind a request's last one hold anything, NaN codes among it
        for i, length in enumerate(lengths):
            if length % block:
                p = int(table[i, length // block])
                pool.k.view(I8)[p, :, length % block:] = 0x7F
                pool.v.view(I8)[p, :, length % block:] = 0x7F
    q = randn_bf16(gen, (sum(counts), hq, dim)).cuda()
    scale = dim ** -0.5 if scale is None else scale
    out = pool.attend(q, table.cuda(), _i32(lengths), _starts(counts), scale, max_q=max(counts), window=window)
    assert pool.status() == 0
    _check(pool, q, table, lengths, counts, out, scale, window, sample)
    return pool, q, table, out


@pytest.mark.parametrize("name", ["int8", "e4m3"])
@pytest.mark.parametrize("hq,heads,dim,block", [
    (4, 2, 64, 16), (16, 8, 128, 16), (8, 1, 256, 32), (8, 1, 512, 16), (3, 1, 128, 64), (16, 1, 128, 128), (5, 5, 64, 32),
])
def test_decode_of_ragged_requests(name, hq, heads, dim, block):
    """One row each; lengths around the edges of tiles, units and pages."""
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300, 1000]
    _attend_case(name, hq, heads, dim, block, lengths, [1] * len(lengths))


@pytest.mark.parametrize("window", [1, 16, 100, 512])
@pytest.mark.parametrize("name,hq,heads,dim,counts", [
    ("int8", 8, 1, 256, [2, 1, 2, 1]), ("e4m3", 8, 4, 128, [1, 8, 3, 1]), ("int8", 4, 1, 128, [40, 7, 100, 1]),
    ("e4m3", 8, 1, 512, [30, 1, 5, 64]),
])
def test_windows(name, hq, heads, dim, counts, window):
    _attend_case(name, hq, heads, dim, 16, [600, 9, 101, 130], counts, window=window)


def test_pages_below_the_window_may_be_unmapped():
    pool, q, table, out = _attend_case("int8", 8, 1, 256, 16, [600, 333], [2, 1], window=100)
    table[0, :(600 - 2 - 100 + 1) // 16] = -1
    table[1, :(333 - 1 - 100 + 1) // 16] = 99999
    got = pool.attend(q, table.cuda(), _i32([600, 333]), _starts([2, 1]), 256 ** -0.5, max_q=2, window=100)
    assert pool.status() == 0 and torch.equal(got, out)


@pytest.mark.parametrize("name", ["int8", "e4m3"])
@pytest.mark.parametrize("hq,heads,dim,block,lengths,counts", [
    (8, 8, 128, 16, [34], [34]), (16, 8, 128, 16, [200, 77, 31], [150, 77, 3]), (8, 1, 256, 32, [333], [129]),
    (8, 1, 512, 16, [150, 33], [70, 33]), (12, 4, 128, 64, [100, 1, 257], [65, 1, 200]), (6, 2, 64, 16, [90, 64], [33, 64]),
    (7, 1, 64, 128, [260], [140]),
])
def test_chunks(name, hq, heads, dim, block, lengths, counts):
    _attend_case(name, hq, heads, dim, block, lengths, counts, sample=12)


def test_a_row_without_keys_is_zero_and_rows_of_no_request_stay():
    """Lengths of 0, more rows than keys, requests without rows, rows behind the last
    and those of requests that were granted none."""
    gen = torch.Generator().manual_seed(4)
    pool = _filled(gen, 10, 2, 128, 16, "e4m3")
    for hq, width in ((4, 1), (16, 1), (40, 3)):
        lengths, counts, granted = [0, 2, 20, 0, 16, 5], [1, 5, 2, 0, 3, 2], [1, 5, 2, 0, 0, 2]
        table, _ = _tables(gen, lengths, 2, 16, 10)
        q = randn_bf16(gen, (20, hq, 128)).cuda()
        out = torch.full_like(q, 3.0)
        pool.attend(q, table.cuda(), _i32(lengths), _starts(counts), 0.1, max_q=5, granted=_i32(granted), out=out)
        assert pool.status() == 0
        assert (out[0] == 0).all() and (out[1:4] == 0).all()  # no key; rows before the first position
        assert (out[8:11] == 3).all() and (out[13:] == 3).all()
        for lo, m, i in ((4, 2, 1), (6, 2, 2), (11, 2, 5)):
            _check(pool, q[lo:lo + m], table[i:i + 1], [lengths[i]], [m], out[lo:lo + m], 0.1, 0)


def test_bad_numbers_on_the_device_are_reported_and_skipped():
    gen = torch.Generator().manual_seed(6)
    pool = _filled(gen, 10, 1, 64, 16, "int8")
    lengths, counts = [40, 33, 64], [1, 2, 1]
    table, _ = _tables(gen, lengths, 4, 16, 10)
    q = randn_bf16(gen, (4, 2, 64)).cuda()
    good = pool.attend(q, table.cuda(), _i32(lengths), _starts(counts), 0.1, max_q=2)
    assert pool.status() == 0
    for lens, starts, granted, rows in (([40, 33, 65], [0, 1, 3, 4], None, [0, 1, 2]), ([-1, 33, 64], [0, 1, 3, 4], None, [1, 2, 3]),
                                        (lengths, [0, 1, 3, 5], None, [0, 1, 2, 3]), (lengths, [0, 1, 3, 4], [-2, 2, 1], [1, 2, 3]),
                                        (lengths, [0, 1, 3, 2], None, [0, 1, 2])):
        out = torch.full_like(q, 5.0)
        pool.attend(q, table.cuda(), _i32(lens), _i32(starts), 0.1, max_q=2,
                    granted=None if granted is None else _i32(granted), out=out)
        assert pool.status() == R.BAD
        assert torch.equal(out[rows], good[rows]), (lens, starts)
    bad = table.clone()
    bad[1, 1] = -1  # rows 16 .. 31 of request 1 are unmapped: unseen
    out = pool.attend(q, bad.cuda(), _i32(lengths), _starts(counts), 0.1, max_q=2)
    assert pool.status() == R.BAD
    assert torch.equal(out[[0, 3]], good[[0, 3]]) and torch.isfinite(out.float()).all()


def test_more_rows_than_max_q_are_reported_and_left():
    gen = torch.Generator().manual_seed(16)
    pool = _filled(gen, 9, 1, 64, 16, "int8")
    table, _ = _tables(gen, [40, 33], 3, 16, 9)
    q = randn_bf16(gen, (5, 1, 64)).cuda()
    out = torch.full_like(q, 5.0)
    pool.attend(q, table.cuda(), _i32([40, 33]), _starts([1, 4]), 0.1, max_q=3, out=out)
    assert pool.status() == R.BAD and (out[4] == 5).all() and not (out[:4] == 5).all(-1).any()


@pytest.mark.parametrize("name", ["int8", "e4m3"])
@pytest.mark.parametrize("count", [1, 24])
def test_extreme_scales(name, count):
    """V pages of zeros, V scales 2^90 apart, negative and zero softmax scales, query
    rows from 2^-100 to 2^100, and keys masked by their scores."""
    gen = torch.Generator().manual_seed(21)
    dim, block, length = 128, 16, 200
    for scale in (0.08, -0.08, 0.0):
        pool = _filled(gen, 14, 2, dim, block, name)
        table, _ = _tables(gen, [length], 13, block, 14)
        for j, e in enumerate((0, -64, 30, -30, 0, 10)):
            pool.v_scale[int(table[0, j])] = 2.0 ** e
        pool.v.view(I8)[int(table[0, 1])] = 0
        pool.v_scale[int(table[0, 6])] = 0.0  # read as 2^-64
        q = randn_bf16(gen, (count, 4, dim)).cuda()
        q[:, 1] *= 2.0 ** -100
        if scale == 0.0:
            q[:, 2] *= 2.0 ** 100
        out = pool.attend(q, table.cuda(), _i32([length]), _starts([count]), scale, max_q=count)
        assert pool.status() == 0
        # V scales differ by more than 4: only rows' own largest terms are resolved
        kv = [R.dequant(pool.k, pool.k_scale), R.dequant(pool.v, pool.v_scale)]
        k, v = (R.rows_of(a, table[0].tolist(), length, block) for a in kv)
        x, got = q.cpu().double().numpy(), out.cpu().double().numpy()
        want, tol = R.attend(x, k, v, length, scale, 0)
        assert (np.abs(got - want) <= tol).all()


def test_query_rows_that_are_not_finite_stay_their_own():
    pool, q, table, out = _attend_case("int8", 16, 2, 128, 16, [300, 90], [1, 1])
    for value in (float("nan"), float("inf")):
        x = q.clone()
        x[0, 3, 5] = value
        got = pool.attend(x, table.cuda(), _i32([300, 90]), _starts([1, 1]), 128 ** -0.5, max_q=1)
        assert got[0, 3].isnan().all()
        got[0, 3] = out[0, 3]
        assert torch.equal(got, out)


def test_strided_queries_and_outputs():
    pool, q, table, out = _attend_case("e4m3", 8, 4, 128, 16, [50, 33], [2, 2])
    wide = torch.zeros((4, 20, 128), dtype=torch.bfloat16, device="cuda")
    wide[:, 6:14] = q
    dst = torch.full((8, 4, 256), 2.0, dtype=torch.bfloat16, device="cuda")
    view = dst[:, :, 128:].transpose(0, 1)
    got = pool.attend(wide[:, 6:14], table.cuda(), _i32([50, 33]), _starts([2, 2]), 128 ** -0.5, max_q=2, out=view)
    assert got is view and torch.equal(view, out) and (dst[:, :, :128] == 2).all()
    wide_table = torch.full((2, 30), -1, dtype=torch.int32)
    wide_table[:, :table.shape[1]] = table
    part = wide_table.cuda()[:, :table.shape[1]]
    assert torch.equal(pool.attend(q, part, _i32([50, 33]), _starts([2, 2]), 128 ** -0.5, max_q=2), out)


@pytest.mark.parametrize("n", [257, 600])
def test_many_requests(n):
    """More requests than threads that divide the keys among them."""
    rng = np.random.default_rng(n)
    lengths = [int(x) for x in rng.integers(0, 60, n)]
    gen = torch.Generator().manual_seed(n)
    pages = sum(-(-x // 16) for x in lengths)
    pool = _filled(gen, pages, 1, 64, 16, "int8")
    table, _ = _tables(gen, lengths, 4, 16, pages)
    counts = [min(1, x) if i % 5 else 2 for i, x in enumerate(lengths)]
    q = randn_bf16(gen, (sum(counts), 2, 64)).cuda()
    out = pool.attend(q, table.cuda(), _i32(lengths), _starts(counts), 0.2, max_q=2)
    assert pool.status() == 0
    _check(pool, q, table, lengths, counts, out, 0.2, 0)


def test_pages_past_two_gib():
    """A pool whose codes pass 2^31 bytes and 2^32: the far pages are addressed."""
    from kvrt import Block8Pool

    heads, dim, block = 8, 512, 16
    pages = (1 << 32) // (heads * dim * block) + 40  # 4.2 GiB of K, as much of V
    pool = Block8Pool.zeros(pages, heads, dim, block_size=block)
    gen = torch.Generator().manual_seed(1)
    ids = [pages - 1, (1 << 31) // (heads * dim * block) + 1, 3, pages - 9]
    table = torch.tensor([ids], dtype=torch.int32)
    length = 59
    x = [randn_bf16(gen, (length, heads, dim)).cuda() for _ in range(2)]
    pool.append(x[0], x[1], _i32([ids[p // 16] * 16 + p % 16 for p in range(length)]))
    k, _, _ = pool.gather(table.cuda(), _i32([length]), length, dtype=torch.float32)
    assert (k[0] - x[0].float().transpose(0, 1)).abs().max() < 0.05
    q = randn_bf16(gen, (2, heads, dim)).cuda()
    out = pool.attend(q, table.cuda(), _i32([length]), _starts([2]), dim ** -0.5, max_q=2)
    small = Block8Pool(*(t[ids].contiguous() for t in (pool.k, pool.v, pool.k_scale, pool.v_scale)))
    near = small.attend(q, _i32([[0, 1, 2, 3]]), _i32([length]), _starts([2]), dim ** -0.5, max_q=2)
    assert pool.status() == 0 and torch.equal(out, near)


# ---- together -------------------------------------------------------------------------------------


@pytest.mark.parametrize("name,hq,heads,dim", [("int8", 16, 8, 128), ("e4m3", 8, 1, 256)])
def test_a_serving_run(name, hq, heads, dim):
    """Prefill, decode steps, rollback, a finished and a new request, as one program
    runs them; each step's attention and batch against 64 bits over the pool's own
    codes, and those near the rows that were appended."""
    from kvrt import Block8Pool, BlockTables

    gen = torch.Generator().manual_seed(8)
    n, block, pages = 4, 16, 80
    tables = BlockTables(n, 20, pages, block_size=block)
    pool = Block8Pool.zeros(pages, heads, dim, block_size=block, dtype=name)
    rows = [np.zeros((0, heads, dim)) for _ in range(n)]
    steps = [([0] * n, [40, 7, 100, 0])] + [(None, [1, 1, 1, 0])] * 3
    steps += [([38, 9, 90, 0], [1, 2, 30, 60]), (None, [1, 1, 1, 1]), ([0, 5, 100, 50], [0, 3, 1, 9]), (None, [21, 1, 1, 1])]
    lens = [0] * n
    for step, (keep, new) in enumerate(steps):
        keep = lens if keep is None else [min(a, b) for a, b in zip(keep, lens)]
        total = sum(new)
        plan = tables.update(_i32(keep), _i32(new), rows=total + 3)
        lens = [a + b for a, b in zip(keep, new)]
        assert plan.lengths.tolist() == lens and plan.granted.tolist() == new
        k, v = (randn_bf16(gen, (total + 3, heads, dim), s).cuda() for s in (1.0, 0.5 + step))
        pool.append(k, v, plan.slot_map)
        q = randn_bf16(gen, (total + 3, hq, dim)).cuda()
        out = torch.full_like(q, 9.0)
        pool.attend(q, tables.table, plan.lengths, plan.starts, dim ** -0.5, max_q=max(new), granted=plan.granted, out=out)
        assert (out[total:] == 9).all()
        table = tables.table.cpu()
        _check(pool, q, table, lens, new, out[:total], dim ** -0.5, 0)
        bk, _, mask = pool.gather(tables.table, plan.lengths, max(lens), dtype=torch.float32)
        at = 0
        for i in range(n):
            rows[i] = np.concatenate([rows[i][:keep[i]], k[at:at + new[i]].double().cpu().numpy()])
            at += new[i]
            got = bk[i, :, :lens[i]].double().cpu().numpy().transpose(1, 0, 2)
            # a page's largest value over 2 * 127, or 2^-4 of the value; a row is coded
            # again each time its page's scale grows, at most 16 times
            big = np.abs(rows[i]).max(initial=0.0)
            assert (np.abs(got - rows[i]) <= 16 * (big / 250 if name == "int8" else np.abs(rows[i]) / 16 + big / 2 ** 16)).all()
            assert mask[i].sum().item() == lens[i]
    assert pool.status() == 0 and tables.status() == 0


@pytest.mark.parametrize("name", ["int8", "e4m3"])
def test_a_captured_step_replays_as_eager_calls_run(name):
    """tables, append and attend in one graph, replayed over page boundaries; the same
    steps eagerly give the same bits."""
    from kvrt import Block8Pool, BlockTables

    gen = torch.Generator().manual_seed(12)
    n, heads, hq, dim = 3, 2, 4, 128

    def make():
        return BlockTables(n, 8, 24), Block8Pool.zeros(24, heads, dim, dtype=name), _i32([0] * n)

    first = [randn_bf16(gen, (60, heads, dim)).cuda() for _ in range(2)]
    k, v = (torch.zeros((n, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros((n, hq, dim), dtype=torch.bfloat16, device="cuda")
    new, scale = _i32([1] * n), dim ** -0.5

    def start(tables, pool, lengths):
        plan = tables.update(lengths, _i32([30, 14, 16]), rows=60)
        pool.append(*first, plan.slot_map)
        lengths.copy_(plan.lengths)

    def step(tables, pool, lengths):
        plan = tables.update(lengths, new, rows=n)
        pool.append(k, v, plan.slot_map)
        out = pool.attend(q, tables.table, plan.lengths, plan.starts, scale, max_q=1, granted=plan.granted)
        lengths.copy_(plan.lengths)
        return out

    eager, graphed = make(), make()
    start(*eager), start(*graphed)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(*graphed)
    for _ in range(25):
        for t in (k, v, q):
            t.copy_(randn_bf16(gen, t.shape))
        want = step(*eager)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        for a, b in zip((eager[0].table, eager[1].k.view(I8), eager[1].v_scale, eager[2]),
                        (graphed[0].table, graphed[1].k.view(I8), graphed[1].v_scale, graphed[2])):
            assert torch.equal(a, b)
    assert graphed[0].status() == 0 and graphed[1].status() == 0


def test_calls_on_two_streams_and_two_graphs_keep_apart():
    """attend only reads a pool: calls that overlap, and graphs replayed side by side,
    give what they give alone."""
    pool, q, table, out = _attend_case("int8", 16, 8, 128, 16, [2000, 1500, 700], [1, 1, 1], sample=1)
    dev, lens, starts = table.cuda(), _i32([2000, 1500, 700]), _starts([1, 1, 1])
    q2 = (q.float() * 0.5).to(torch.bfloat16)
    torch.cuda.synchronize()
    call = lambda x: pool.attend(x, dev, lens, starts, 128 ** -0.5, max_q=1)  # noqa: E731
    alone = call(q2)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call((q, q2)[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, out) for x in got[0]) and all(torch.equal(x, alone) for x in got[1])
    graphs, outs = [], []
    for x in (q, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(x))
        graphs.append(g)
    for _ in range(5):
        for t in outs:
            t.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], out) and torch.equal(outs[1], alone)


def test_results_do_not_change_between_calls():
    """No order of workgroups shows in a result."""
    pool, q, table, out = _attend_case("e4m3", 8, 1, 256, 16, [900, 3000], [2, 1], sample=1)
    for _ in range(20):
        got = pool.attend(q, table.cuda(), _i32([900, 3000]), _starts([2, 1]), 256 ** -0.5, max_q=2)
        assert (bits(got) == bits(out)).all()


@pytest.mark.parametrize("name", ["int8", "e4m3"])
@pytest.mark.parametrize("block,dim", [(64, 256), (128, 128), (128, 512)])
def test_append_long_runs(name, block, dim):
    """Runs longer than the slots a wave looks at together, from the middle of pages
    too, in a call whose waves take sixteen slots each."""
    from kvrt import Block8Pool

    gen = torch.Generator().manual_seed(block + dim)
    heads, pages = 8, 12
    pool = Block8Pool.zeros(pages, heads, dim, block_size=block, dtype=name)
    slots = [5] + list(range(3 * block + 2, 4 * block)) + [-1] + list(range(6 * block, 9 * block - 1)) + [11 * block]
    slots += [-1] * (300 - len(slots))
    x = [randn_bf16(gen, (len(slots), heads, dim)) for _ in range(2)]
    pool.append(x[0].cuda(), x[1].cuda(), _i32(slots))
    for codes, scale, rows in ((pool.k, pool.k_scale, x[0]), (pool.v, pool.v_scale, x[1])):
        got, after = codes.float().cpu().double().numpy(), scale.cpu().numpy()
        ref = _append_reference(codes, np.zeros((pages, heads), np.float32), rows.float().numpy(), slots)
        for p in range(pages):
            if p not in ref:
                assert (after[p] == 0).all() and (got[p] == 0).all(), p
                continue
            first, m, s1, _, v = ref[p]
            assert (after[p] == s1).all(), p
            exact = v.transpose(1, 0, 2) / s1.astype(np.float64)[:, None, None]
            assert _near(got[p, :, first:first + m], exact, codes.dtype).all(), p
            assert (got[p, :, :first] == 0).all() and (got[p, :, first + m:] == 0).all(), p


@pytest.mark.parametrize("n,block", [(3, 16), (20, 16), (70, 32)])
def test_tables_release_many_pages(n, block):
    """A few pages and hundreds of them go back in one call, and are handed out again
    in the same one."""
    from kvrt import BlockTables

    rng = np.random.default_rng(n)
    width = 700
    t, ref = BlockTables(n, width, n * width, block_size=block), R.Tables(n, width, n * width, block)
    full = [int(rng.integers(1, width * block + 1)) if i % 4 else 3 * block for i in range(n)]
    want = ref.update([0] * n, full, 0)
    plan = t.update(_i32([0] * n), _i32(full), rows=0)  # no row fits: every request is refused
    assert plan.granted.tolist() == want[3] and t.status() != 0
    want = ref.update([0] * n, full, sum(full))
    _compare_tables(t, ref, t.update(_i32([0] * n), _i32(full), rows=sum(full)), want, "grown")
    keep = [x if i % 3 == 0 else x // 2 if i % 3 == 1 else 0 for i, x in enumerate(full)]
    new = [0 if i % 2 else min(5 * block, width * block - keep[i]) for i in range(n)]
    want = ref.update(keep, new, sum(new))
    _compare_tables(t, ref, t.update(_i32(keep), _i32(new), rows=sum(new)), want, "cut")
    want = ref.update([0] * n, [1] * n, n)
    _compare_tables(t, ref, t.update(_i32([0] * n), _i32([1] * n), rows=n), want, "emptied")


@pytest.mark.parametrize("name,dim,n", [("int8", 64, 70), ("e4m3", 128, 65), ("int8", 256, 70), ("e4m3", 512, 66)])
def test_chunks_of_many_requests(name, dim, n):
    """More requests than a wave has lanes, some of them without rows."""
    rng = np.random.default_rng(n + dim)
    counts = [int(x) for x in rng.integers(0, 40, n)]
    counts[3] = 0
    lengths = [c + int(x) for c, x in zip(counts, rng.integers(0, 50, n))]
    _attend_case(name, 2, 1, dim, 16, lengths, counts, sample=3)


@pytest.mark.parametrize("name,hq,heads,dim,lengths,counts,window", [
    ("int8", 8, 1, 256, [3000], [40], 0), ("e4m3", 16, 2, 512, [2100], [33], 0), ("int8", 16, 8, 128, [2500, 90], [20, 34], 0),
    ("e4m3", 8, 1, 256, [2900, 1400], [40, 300], 1000), ("int8", 2, 1, 64, [4000], [65], 0), ("int8", 8, 1, 512, [2000], [40], 700),
])
def test_chunks_over_long_contexts(name, hq, heads, dim, lengths, counts, window):
    """Keys divided over workgroups, many steps of each, joined by a second launch; and
    the same call on another stream."""
    pool, q, table, out = _attend_case(name, hq, heads, dim, 16, lengths, counts, window=window, sample=4)
    lens, starts, dev = _i32(lengths), _starts(counts), table.cuda()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        again = pool.attend(q, dev, lens, starts, dim ** -0.5, max_q=max(counts), window=window)
    s.synchronize()
    assert torch.equal(again, out)


@pytest.mark.parametrize("hq,heads,dim,count", [(2, 1, 128, 3), (8, 1, 256, 40), (4, 2, 64, 90)])
def test_a_window_past_the_table_is_none(hq, heads, dim, count):
    """More rows than keys, and the largest window a call can name."""
    pool, q, table, out = _attend_case("int8", hq, heads, dim, 16, [2, count + 9], [3, count])
    for window in (2 ** 31 - 1, 2 ** 30, 10 ** 6):
        got = pool.attend(q, table.cuda(), _i32([2, count + 9]), _starts([3, count]), dim ** -0.5, max_q=count, window=window)
        assert torch.equal(got, out), window
    assert pool.status() == 0
