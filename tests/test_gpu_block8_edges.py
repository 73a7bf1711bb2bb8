"""Calls at the edges of what 8-bit pages take: tables without columns."""
from __future__ import annotations

import pytest
import torch

from tests import block8_ref as R
from tests.helpers import randn_bf16

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("hq,heads,dim,counts", [(4, 2, 64, [1, 1, 1]), (16, 8, 128, [1, 2, 0]), (8, 1, 512, [2, 1, 1]),
                                                 (8, 2, 128, [40, 1, 90]), (8, 1, 256, [70, 0, 3]), (8, 1, 512, [33, 5, 0])])
def test_a_table_without_columns_gives_zero_rows(hq, heads, dim, counts):
    from kvrt import Block8Pool

    pool = Block8Pool.zeros(4, heads, dim)
    n, rows = len(counts), sum(counts)
    table = torch.empty((n, 0), dtype=torch.int32, device="cuda")
    starts = _i32([0, *torch.tensor(counts).cumsum(0).tolist()])
    q = randn_bf16(torch.Generator().manual_seed(1), (rows + 2, hq, dim)).cuda()
    out = torch.full_like(q, 3.0)
    got = pool.attend(q, table, _i32([0] * n), starts, 0.1, max_q=max(counts), out=out)
    assert got is out and pool.status() == 0
    assert (out[:rows] == 0).all() and (out[rows:] == 3).all()
    pool.attend(q, table, _i32([0, 5, 0]), starts, 0.1, max_q=max(counts), out=out)  # no column holds a key
    assert pool.status() == R.BAD and (out[:rows] == 0).all()
    k, v, mask = pool.gather(table, _i32([0] * n), 3)
    assert (k == 0).all() and (v == 0).all() and not mask.any()


@pytest.mark.parametrize("hq,count", [(2, 1), (4, 40)])
def test_windows_and_row_counts_past_32_bits(hq, count):
    """A window of any size past the keys is none; negative numbers are refused, also
    where their lowest 32 bits are not."""
    from kvrt import Block8Pool, KVRTError

    gen = torch.Generator().manual_seed(2)
    pool = Block8Pool.zeros(6, 2, 128)
    x = randn_bf16(gen, (80, 2, 128)).cuda()
    pool.append(x, x, _i32([*range(80)]))
    q, table = randn_bf16(gen, (count, hq, 128)).cuda(), _i32([[0, 1, 2, 3, 4]])
    call = lambda **kw: pool.attend(q, table, _i32([80]), _i32([0, count]), 0.1, **{"max_q": count, **kw})  # noqa: E731
    want, short = call(), call(window=5)
    assert not torch.equal(want, short)
    for window in (2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 40 + 7, 2 ** 64 + 5):
        assert torch.equal(call(window=window), want), window
    assert torch.equal(call(max_q=2 ** 32 + count - 1), want) and torch.equal(call(max_q=2 ** 64), want)
    for bad in (dict(window=-1), dict(window=-2 ** 32 + 5), dict(window=-2 ** 40), dict(max_q=-2 ** 32 + count),
                dict(max_q=-2 ** 31)):
        with pytest.raises(KVRTError):
            call(**bad)
    assert pool.status() == 0


@pytest.mark.parametrize("n", [64, 65, 700])
@pytest.mark.parametrize("count", [1, 40])
def test_bad_numbers_of_requests_without_rows_are_reported(n, count):
    """Behind the last request with rows too, however many requests there are."""
    from kvrt import Block8Pool

    pool = Block8Pool.zeros(4, 1, 64)
    x = randn_bf16(torch.Generator().manual_seed(3), (64, 1, 64)).cuda()
    pool.append(x, x, _i32([*range(64)]))
    table = torch.full((n, 4), -1, dtype=torch.int32)
    table[1] = torch.arange(4)
    lengths, starts = [0] * n, [0, 0] + [count] * (n - 1)
    lengths[1] = 64
    call = lambda lens: pool.attend(x[:count], table.cuda(), _i32(lens), _i32(starts), 0.1, max_q=count)  # noqa: E731
    want = call(lengths)
    assert pool.status() == 0
    for i in (0, 2, n - 2, n - 1):
        for bad in (65, -1):
            lens = list(lengths)
            lens[i] = bad
            assert torch.equal(call(lens), want)
            assert pool.status() == R.BAD, (i, bad)
