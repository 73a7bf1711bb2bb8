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
