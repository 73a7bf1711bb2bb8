"""Decode attention where a head's keys lie over several workgroups, against float64:
divisions that let the launch join every head, joins of more partials than are read
in one order, and more requests than a wave has lanes among all of them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_gpu_block8 import _attend_case, _i32, _starts

pytestmark = pytest.mark.gpu


def _again(pool, q, table, out, lengths, counts):
    """The same bits from another call, and from one on another stream."""
    args = (q, table.cuda(), _i32(lengths), _starts(counts), pool.head_dim ** -0.5)
    assert torch.equal(pool.attend(*args, max_q=max(counts)), out)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = pool.attend(*args, max_q=max(counts))
    side.synchronize()
    assert torch.equal(got, out) and pool.status() == 0


@pytest.mark.parametrize("name", ["int8", "e4m3"])
@pytest.mark.parametrize("few,short,n", [([8100], 100, 64), ([8000, 4100, 2000], 40, 65), ([4300, 4100], 100, 64),
                                         ([4250, 1], 130, 130)])
def test_few_long_requests_among_many_short_ones(name, few, short, n):
    """16 heads over 8, D 128: a head may have more units than a workgroup joins (32) beside
    512 heads and more, so the keys are divided such that the launch joins every head;
    with the longest requests a workgroup takes more units for that (three, not two)."""
    rng = np.random.default_rng(n)
    lengths = [int(x) for x in rng.integers(1, short, n)]
    for i, x in enumerate(few):
        lengths[(7 + 31 * i) % n] = x
    _again(*_attend_case(name, 16, 8, 128, 16, lengths, [1] * n), lengths, [1] * n)


@pytest.mark.parametrize("name,hq,heads,dim,lengths,counts", [
    ("e4m3", 8, 1, 512, [8192, 5000, 4100, 33], [2, 2, 2, 2]), ("int8", 16, 1, 512, [9000], [1]),
    ("int8", 16, 1, 256, [8000, 300], [1, 1]), ("e4m3", 16, 1, 128, [7000, 6000], [1, 1]), ("int8", 16, 1, 64, [8000], [1]),
    ("e4m3", 2, 1, 64, [5000, 6500], [8, 3]),
])
def test_joins_of_many_partials(name, hq, heads, dim, lengths, counts):
    """A unit a workgroup: 33 to 71 partials of a head, joined in interleaved orders (two at
    D 512, sixteen at D 64)."""
    _again(*_attend_case(name, hq, heads, dim, 16, lengths, counts), lengths, counts)


@pytest.mark.parametrize("name,hq,heads,dim,n,q,long", [
    ("int8", 16, 8, 128, 70, 1, 3500),   # joined in the launch
    ("e4m3", 4, 4, 64, 100, 1, 3000),    # the same
    ("int8", 16, 1, 256, 70, 1, 4000),   # three partials in the launch, more in a second one
    ("e4m3", 8, 1, 512, 66, 2, 3000),    # all in a second one
    ("int8", 16, 1, 512, 300, 1, 1500),  # the same, more requests than threads
    ("e4m3", 16, 2, 512, 300, 1, 1500),  # divided such that the launch joins every head
])
def test_joins_among_more_requests_than_lanes(name, hq, heads, dim, n, q, long):
    rng = np.random.default_rng(dim + n)
    lengths = [int(x) for x in rng.integers(1, 200, n)]
    counts = [min(q, x) for x in lengths]
    for i, length in ((0, long), (n // 2, long // 2), (n - 2, long - 13)):
        lengths[i], counts[i] = length, q
    lengths[5] = counts[5] = 0
    _again(*_attend_case(name, hq, heads, dim, 16, lengths, counts), lengths, counts)
