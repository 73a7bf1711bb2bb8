"""A pool's tensors are its own attributes: the calls use those it holds when they are
made, by the native calls and by the general path alike."""
from __future__ import annotations

import pytest
import torch

from tests.helpers import randn_bf16

pytestmark = pytest.mark.gpu

I8 = torch.int8


class _General:
    """Stands in for the native module: every call takes the general path."""

    def __getattr__(self, name):
        return lambda *a: 1


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pool(dtype, general):
    from kvrt import Block8Pool

    pool = Block8Pool.zeros(6, 2, 64, dtype=dtype)
    if general:
        pool._call = _General()
    return pool


TABLE, LENGTHS, SLOTS = [[4, 1, 2]], [35], [*range(64, 80), *range(16, 35)]


def _use(pool, x, q):
    """Rows written, read back and attended over."""
    pool.append(x, x * 2, _i32(SLOTS))
    k, v, mask = pool.gather(_i32(TABLE), _i32(LENGTHS), 40)
    out = pool.attend(q, _i32(TABLE), _i32(LENGTHS), _i32([0, 2]), 0.125, max_q=2)
    chunk = pool.attend(x.repeat(1, 2, 1), _i32(TABLE), _i32(LENGTHS), _i32([0, 35]), 0.125, max_q=35)
    assert pool.status() == 0
    return k, v, mask, out, chunk


@pytest.mark.parametrize("general", [False, True])
@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_reassigned_tensors_are_the_ones_used(dtype, general):
    gen = torch.Generator().manual_seed(4)
    x, q = randn_bf16(gen, (35, 2, 64)).cuda(), randn_bf16(gen, (2, 4, 64)).cuda()
    want = _use(_pool(dtype, general), x, q)
    for names in (("k",), ("v",), ("k_scale", "v_scale"), ("k", "v", "k_scale", "v_scale")):
        pool = _pool(dtype, general)
        old = {name: getattr(pool, name) for name in names}  # kept alive
        for name, t in old.items():
            setattr(pool, name, torch.zeros_like(t))
        got = _use(pool, x, q)
        for a, b in zip(got, want):
            assert torch.equal(a, b), names
        for name, t in old.items():
            assert (t.view(torch.uint8) == 0).all() and not (getattr(pool, name).view(torch.uint8) == 0).all(), name


def test_storage_exchanged_under_a_tensor_is_the_one_used():
    gen = torch.Generator().manual_seed(5)
    x, q = randn_bf16(gen, (35, 2, 64)).cuda(), randn_bf16(gen, (2, 4, 64)).cuda()
    want = _use(_pool("int8", False), x, q)
    pool = _pool("int8", False)
    old = torch.zeros_like(pool.k)
    pool.k.data, old = old, pool.k.data
    for a, b in zip(_use(pool, x, q), want):
        assert torch.equal(a, b)
    assert (old == 0).all() and not (pool.k == 0).all()


@pytest.mark.parametrize("general", [False, True])
def test_reassigned_tensors_are_checked(general):
    x = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device="cuda")
    table, one, starts = _i32([[0, 1]]), _i32([1]), _i32([0, 1])
    bad = {"k": (torch.zeros((5, 2, 16, 64), dtype=I8), torch.zeros((6, 2, 16, 64)), torch.zeros((6, 2, 64, 16), dtype=I8),
                 torch.zeros((6, 16, 2, 64), dtype=I8).transpose(1, 2), torch.zeros((6, 2, 16, 64), dtype=torch.uint8),
                 torch.zeros((6, 2, 16, 64), dtype=torch.float8_e4m3fn)),
           "v_scale": (torch.zeros((6, 1)), torch.zeros(12), torch.zeros((6, 2), dtype=torch.float64),
                       torch.zeros((2, 6)).t())}
    for name, tensors in bad.items():
        for t in [*(t.cuda() for t in tensors), torch.zeros((6, 2, 16, 64), dtype=I8) if name == "k" else torch.zeros((6, 2))]:
            pool = _pool("int8", general)
            keep = getattr(pool, name)
            setattr(pool, name, t)
            for call in (lambda: pool.append(x, x, one), lambda: pool.gather(table, one, 3),
                         lambda: pool.attend(x, table, one, starts, 1.0, max_q=1)):
                with pytest.raises(ValueError, match=name):
                    call()
            setattr(pool, name, keep)
            pool.append(x, x, one)
            assert pool.status() == 0
