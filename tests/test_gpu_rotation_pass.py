"""Heads and dims that a rotation neither norms nor turns come out bit for bit, whatever they
and their neighbours hold."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
# infinities, NaN (one of them signalling), zeros of both signs, the smallest and largest numbers
ODD = [0x7F80, 0xFF80, 0x7FC0, 0xFFC1, 0x7F81, 0x8000, 0x0000, 0x0001, 0x8001, 0x7F7F, 0xFF7F]


def _bits(x):
    return x.view(torch.int16)


def _heads(gen, n, h, q, d, odd_dims):
    """Rows with odd values among the dims of odd_dims, at other places in each row."""
    x = torch.randn(n, h, q, d, generator=gen, device="cuda").to(BF16).view(torch.int16)
    values = torch.tensor([v - 65536 if v > 32767 else v for v in ODD], dtype=torch.int16, device="cuda")
    if len(odd_dims):
        dims = torch.tensor(list(odd_dims), device="cuda")
        at = torch.rand(x.shape[:-1] + (len(odd_dims),), generator=gen, device="cuda") < 0.3
        which = torch.randint(len(ODD), at.shape, generator=gen, device="cuda")
        x[..., dims] = torch.where(at, values[which], x[..., dims])
    return x.view(BF16)


# heads of a launch: one a group, four a group, and past a million lanes
@pytest.mark.parametrize("n,q", [(3, 5), (2, 800), (4, 8192)])
@pytest.mark.parametrize("d,freqs", [(64, 8), (64, 24), (128, 32), (256, 64), (512, 64), (128, 0), (128, 64)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_dims_past_the_pairs_and_value_heads(n, q, d, freqs, adjacent):
    from kvrt import HeadRotation

    if n * q > 10000 and d > 128:
        q //= d // 128
    gen = torch.Generator(device="cuda").manual_seed(d + freqs + n)
    inv = 1e4 ** (-torch.arange(freqs, dtype=torch.float64) / max(freqs, 1))
    rest = range(2 * freqs, d)
    x = [_heads(gen, n, h, q, d, dims) for h, dims in ((9, rest), (3, rest), (3, range(d)))]
    pos = torch.randint(0, 9000, (n, q), generator=gen, device="cuda")
    got = HeadRotation(d, inv, adjacent=adjacent, norm="none", scaling=1.25).apply(*x, positions=pos)
    for name, a, b in zip("qkv", x, got):
        part = slice(2 * freqs if name != "v" else 0, None)
        assert torch.equal(_bits(a[..., part]), _bits(b[..., part])), name
    # turned dims beside them are numbers
    for b in got[:2]:
        assert bool(b[..., :2 * freqs].isfinite().all())
    # values pass beside normed heads as well
    clean = [_heads(gen, n, 9, q, d, ()), _heads(gen, n, 3, q, d, ())]
    got = HeadRotation(d, inv, adjacent=adjacent, norm="qk").apply(*clean, x[2], positions=pos)
    assert torch.equal(_bits(got[2]), _bits(x[2]))
    assert bool(got[0].isfinite().all()) and bool(got[1].isfinite().all())
