"""Every rotation kernel against the definition in 64 bits (tests/test_gpu_rotation.py derives the
tolerance): head_dim, order of pairs, one head of a group of lanes, four, four past a million
lanes, with and without dims that pass; and tables that end in zeros."""
from __future__ import annotations

import pytest
import torch

from test_gpu_rotation import _check, _freqs, _positions

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("lanes", [3000, 400_000, 1_300_000])  # up to 160 Ki: one head; past 1 Mi: around the L2
@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("norm", ["qkv", "none"])
def test_every_kernel(lanes, d, adjacent, norm):
    from kvrt import HeadRotation

    gen = torch.Generator(device="cuda").manual_seed(d + lanes)
    hq, hkv, n, freqs = 6, 1, 2, d // 4
    q = -(-lanes // (n * (hq + 2 * hkv) * (d // 16)))
    parts = torch.randn(n, q, hq + 2 * hkv, d, generator=gen, device="cuda").to(BF16).split([hq, hkv, hkv], 2)
    qw = None if norm == "none" else torch.rand(d, generator=gen, device="cuda") + 0.5
    which = [f % 2 for f in range(freqs)]
    rot = HeadRotation(d, _freqs(freqs), axes=which, adjacent=adjacent, norm=norm, q_weight=qw, scaling=0.75)
    pos = _positions(gen, 2, n, q, 100000)
    got = rot.apply(*(p.transpose(1, 2) for p in parts), positions=pos)
    for g, p, kind, w in zip(got, parts, "qkv", (qw, None, None)):
        _check(g, p.transpose(1, 2), kind, (_freqs(freqs), which, adjacent, norm, w, 1e-6, 0.75), pos)


@pytest.mark.parametrize("d,turn,zeros", [(512, 64, 192), (256, 32, 96), (64, 8, 8)])
@pytest.mark.parametrize("scaling", [1.0, 1.5])
def test_frequencies_that_end_in_zeros(d, turn, zeros, scaling):
    """Pairs (i, i + d / 2) of which the first `turn` turn: a full layer whose positions reach a
    part of its dims. A zero's pair is its scaling-fold."""
    from kvrt import HeadRotation

    gen = torch.Generator(device="cuda").manual_seed(d)
    x = torch.randn(2, 8, 40, d, generator=gen, device="cuda").to(BF16)
    freq = torch.cat((_freqs(turn), torch.zeros(zeros)))
    pos = _positions(gen, 1, 2, 40, 16384)
    for norm in ("qk", "none"):
        got = HeadRotation(d, freq, norm=norm, scaling=scaling).apply(x, positions=pos)[0]
        _check(got, x, "q", (freq, [0] * (turn + zeros), False, norm, None, 1e-6, scaling), pos)
        if norm == "none" and scaling == 1.0:
            f = turn + zeros
            assert torch.equal(got[..., turn:f], x[..., turn:f]) and torch.equal(got[..., f + turn:], x[..., f + turn:])
