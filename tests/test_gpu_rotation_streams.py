"""A rotation is ready when its constructor returns, on whatever stream it is then used."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_used_on_another_stream_than_it_was_made_on():
    from kvrt import HeadRotation

    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, 4, 3, 128, generator=gen, device="cuda").to(BF16)
    w = torch.rand(128, generator=gen, device="cuda") + 0.5
    freq = (1e4 ** (-torch.arange(64, device="cuda", dtype=torch.float64) / 64))
    pos = torch.arange(6, device="cuda").reshape(2, 3)
    want = HeadRotation(128, freq, q_weight=w).apply(x, positions=pos)[0].clone()
    a = torch.randn(4096, 4096, device="cuda")
    made, used = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(made):
            for _ in range(20):
                a = (a @ a).clamp(-1, 1)  # work ahead of the copies of the weights
            rot = HeadRotation(128, freq.cpu(), q_weight=w)
        with torch.cuda.stream(used):
            got = rot.apply(x, positions=pos)[0]
        used.synchronize()
        assert torch.equal(got, want)
        torch.cuda.synchronize()
