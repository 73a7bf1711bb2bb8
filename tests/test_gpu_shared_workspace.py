"""The workspace that the parts of attention behind a shared prefix are left in: how far it
grows, and calls that it does not grow for."""
from __future__ import annotations

import pytest
import torch

from shared_ref import Sessions

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _taken() -> int:
    """GPU memory in use beside torch's own."""
    torch.cuda.synchronize()
    free, total = torch.cuda.mem_get_info()
    return total - free - torch.cuda.memory_reserved()


def test_calls_of_rising_size_do_not_pile_up_workspaces():
    """Every call of a rising sequence needs a little more than the one before: what is kept of
    earlier workspaces stays below the last one, which is at most twice the largest need."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    top, hq, d = 260, 8, 512
    s = Sessions(gen, [top] * 4, 1400, hkv=1, d=d, spare=4)
    q = torch.randn(4, hq, top, d, generator=gen, device="cuda").to(BF16)
    s.rt.attend_shared(0, q[:, :, :1].contiguous(), range(4), 0.04, prefix_slot=4)
    before = _taken()
    for qn in range(8, top + 1):
        x = q[:, :, :qn].contiguous()
        got = s.rt.attend_shared(0, x, range(4), 0.04, prefix_slot=4)
        if qn % 63 == 8:
            s.check(got, x, 0.04)
    # of a call: 4 * 8 * 260 rows of 512 fp32 values and two more, in at most 32 parts where rows
    # are few and 8 where they fill the card; 4 * 8 * 64 rows of 32 parts are as many bytes
    need = 4 * hq * top * (d * 4 + 8) * 8
    assert _taken() - before <= 4 * need, (_taken() - before, need)


@pytest.mark.parametrize("d,hq,hkv,qn,lens,prefix", [(64, 32, 1, 32, [1200], 300), (512, 8, 1, 2, [700] * 5, 4000),
                                                     (256, 8, 1, 100, [300, 900], 3000)])
def test_a_capture_takes_a_division_that_fits(d, hq, hkv, qn, lens, prefix):
    """First calls inside a capture, the workspace as it was at creation; the same call again
    once an eager one has grown it."""
    gen = torch.Generator(device="cuda").manual_seed(d)
    s = Sessions(gen, lens, prefix, hkv=hkv, d=d)
    q = torch.randn(len(lens), hq, qn, d, generator=gen, device="cuda").to(BF16)
    for eager in (False, True):
        if eager:
            s.check(s.rt.attend_shared(0, q, range(s.n), d ** -0.5, prefix_slot=s.n), q, d ** -0.5)
        s.rt.synchronize()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = s.rt.attend_shared(0, q, range(s.n), d ** -0.5, prefix_slot=s.n)
        s.rt.synchronize()
        for _ in range(3):
            q.copy_(torch.randn(q.shape, generator=gen, device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            s.check(got, q, d ** -0.5)
    assert s.rt.health() == 0
