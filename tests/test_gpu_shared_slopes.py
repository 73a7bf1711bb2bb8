"""Slopes at the ends of fp32's range, behind a shared prefix."""
from __future__ import annotations

import pytest
import torch

from shared_ref import Sessions, attend

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
MOST = torch.finfo(torch.float32).max


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("qn,hq,d,layout", [(1, 4, 128, "contig"), (2, 40, 64, "paged"), (70, 4, 64, "contig"), (60, 8, 512, "paged"),
                                            (60, 8, 256, "contig")])
def test_slopes_that_overflow_in_log2_units(qn, hq, d, layout):
    """fp32's largest slope leaves a query its own key alone, whose bias is 0 however steep it is:
    its value, to the last bit (one weight of itself over itself, 2^-17 off at most)."""
    s = Sessions(_gen(2), [qn + 200, qn + 3], 150, hkv=2, d=d, q=qn, layout=layout)
    q = torch.randn(2, hq, qn, d, generator=s.gen, device="cuda").to(BF16)
    slopes = torch.full((hq,), 0.01, device="cuda")
    slopes[1::2] = MOST
    slopes[0] = 3e38
    steep = slopes > 1
    for cap in (0.0, 20.0):
        got = s.rt.attend_shared(0, q, range(2), d ** -0.5, prefix_slot=2, slopes=slopes, softcap=cap)
        for i in range(2):
            keys, values = (torch.cat((x[2], x[i]), 1) for x in (s.k, s.v))
            total = keys.shape[1]
            own = values[:, total - qn:].repeat_interleave(hq // 2, 0)
            assert torch.equal(got[i][steep], own[steep])
            want, tol = attend(q[i], keys, values, list(range(total - qn, total)), d ** -0.5, cap=cap,
                               slopes=torch.where(steep, 0.01, slopes))
            assert bool(((got[i].double() - want).abs() <= tol)[~steep].all())
    slopes[1] = float("nan")
    got = s.rt.attend_shared(0, q, range(2), d ** -0.5, prefix_slot=2, slopes=slopes)
    assert bool(got[:, 1].isnan().all()) and bool(got[:, 0].isfinite().all()) and bool(got[:, 2:].isfinite().all())
