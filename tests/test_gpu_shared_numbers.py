"""Caps and scales at the ends of fp32's range, behind a shared prefix."""
from __future__ import annotations

import pytest
import torch

from shared_ref import Sessions

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def test_caps_that_fp32_does_not_hold():
    """A cap that fp32 rounds to 0 would be none; a quotient of scale and cap that overflows in
    the tanh's units would make a product of 0 NaN."""
    from kvrt import KVRTError

    s = Sessions(_gen(1), [40, 33], 50, hkv=1, d=64)
    q = torch.zeros(2, 2, 1, 64, device="cuda", dtype=BF16)
    for cap in (1e-60, 2.0 ** -150):
        with pytest.raises(ValueError):
            s.rt.attend_shared(0, q, range(2), 0.1, prefix_slot=2, softcap=cap)
    for scale, cap in ((1e30, 5e-9), (-1e30, 5e-9), (2e38, 1.0)):
        with pytest.raises(KVRTError) as e:
            s.rt.attend_shared(0, q, range(2), scale, prefix_slot=2, softcap=cap)
        assert e.value.code == -1
    # one that does not: all scores are 0
    s.check(s.rt.attend_shared(0, q, range(2), 1e29, prefix_slot=2, softcap=1e-9), q, 1e29, cap=1e-9)
    s.check(s.rt.attend_shared(0, q, range(2), 0.0, prefix_slot=2, softcap=2.0 ** -149), q, 0.0, cap=2.0 ** -149)
