"""Every kernel of attention behind a shared prefix against the definition in 64 bits
(tests/shared_ref.py): tests/test_shared_plan.py holds that the shapes run all of them."""
from __future__ import annotations

import pytest
import torch

from shared_forms import SHAPES, call
from shared_plan import plans
from shared_ref import Sessions
from test_gpu_shared_values import same_class

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_every_kernel(shape):
    c = call(*shape)
    n, d, hq, qn, prefix, masked = len(c["own"]), c["d"], c["hq"], c["q"], c["prefix"], not c["tiles"]
    gen = torch.Generator(device="cuda").manual_seed(d + hq + qn + n)
    s = Sessions(gen, c["own"], prefix or 0, hkv=c["hkv"], d=d, layout=c["layout"], window=c["window"], q=qn)
    masks = None
    if masked:  # of the first session's rows ahead of its queries, or of the prefix
        slot, rows = (n, prefix) if prefix else (0, max(c["own"][0] - qn, 1))
        masks = [None] * (n + 1)
        masks[slot] = torch.rand(min(rows, 70), generator=gen, device="cuda") < 0.6
        s.rt.set_prefix_attention(slot, masks[slot])
    slopes = torch.linspace(-0.01, 0.03, hq, device="cuda")
    for kw in ({}, dict(cap=15.0, slopes=slopes)):
        q = torch.randn(n, hq, qn, d, generator=gen, device="cuda").to(BF16)
        before = s.rt.counters()["launches"]
        got = s.rt.attend_shared(0, q, range(n), d ** -0.5, prefix_slot=None if prefix is None else n, softcap=kw.get("cap", 0.0),
                                 slopes=kw.get("slopes"))
        launches = s.rt.counters()["launches"] - before
        s.check(got, q, d ** -0.5, shared=prefix is not None, masks=masks, **kw)
        plan = plans([c])
        if plan is not None:  # (the division that the host test counts is the one that ran)
            p = plan[0]
            assert launches == (2 if (p["ranges"] if p["tiles"] else p["parts"]) > 1 else 1)
    assert s.rt.health() == 0


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_infinities_in_every_kernel(shape):
    """Infinities and NaN in the first, middle and last rows of the prefix and of the sessions."""
    c = call(*shape)
    n, d, hq, qn, prefix = len(c["own"]), c["d"], c["hq"], c["q"], c["prefix"]
    gen = torch.Generator(device="cuda").manual_seed(d + hq + qn + n + 1)
    s = Sessions(gen, c["own"], prefix or 0, hkv=c["hkv"], d=d, layout=c["layout"], window=c["window"], q=qn)
    for i in range(n + 1):
        rows = s.v[i].shape[1]
        if rows:
            s.v[i][:, 0, 1], s.v[i][:, rows // 2, d // 2 + 1], s.v[i][:, -1, d - 2] = float("inf"), float("-inf"), float("inf")
            s.v[i][:, rows // 3, 3], s.v[i][:, rows // 2, 3], s.v[i][:, rows // 5, 9] = float("-inf"), float("inf"), float("nan")
            s.load(i)
    masks = None
    if not c["tiles"]:
        slot, rows = (n, prefix) if prefix else (0, max(c["own"][0] - qn, 1))
        masks = [None] * (n + 1)
        masks[slot] = torch.rand(min(rows, 70), generator=gen, device="cuda") < 0.6
        s.rt.set_prefix_attention(slot, masks[slot])
    q = torch.randn(n, hq, qn, d, generator=gen, device="cuda").to(BF16)
    got = s.rt.attend_shared(0, q, range(n), d ** -0.5, prefix_slot=None if prefix is None else n)
    same_class(s, got, q, d ** -0.5, shared=prefix is not None, masks=masks)
    # the answer in the queries' place
    place = q.clone()
    again = s.rt.attend_shared(0, place, range(n), d ** -0.5, prefix_slot=None if prefix is None else n, out=place)
    assert again is place and torch.equal(place.view(torch.int16), got.view(torch.int16))
    assert s.rt.health() == 0
