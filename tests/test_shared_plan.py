"""How calls behind a shared prefix are divided (csrc/kvrt_shared_plan.h, compiled for the host)."""
from __future__ import annotations

import random

import pytest

from shared_forms import SHAPES, call
from shared_plan import every_form, forms, plans


def _plans(calls):
    got = plans(calls)
    if got is None:
        pytest.skip("g++ or HIP's headers not available")
    assert len(got) == len(calls)
    return got


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def test_partials_take_no_more_than_the_room_there_is():
    rng = random.Random(3)
    calls = []
    for _ in range(4000):
        hkv, q = rng.choice([1, 2, 8]), _log(rng, 1, 2048)
        n = _log(rng, 1, 64)
        hq = hkv * rng.choice([1, 2, 3, 8])
        if n * hq * q > 1 << 22:
            continue
        calls.append(dict(d=rng.choice([64, 128, 256, 512]), hkv=hkv, hq=hq, q=q, layout=rng.choice(["contig", "ring", "paged"]),
                          own=[q + _log(rng, 1, 5000) - 1 for _ in range(n)], prefix=rng.choice([None, 0, _log(rng, 1, 70000)]),
                          tiles=rng.random() < 0.7, window=rng.choice([0, 0, 1000]), room=rng.choice([0, 0, 1 << 20, 30 << 20, 256 << 20])))
    for c, p in zip(calls, _plans(calls)):
        assert p["bytes"] <= c["room"], (c, p)
        if c["room"] == 0:
            assert p["ranges" if p["tiles"] else "parts"] == 1
        if not c["tiles"]:
            assert not p["tiles"]


def test_one_call_grows_the_workspace_to_a_gigabyte_at_most():
    calls = [dict(d=512, hkv=1, hq=8, q=q, own=[q + 3] * 4, prefix=1400) for q in range(16, 2049)]
    calls += [dict(d=512, hkv=8, hq=64, q=q, own=[32768] * 16, prefix=16384) for q in (1, 7, 100, 4096)]
    assert max(p["bytes"] for p in _plans(calls)) <= 1 << 30


def test_the_gpu_tests_run_every_kernel():
    """The model picks the kernel, so that a change of its constants moves what a shape covers:
    tests/test_gpu_shared_forms.py then needs others for the forms named here."""
    calls = [call(*s) for s in SHAPES]
    ran = set().union(*(forms(c, p) for c, p in zip(calls, _plans(calls))))
    assert ran == every_form(), sorted(map(str, every_form() - ran))
