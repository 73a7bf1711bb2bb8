"""Infinities and NaN among the rows that queries see, behind a shared prefix: the answers'
class (a number, which infinity, NaN) is the definition's, wherever the rows lie."""
from __future__ import annotations

import pytest
import torch

from shared_ref import Sessions, attend

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
INF = float("inf")


def same_class(s, got, q, scale, *, shared=True, masks=None, **kw):
    """got against the reference: numbers within its tolerance, the same infinities, NaN for NaN."""
    qn = q.shape[2]
    for i in range(s.n):
        parts = ([s.n] if shared else []) + [i]
        keys, values = (torch.cat([x[j] for j in parts], 1) for x in (s.k, s.v))
        total = keys.shape[1]
        visible = torch.ones(total, dtype=torch.bool, device="cuda")
        for j, at in zip(parts, (0, s.k[s.n].shape[1] if shared else 0)):
            m = masks[j] if masks is not None else None
            if m is not None:
                visible[at:at + min(m.numel(), s.k[j].shape[1])] = m[:s.k[j].shape[1]]
        want, tol = attend(q[i], keys, values, list(range(total - qn, total)), scale, window=s.window, visible=visible, **kw)
        x = got[i].double()
        number = want.isfinite()
        assert bool(((x - want).abs() <= tol)[number].all()), i
        assert torch.equal(x.isnan(), want.isnan()), (i, int((x.isnan() != want.isnan()).sum()))
        assert torch.equal(x[~number].nan_to_num(7.0), want[~number].nan_to_num(7.0)), i


# lens, prefix, hq, hkv, d, layout, window, q
SHAPES = [
    ([70], 0, 8, 1, 256, "contig", 0, 1),
    ([70, 33], 0, 4, 4, 64, "contig", 0, 1),
    ([130, 64, 200], 512, 16, 8, 128, "contig", 0, 2),
    ([610, 500, 400, 333], 700, 16, 8, 128, "contig", 0, 1),
    (list(range(1, 65)), 260, 16, 8, 128, "contig", 0, 1),
    ([100, 200, 90] * 14, 260, 8, 1, 256, "contig", 0, 1),
    (list(range(3, 43)), 177, 8, 1, 512, "contig", 0, 2),
    ([300, 120, 90], 200, 8, 1, 256, "ring", 128, 1),
    ([100, 90, 33, 256], 130, 8, 1, 512, "paged", 0, 2),
    ([100, 90, 133], 130, 16, 8, 64, "paged", 0, 1),
    ([64], 300, 16, 8, 128, "contig", 0, 64),
    ([260, 200], 333, 16, 8, 128, "contig", 100, 150),
    ([70, 61], 100, 8, 1, 512, "contig", 0, 41),
    ([450, 300], 1000, 8, 1, 512, "contig", 0, 45),
    ([333], 1400, 8, 1, 256, "ring", 700, 60),
    ([75, 90], 200, 16, 8, 128, "paged", 0, 75),
    ([300, 64], 515, 8, 2, 64, "paged", 0, 64),
    ([700, 650], 130, 16, 8, 128, "contig", 0, 300),
]


@pytest.mark.parametrize("lens,prefix,hq,hkv,d,layout,window,qn", SHAPES)
@pytest.mark.parametrize("cap", [0.0, 9.0])
def test_a_seen_infinity_of_v_stays_one(lens, prefix, hq, hkv, d, layout, window, qn, cap):
    """Weights of the rows are above 2^-30: an infinity times one is that infinity, two of
    unlike sign are NaN. Rows in tiles that all queries see and in those that some see."""
    gen = torch.Generator(device="cuda").manual_seed(d + qn)
    s = Sessions(gen, lens, prefix, hkv=hkv, d=d, layout=layout, window=window, q=qn)
    for i in range(s.n + 1):
        rows = s.v[i].shape[1]
        for j, (dim, x) in enumerate([(1, INF), (2, -INF), (d // 2, INF), (d - 1, -INF), (5, INF), (5, -INF), (7, float("nan"))]):
            if i != 0 and rows:  # (session 0 sees those of the prefix alone)
                s.v[i][:, (3 + 17 * j) % rows, dim] = x
        s.load(i)
    q = torch.randn(s.n, hq, qn, d, generator=gen, device="cuda").to(BF16)
    got = s.rt.attend_shared(0, q, range(s.n), d ** -0.5, prefix_slot=s.n, softcap=cap)
    same_class(s, got, q, d ** -0.5, cap=cap)
    got = s.rt.attend_shared(0, q, range(s.n), d ** -0.5, softcap=cap)
    same_class(s, got, q, d ** -0.5, shared=False, cap=cap)
    assert s.rt.health() == 0


@pytest.mark.parametrize("lens,prefix,hq,hkv,d,layout,window,qn", SHAPES[2:4] + SHAPES[6:7] + SHAPES[10:14])
@pytest.mark.parametrize("cap", [0.0, 9.0, 100.0])
def test_a_seen_infinity_of_k(lens, prefix, hq, hkv, d, layout, window, qn, cap):
    """A score of -infinity weighs nothing and one of infinity makes the row NaN; capped they
    are the cap."""
    gen = torch.Generator(device="cuda").manual_seed(d + qn)
    s = Sessions(gen, lens, prefix, hkv=hkv, d=d, layout=layout, window=window, q=qn)
    for i in range(1, s.n + 1):
        s.k[i][:, s.k[i].shape[1] // 2, 3] = INF
        s.load(i)
    q = torch.randn(s.n, hq, qn, d, generator=gen, device="cuda").to(BF16)
    got = s.rt.attend_shared(0, q, range(s.n), d ** -0.5, prefix_slot=s.n, softcap=cap)
    same_class(s, got, q, d ** -0.5, cap=cap)
    assert s.rt.health() == 0
