"""Attention behind a shared prefix, with capped and biased scores, against the definition in
64 bits (tests/shared_ref.py, which derives the tolerance)."""
from __future__ import annotations

import pytest
import torch

from shared_ref import Sessions, attend

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _q(gen, n, hq, qn, d, by=1.0):
    return (by * torch.randn(n, hq, qn, d, generator=gen, device="cuda")).to(BF16)


DECODES = [
    # lens, prefix, hq, hkv, d, layout, window, q
    ([1], 1, 8, 1, 256, "contig", 0, 1),
    ([1, 2, 3], 0, 16, 8, 128, "contig", 0, 1),
    ([5, 1, 33], 31, 16, 8, 128, "contig", 0, 1),
    ([40, 7, 64, 65], 97, 4, 4, 64, "contig", 0, 1),
    ([130, 64, 200], 512, 16, 8, 128, "contig", 0, 2),
    ([610, 500, 400, 333], 700, 16, 8, 128, "contig", 0, 1),
    ([2, 400], 300, 8, 1, 256, "contig", 0, 2),
    ([100, 31, 1, 64, 250], 333, 8, 1, 512, "contig", 0, 1),
    ([90, 17], 65, 8, 1, 512, "contig", 0, 2),
    ([33] * 17, 129, 12, 4, 128, "contig", 0, 1),
    (list(range(1, 65)), 260, 16, 8, 128, "contig", 0, 1),
    (list(range(70, 6, -1)), 100, 8, 1, 256, "contig", 0, 1),
    (list(range(3, 43)), 77, 8, 1, 512, "contig", 0, 2),
    ([300, 12, 90], 200, 16, 8, 128, "contig", 128, 1),
    ([300, 12, 90], 200, 8, 1, 256, "ring", 128, 1),
    ([20, 2, 700], 600, 16, 8, 64, "ring", 64, 2),
    ([5, 6, 9], 40, 4, 2, 128, "ring", 7, 1),
    ([5, 6, 9], 40, 4, 2, 128, "ring", 30, 2),
    ([100, 1, 33, 256], 130, 16, 8, 128, "paged", 0, 1),
    ([100, 2, 33, 256], 130, 8, 1, 512, "paged", 0, 2),
    ([100, 2, 33, 256], 130, 8, 1, 256, "paged", 90, 1),
    ([30, 31, 32], 15, 4, 2, 64, "paged", 0, 1),
]


@pytest.mark.parametrize("lens,prefix,hq,hkv,d,layout,window,qn", DECODES)
@pytest.mark.parametrize("score", ["plain", "capped", "biased", "both"])
def test_decode_steps(lens, prefix, hq, hkv, d, layout, window, qn, score):
    gen = _gen(len(lens) + prefix + d)
    s = Sessions(gen, lens, prefix, hkv=hkv, d=d, layout=layout, window=window, q=qn)
    cap = 12.0 if score in ("capped", "both") else 0.0
    slopes = torch.rand(hq, generator=gen, device="cuda") * 0.3 if score in ("biased", "both") else None
    q = _q(gen, len(lens), hq, qn, d, 2.0 if cap else 1.0)
    got = s.rt.attend_shared(0, q, range(s.n), d ** -0.5, prefix_slot=s.n, softcap=cap, slopes=slopes)
    s.check(got, q, d ** -0.5, cap=cap, slopes=slopes)
    got = s.rt.attend_shared(0, q, range(s.n), d ** -0.5, softcap=cap, slopes=slopes)
    s.check(got, q, d ** -0.5, shared=False, cap=cap, slopes=slopes)
    assert s.rt.health() == 0


CHUNKS = [
    ([3, 5], 9, 16, 8, 128, "contig", 0, 3),
    ([40, 17, 100], 65, 16, 8, 128, "contig", 0, 17),
    ([64], 300, 16, 8, 128, "contig", 0, 64),
    ([200, 129], 31, 8, 4, 128, "contig", 0, 129),
    ([50, 33], 100, 8, 1, 256, "contig", 0, 20),
    ([70, 41], 100, 8, 1, 512, "contig", 0, 41),
    ([300, 20], 90, 12, 4, 64, "contig", 0, 20),
    ([260, 200], 333, 16, 8, 128, "contig", 100, 150),
    ([260, 200], 64, 8, 1, 256, "ring", 100, 33),
    ([75, 90], 200, 16, 8, 128, "paged", 0, 75),
    ([75, 90], 200, 8, 1, 256, "paged", 60, 30),
    ([600], 0, 16, 8, 128, "contig", 0, 600),
    ([20, 33], 0, 8, 1, 256, "contig", 0, 3),
    ([900], 701, 8, 4, 128, "contig", 0, 40),
    ([45, 300], 1000, 8, 1, 512, "contig", 0, 45),
    ([333], 1400, 8, 1, 256, "ring", 700, 60),
    ([1203, 64], 515, 8, 2, 64, "paged", 0, 64),
    ([400, 390, 64], 64, 16, 4, 128, "paged", 0, 33),
    ([64, 65], 1, 8, 1, 256, "contig", 0, 64),
    ([100, 90], 33, 8, 2, 128, "contig", 10, 90),
    ([700] * 9, 130, 16, 8, 128, "contig", 0, 300),
]


@pytest.mark.parametrize("lens,prefix,hq,hkv,d,layout,window,qn", CHUNKS)
@pytest.mark.parametrize("score", ["plain", "both"])
def test_chunks(lens, prefix, hq, hkv, d, layout, window, qn, score):
    gen = _gen(len(lens) + prefix + d + qn)
    s = Sessions(gen, lens, prefix, hkv=hkv, d=d, layout=layout, window=window, q=qn)
    cap = 12.0 if score == "both" else 0.0
    slopes = torch.rand(hq, generator=gen, device="cuda") * 0.3 if score == "both" else None
    q = _q(gen, len(lens), hq, qn, d)
    got = s.rt.attend_shared(0, q, range(s.n), d ** -0.5, prefix_slot=s.n, softcap=cap, slopes=slopes)
    s.check(got, q, d ** -0.5, cap=cap, slopes=slopes)
    assert s.rt.health() == 0


@pytest.mark.parametrize("block", [1, 4, 16, 64])
def test_pages_of_any_size(block):
    gen = _gen(block)
    s = Sessions(gen, [50, 3, 129], 70, hkv=2, d=128, layout="paged", block=block)
    q = _q(gen, 3, 4, 1, 128)
    s.check(s.rt.attend_shared(0, q, range(3), 0.1, prefix_slot=3), q, 0.1)
    assert s.rt.health() == 0


@pytest.mark.parametrize("scale", [0.0, -0.25, 1.0, 30.0])
@pytest.mark.parametrize("cap", [0.0, 1e-3, 5.0, 1e6])
def test_scales_and_caps(scale, cap):
    gen = _gen(3)
    s = Sessions(gen, [70, 45], 130, hkv=2, d=64)
    q = _q(gen, 2, 8, 1, 64)
    s.check(s.rt.attend_shared(0, q, range(2), scale, prefix_slot=2, softcap=cap), q, scale, cap=cap)


@pytest.mark.parametrize("lens,qn,hq", [([60, 45, 90], 1, 4), ([60, 45, 90], 40, 4), ([60, 64, 90], 2, 40)])
def test_masks_of_the_prefix_and_of_the_sessions(lens, qn, hq):
    gen = _gen(qn)
    s = Sessions(gen, lens, 150, hkv=2, d=128)
    masks = [torch.rand(20, generator=gen, device="cuda") < 0.5, None,
             torch.zeros(90 - qn, dtype=torch.bool, device="cuda"), torch.rand(140, generator=gen, device="cuda") < 0.3]
    for slot, m in enumerate(masks):
        if m is not None:
            s.rt.set_prefix_attention(slot, m)
    q = _q(gen, 3, hq, qn, 128)
    s.check(s.rt.attend_shared(0, q, range(3), 0.09, prefix_slot=3), q, 0.09, masks=masks)
    # a canonical mask: only the first and last of 34 positions are seen; the hidden rows hold
    # infinities and NaN
    s.k[3][:, 1:33] = float("inf")
    s.v[3][:, 1:33] = float("nan")
    s.rt.set_prefix_attention(3, None)
    s.load(3)
    masks[3] = torch.zeros(34, dtype=torch.bool, device="cuda")
    masks[3][0] = masks[3][33] = True
    s.rt.set_prefix_attention(3, masks[3])
    got = s.rt.attend_shared(0, q, range(3), 0.09, prefix_slot=3)
    assert bool(got.isfinite().all())
    s.check(got, q, 0.09, masks=masks)


@pytest.mark.parametrize("qn,hq,hkv,d,layout,more", [
    (2, 8, 1, 256, "contig", 0), (2, 16, 8, 128, "paged", 0), (50, 8, 4, 128, "contig", 0), (40, 8, 1, 512, "paged", 0),
    (40, 4, 1, 64, "contig", 0), (40, 8, 1, 512, "contig", 1000), (90, 4, 4, 128, "contig", 900),
    (70, 8, 1, 256, "contig", 1000), (34, 2, 1, 64, "paged", 1100), (9, 8, 2, 128, "contig", 0)])
def test_a_row_that_a_query_does_not_see_does_not_reach_it(qn, hq, hkv, d, layout, more):
    gen = _gen(d)
    s = Sessions(gen, [qn + 30, qn + 1], 40 + more, hkv=hkv, d=d, q=qn, layout=layout)
    s.k[0][:, -1] = float("nan")            # seen by the last query only
    s.v[0][:, -1, ::3] = float("inf")
    s.v[1][:, -1] = float("nan")
    s.v[1][:, -2, 1::2] = float("-inf")     # seen by the last two
    for i in range(2):
        s.load(i)
    q = _q(gen, 2, hq, qn, d)
    got = s.rt.attend_shared(0, q, range(2), d ** -0.5, prefix_slot=2)
    assert bool(got[0, :, :-1].isfinite().all()) and bool(got[0, :, -1].isnan().all())
    s.check(got, q, d ** -0.5)
    if qn > 2:
        assert bool(got[1, :, :-2].isfinite().all())
    assert bool(got[1, :, -1].isnan().all())
    assert not bool(got[1, :, -2, 1::2].isfinite().any()) and bool(got[1, :, -2, ::2].isfinite().all())
    q[:, 0] = float("nan")                  # a head's query reaches no other head
    again = s.rt.attend_shared(0, q, range(2), d ** -0.5, prefix_slot=2)
    assert bool(again[:, 0].isnan().all()) and torch.equal(again[:, 1:].nan_to_num(7.0), got[:, 1:].nan_to_num(7.0))


def test_a_window_hides_the_prefix_of_some():
    gen = _gen(11)
    for layout in ("contig", "ring", "paged"):
        s = Sessions(gen, [3, 50, 63, 64, 65, 200], 90, hkv=2, d=128, layout=layout, window=64)
        s.v[6][:, :20] = float("nan")  # rows that no session sees any more
        s.load(6)
        q = _q(gen, 6, 4, 1, 128)
        got = s.rt.attend_shared(0, q, range(6), 0.09, prefix_slot=6)
        s.v[6][:, :20] = 0
        s.check(got, q, 0.09)


def test_same_as_a_clone_of_the_prefix():
    """The answer of sessions that hold a copy of the prefix, to the two calls' errors."""
    gen = _gen(12)
    s = Sessions(gen, [40, 21], 100, hkv=8, d=128)
    q = _q(gen, 2, 16, 1, 128)
    got = s.rt.attend_shared(0, q, range(2), 0.09, prefix_slot=2)
    from kvrt import KVRuntime, LayerSpec

    rt = KVRuntime([LayerSpec(kv_heads=8, head_dim=128)], n_slots=2, capacity=200)
    for i in range(2):
        rt.import_(i, 0, torch.cat((s.k[2], s.k[i]), 1)[None], torch.cat((s.v[2], s.v[i]), 1)[None])
    want = rt.attend(0, q, range(2), 0.09)
    assert float((got.float() - want.float()).abs().max()) <= 2 ** -7 * float(want.float().abs().max())


def test_shared_layers_read_their_source():
    from kvrt import KVRuntime, LayerSpec

    gen = _gen(13)
    rt = KVRuntime([LayerSpec(kv_heads=2, head_dim=64), LayerSpec(kv_heads=2, head_dim=64, shared_src=0)], n_slots=3,
                   capacity=64)
    for slot, rows in enumerate((10, 20, 33)):
        rt.import_(slot, 0, *(torch.randn(1, 2, rows, 64, generator=gen, device="cuda").to(BF16) for _ in range(2)))
    q = _q(gen, 2, 4, 1, 64)
    a, b = (rt.attend_shared(layer, q, [0, 1], 0.1, prefix_slot=2) for layer in (0, 1))
    assert torch.equal(a, b)
    swapped = rt.attend_shared(0, q.flip(0).contiguous(), [1, 0], 0.1, prefix_slot=2)
    assert torch.equal(swapped.flip(0), a)


@pytest.mark.parametrize("layout,window", [("contig", 0), ("ring", 48), ("paged", 0)])
def test_a_captured_step_replays_as_lengths_grow(layout, window):
    gen = _gen(14)
    lens = [30, 5, 61]
    s = Sessions(gen, lens, 75, hkv=2, d=128, layout=layout, window=window, spare=40)
    q = _q(gen, 3, 8, 1, 128)
    k, v = (torch.randn(3, 2, 1, 128, generator=gen, device="cuda").to(BF16) for _ in range(2))
    if layout == "paged":
        for i in range(3):
            s.rt.reserve(i, 20)
    s.rt.attend_shared(0, q, range(3), 0.09, prefix_slot=3)
    torch.cuda.synchronize()
    s.rt.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.rt.append(0, k, v, range(3))
        got = s.rt.attend_shared(0, q, range(3), 0.09, prefix_slot=3)
    s.rt.sync_lengths()
    assert [s.rt.seq_length(i) for i in range(3)] == lens  # nothing ran yet
    for step in range(6):
        q.copy_(_q(gen, 3, 8, 1, 128))
        k.copy_(torch.randn(3, 2, 1, 128, generator=gen, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for i in range(3):
            s.k[i], s.v[i] = torch.cat((s.k[i], k[i]), 1), torch.cat((s.v[i], v[i]), 1)
        s.check(got, q, 0.09)
    assert s.rt.health() == 0


def test_a_capture_without_workspace():
    """A first call inside a capture, whose partials do not fit: the undivided form."""
    gen = _gen(15)
    s = Sessions(gen, [1200], 300, hkv=1, d=64)
    q = _q(gen, 1, 32, 32, 64)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    s.rt.synchronize()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = s.rt.attend_shared(0, q, range(1), 0.12, prefix_slot=1)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        s.check(got, q, 0.12)


def test_rotated_appended_and_attended():
    """A decode step and a chunk as a model makes them: heads normed and rotated at their
    positions behind the prefix, rows appended, attention over prefix and rows."""
    from kvrt import HeadRotation

    gen = _gen(16)
    n, hq, hkv, d, p = 3, 16, 8, 128, 50
    lens = [20, 33, 7]
    inv = 1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)
    qw, kw = (torch.rand(d, generator=gen, device="cuda") + 0.5 for _ in range(2))
    rot = HeadRotation(d, inv, axes=[f % 3 for f in range(64)], q_weight=qw, k_weight=kw)
    s = Sessions(gen, lens, p, hkv=hkv, d=d)
    for qn in (1, 1, 2, 1):
        x = torch.randn(n, qn, hq + 2 * hkv, d, generator=gen, device="cuda").to(BF16)
        q, k, v = (t.transpose(1, 2) for t in x.split([hq, hkv, hkv], 2))
        base = p + torch.tensor(s.lens, device="cuda")[:, None] + torch.arange(qn, device="cuda")
        pos = torch.stack((base, base // 2, torch.zeros_like(base)))
        rq, rk, _ = rot.apply(q, k, positions=pos)

        def exact(t, weight):
            y = t.double()
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.double()
            angle = pos.double()[[f % 3 for f in range(64)]].permute(1, 2, 0)[:, None] * inv.cuda()
            a, b = y[..., :64], y[..., 64:]
            return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)

        for got, t, w in ((rq, q, qw), (rk, k, kw)):
            want = exact(t, w)
            pair = want.unflatten(-1, (2, 64)).norm(dim=-2).repeat(1, 1, 1, 2)
            assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -17 * pair).all())
        s.append(rk, v.contiguous())
        got = s.rt.attend_shared(0, rq, range(n), d ** -0.5, prefix_slot=n, softcap=30.0)
        s.check(got, rq, d ** -0.5, cap=30.0)
    assert s.rt.health() == 0


def test_refusals():
    from kvrt import KVRTError, KVRuntime, LayerSpec

    gen = _gen(17)
    s = Sessions(gen, [20, 2], 30, hkv=2, d=64)
    rt, q = s.rt, _q(gen, 2, 4, 1, 64)
    ok = dict(prefix_slot=2)
    good = rt.attend_shared(0, q, [0, 1], 0.1, **ok)
    before = rt.counters()

    def refused(code, layer=0, q=q, slots=(0, 1), scale=0.1, **kw):
        with pytest.raises(KVRTError) as e:
            rt.attend_shared(layer, q, slots, scale, **{**ok, **kw})
        assert e.value.code == code

    inf, nan = float("inf"), float("nan")
    for kw in (dict(layer=1), dict(layer=-1), dict(slots=(0, 0)), dict(slots=(0, 3)), dict(slots=(0, 2)), dict(slots=(0,)),
               dict(prefix_slot=3), dict(scale=nan), dict(scale=inf), dict(softcap=-1.0), dict(softcap=nan),
               dict(softcap=inf), dict(scale=1e30, softcap=1e-30), dict(q=q[:1]), dict(q=q[:, :3].contiguous()),
               dict(q=q[..., :32].contiguous()), dict(q=q.float()), dict(q=q[:, :, :0]),
               dict(q=torch.zeros(2, 4, 60, 64, device="cuda", dtype=BF16)), dict(out=q[:, :2]), dict(out=q.float()),
               dict(out=torch.zeros(2, 8, 1, 64, device="cuda", dtype=BF16)[:, ::2])):
        refused(-1, **kw)
    refused(-2, q=torch.zeros(2, 4, 3, 64, device="cuda", dtype=BF16))  # more queries than slot 1 has rows
    for bad in (torch.ones(3, device="cuda"), torch.ones(4), torch.ones(4, device="cuda", dtype=BF16),
                torch.ones(8, device="cuda")[::2], torch.ones(1, 4, device="cuda")):
        with pytest.raises(ValueError):
            rt.attend_shared(0, q, [0, 1], 0.1, prefix_slot=2, slopes=bad)
    with pytest.raises(ValueError):
        rt.attend_shared(0, q, [0, 1], 0.1, prefix_slot=-1)
    with pytest.raises(ValueError):
        rt.attend_shared(0, q.cpu(), [0, 1], 0.1)
    assert rt.counters() == before
    assert torch.equal(rt.attend_shared(0, q, [0, 1], 0.1, **ok), good)
    int8 = KVRuntime([LayerSpec(kv_heads=2, head_dim=64, layout="paged", dtype="int8")], n_slots=2, capacity=32,
                     pool_pages=8)
    int8.append(0, *(torch.zeros(2, 2, 1, 64, device="cuda", dtype=BF16),) * 2, [0, 1])
    with pytest.raises(KVRTError):
        int8.attend_shared(0, q[:1], [0], 0.1, prefix_slot=1)
    # rows that are gone: a ring's, after a rollback, and evicted pages of either slot
    ring = Sessions(gen, [100], 100, hkv=2, d=64, layout="ring", window=32)
    ring.rt.truncate(1, 0)
    assert ring.rt.attend_shared(0, q[:1], [0], 0.1, prefix_slot=1).isfinite().all()
    with pytest.raises(KVRTError):
        ring.rt.attend_shared(0, torch.zeros(1, 4, 3, 64, device="cuda", dtype=BF16), [0], 0.1)
    for slot in (0, 1):
        paged = Sessions(gen, [40], 40, hkv=2, d=64, layout="paged", window=20)
        paged.rt.evict(slot, 32)
        if slot == 0:
            with pytest.raises(KVRTError):
                paged.rt.attend_shared(0, q[:1], [0], 0.1, prefix_slot=1)
        else:  # the window no longer reaches the prefix
            assert paged.rt.attend_shared(0, q[:1], [0], 0.1, prefix_slot=1).isfinite().all()
            paged.rt.truncate(0, 3)
            with pytest.raises(KVRTError):
                paged.rt.attend_shared(0, q[:1], [0], 0.1, prefix_slot=1)


@pytest.mark.parametrize("cap", [0.5, 63.0, 65.0, 2e4])
@pytest.mark.parametrize("qn,hq,d,layout", [(1, 8, 128, "contig"), (70, 4, 64, "paged"), (40, 8, 256, "contig")])
def test_chunks_capped_on_both_sides_of_the_series(cap, qn, hq, d, layout):
    gen = _gen(int(cap) + qn)
    s = Sessions(gen, [qn + 200, qn], 410, hkv=2, d=d, q=qn, layout=layout)
    q = _q(gen, 2, hq, qn, d)
    slopes = torch.linspace(-0.02, 0.05, hq, device="cuda")
    for scale in (0.3, -2.0, 1e-4):
        s.check(s.rt.attend_shared(0, q, range(2), scale, prefix_slot=2, softcap=cap, slopes=slopes), q, scale, cap=cap,
                slopes=slopes)


@pytest.mark.parametrize("layout,window", [("contig", 0), ("ring", 900), ("paged", 0)])
def test_a_captured_chunk_replays_as_lengths_grow(layout, window):
    """Key ranges of a chunk are the device's own: sized for the lengths that the capture
    knew, right for those of each replay, between other calls that use the workspace."""
    gen = _gen(17)
    lens = [40, 33]
    s = Sessions(gen, lens, 700, hkv=1, d=256, layout=layout, window=window, spare=200, q=40,
                 ring=1000 if layout == "ring" else None)
    q = _q(gen, 2, 8, 40, 256)
    k, v = (torch.randn(2, 1, 30, 256, generator=gen, device="cuda").to(BF16) for _ in range(2))
    if layout == "paged":
        for i in range(2):
            s.rt.reserve(i, 160)
    other = _q(gen, 2, 8, 1, 256)
    s.check(s.rt.attend_shared(0, q[:, :, :33].contiguous(), range(2), 0.06, prefix_slot=2), q[:, :, :33], 0.06)
    s.check(s.rt.attend_shared(0, other, range(2), 0.06, prefix_slot=2), other, 0.06)
    torch.cuda.synchronize()
    s.rt.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for j in range(30):  # (rows are appended at most two at a time)
            s.rt.append(0, k[:, :, j:j + 1].contiguous(), v[:, :, j:j + 1].contiguous(), range(2))
        got = s.rt.attend_shared(0, q, range(2), 0.06, prefix_slot=2, softcap=30.0)
    for step in range(4):
        q.copy_(_q(gen, 2, 8, 40, 256))
        graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            s.k[i], s.v[i] = torch.cat((s.k[i], k[i]), 1), torch.cat((s.v[i], v[i]), 1)
        s.check(got, q, 0.06, cap=30.0)
        s.rt.synchronize()  # (the capture bound another stream)
        s.rt.sync_lengths()
        eager = s.rt.attend_shared(0, other, range(2), 0.06, prefix_slot=2)
        s.check(eager, other, 0.06)
        s.rt.synchronize()
    assert s.rt.health() == 0


def test_answers_go_to_memory_of_the_same_gpu():
    s = Sessions(_gen(18), [9], 5, hkv=1, d=64)
    q = _q(s.gen, 1, 2, 1, 64)
    with pytest.raises(ValueError):
        s.rt.attend_shared(0, q, [0], 0.1, prefix_slot=1, out=torch.zeros(1, 2, 1, 64, dtype=BF16))
    out = torch.full((2, 2, 1, 64), 7.0, device="cuda", dtype=BF16)
    got = s.rt.attend_shared(0, q, [0], 0.1, prefix_slot=1, out=out[:1])
    s.check(got, q, 0.1)
    assert bool((out[1] == 7).all())
    again = q.clone()
    assert torch.equal(s.rt.attend_shared(0, again, [0], 0.1, prefix_slot=1, out=again), got) and torch.equal(again, got)


@pytest.mark.parametrize("layout", ["contig", "paged"])
@pytest.mark.parametrize("hkv,d,n", [(8, 128, 5), (1, 512, 3), (2, 64, 1)])
def test_a_captured_step_replays_on_sessions_many_times_as_long(layout, hkv, d, n):
    """A launch's ranges are made for the lengths at its capture: longer sessions take longer
    ranges, and ones of unequal growth each their share."""
    gen = _gen(d)
    s = Sessions(gen, [33] * n, 300, hkv=hkv, d=d, layout=layout, spare=4000)
    q = _q(gen, n, 2 * hkv, 1, d)
    if layout == "paged":
        for i in range(n):
            s.rt.reserve(i, 3900)
    s.check(s.rt.attend_shared(0, q, range(n), 0.1, prefix_slot=n), q, 0.1)
    s.rt.synchronize()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = s.rt.attend_shared(0, q, range(n), 0.1, prefix_slot=n)
    for step, lens in enumerate(([700] * n, [3800, 40, 900, 2000, 1][:n], [1] * n, [5, 3900, 17, 33, 64][:n])):
        s.rt.synchronize()
        s.rt.sync_lengths()
        for i, rows in enumerate(lens):
            s.rt.truncate(i, 0)
            s.k[i], s.v[i] = (torch.randn(hkv, rows, d, generator=gen, device="cuda").to(BF16) for _ in range(2))
            s.rt.import_(i, 0, s.k[i][None], s.v[i][None])
        s.lens = list(lens)
        s.rt.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        s.check(got, q, 0.1)
    assert s.rt.health() == 0


def test_two_captured_calls_and_a_larger_one_between_them():
    """Captured calls of one runtime keep the workspace that they were captured with."""
    gen = _gen(20)
    s = Sessions(gen, [500, 420, 60], 900, hkv=2, d=128, spare=100)
    a, b, c = (_q(gen, 3, 16, qn, 128) for qn in (1, 40, 60))
    small = _q(gen, 1, 16, 1, 128)
    s.rt.attend_shared(0, a, range(3), 0.1, prefix_slot=3)
    s.rt.synchronize()
    graphs, outs = [], []
    for q in (a, b):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.rt.attend_shared(0, q, range(3), 0.1, prefix_slot=3, softcap=20.0))
        s.rt.synchronize()
        graphs.append(g)
    for step in range(3):
        for x in (a, b):
            x.copy_(_q(gen, 3, 16, x.shape[2], 128))
        graphs[step % 2].replay()
        graphs[1 - step % 2].replay()
        torch.cuda.synchronize()
        s.check(outs[0], a, 0.1, cap=20.0)
        s.check(outs[1], b, 0.1, cap=20.0)
        eager = s.rt.attend_shared(0, c, range(3), 0.1, prefix_slot=3)
        s.check(eager, c, 0.1)
        s.rt.synchronize()


def test_rows_behind_the_items_stay_as_they_were():
    gen = _gen(21)
    for qn, d, hkv in ((1, 128, 2), (30, 64, 1), (70, 256, 1), (3, 512, 1)):
        s = Sessions(gen, [80, 130], 200, hkv=hkv, d=d)
        q = _q(gen, 2, 4 * hkv, qn, d)
        room = torch.full((4, 4 * hkv, qn, d), 3.0, device="cuda", dtype=BF16)
        s.check(s.rt.attend_shared(0, q, range(2), 0.1, prefix_slot=2, out=room[1:3]), q, 0.1)
        assert bool((room[0] == 3).all()) and bool((room[3] == 3).all())


@pytest.mark.parametrize("hq,d", [(16, 64), (64, 64), (64, 128), (64, 256), (64, 512)])
@pytest.mark.parametrize("imported", [False, True])
@pytest.mark.parametrize("qn,prefix,evict_prefix", [(30, 0, 0), (30, 50, 0), (30, 300, 0), (300, 620, 496)])
def test_chunks_over_evicted_pages(qn, prefix, evict_prefix, imported, hq, d):
    """Pages ahead of the window are gone, also those that share a 32-key tile with its start."""
    from kvrt import KVRuntime

    window = 500
    s = Sessions(_gen(qn), [679, 679], prefix, hkv=1, d=d, layout="paged", window=window, q=qn)
    q = _q(s.gen, 2, hq, qn, d)
    oldest = 679 - qn - window + 1
    for i in range(2):
        if oldest >= 16:
            s.rt.evict(i, oldest // 16 * 16)
    if evict_prefix:
        s.rt.evict(2, evict_prefix)
    kept = [oldest // 16 * 16 if oldest >= 16 else 0] * 2 + [evict_prefix]
    if imported:  # sessions that never had those pages
        s.rt = KVRuntime(s.rt.layers, n_slots=3, capacity=700, max_q=2, block_size=16, pool_pages=150, pool_seed=3)
        for i, first in enumerate(kept):
            s.rt.import_(i, 0, s.k[i][None].contiguous(), s.v[i][None].contiguous(), first_pos=first)
    got = s.rt.attend_shared(0, q, range(2), 0.1, prefix_slot=2)
    torch.cuda.synchronize()
    assert s.rt.health() == 0
    s.check(got, q, 0.1)


def test_refusals_of_scales_past_fp32_in_log2_units():
    from kvrt import KVRTError

    s = Sessions(_gen(22), [9], 5, hkv=1, d=64)
    q = _q(s.gen, 1, 2, 1, 64)
    for kw in (dict(scale=3e38), dict(scale=-3e38), dict(scale=0.1, softcap=3e38)):
        with pytest.raises(KVRTError) as e:
            s.rt.attend_shared(0, q, [0], prefix_slot=1, **kw)
        assert e.value.code == -1
    s.check(s.rt.attend_shared(0, q, [0], 0.1, prefix_slot=1, softcap=2e38), q, 0.1)
    for none in ([], ()):
        with pytest.raises(KVRTError):
            s.rt.attend_shared(0, q[:0], none, 0.1, prefix_slot=1)


@pytest.mark.parametrize("hq,hkv", [(6, 2), (5, 1), (21, 3), (11, 11)])
@pytest.mark.parametrize("qn,d,layout,window", [(1, 64, "paged", 0), (2, 256, "contig", 0), (33, 128, "paged", 50),
                                                (130, 64, "contig", 0), (47, 512, "ring", 90)])
def test_groups_of_odd_numbers_of_heads(hq, hkv, qn, d, layout, window):
    gen = _gen(hq * qn)
    s = Sessions(gen, [qn + 5, 171, qn], 97, hkv=hkv, d=d, layout=layout, window=window, q=qn)
    q = _q(gen, 3, hq, qn, d)
    slopes = torch.linspace(-0.03, 0.04, hq, device="cuda")
    s.check(s.rt.attend_shared(0, q, range(3), 0.11, prefix_slot=3), q, 0.11)
    s.check(s.rt.attend_shared(0, q, range(3), 0.11, prefix_slot=3, softcap=9.0, slopes=slopes), q, 0.11, cap=9.0,
            slopes=slopes)


@pytest.mark.parametrize("layout", ["contig", "paged"])
def test_rows_past_32_bits_of_bytes_and_elements(layout):
    """A prefix of 8.5 million rows of 1 KiB, whose end lies 8.7 GB behind its slot's start, and
    sessions in slots behind it."""
    from kvrt import KVRuntime, LayerSpec

    gen = _gen(23)
    rows, window, d = 8_500_000, 70, 512
    rt = KVRuntime([LayerSpec(kv_heads=1, head_dim=d, layout=layout, window=window)], n_slots=3, capacity=rows + 20,
                   block_size=64, pool_pages=rows // 64 + 20 if layout == "paged" else 0, pool_seed=5)
    k, v = (torch.zeros(1, 1, rows, d, device="cuda", dtype=BF16) for _ in range(2))
    for t in (k, v):
        t[:, :, -200:] = torch.randn(200, d, generator=gen, device="cuda")
    rt.import_(0, 0, k, v)
    own = [[torch.randn(1, n, d, generator=gen, device="cuda").to(BF16) for _ in range(2)] for n in (33, 61)]
    for i, (a, b) in enumerate(own):
        rt.import_(i + 1, 0, a[None], b[None])
    for hq, qn in ((4, 1), (32, 33)):
        q = _q(gen, 2, hq, qn, d)
        got = rt.attend_shared(0, q, [1, 2], 0.05, prefix_slot=0)
        for i, (a, b) in enumerate(own):
            keys, values = torch.cat((k[0][:, -200:], a), 1), torch.cat((v[0][:, -200:], b), 1)
            n = keys.shape[1]
            want, tol = attend(q[i], keys, values, list(range(n - qn, n)), 0.05, window=window)
            assert bool(((got[i].double() - want).abs() <= tol).all())
    assert rt.health() == 0


@pytest.mark.parametrize("block", [1, 8, 128])
@pytest.mark.parametrize("d,window", [(64, 0), (128, 333), (512, 90)])
def test_chunks_on_pages_of_any_size(block, d, window):
    gen = _gen(block + d)
    s = Sessions(gen, [611, 45], 270, hkv=1, d=d, layout="paged", block=block, window=window, q=45)
    q = _q(gen, 2, 32, 45, d)
    s.check(s.rt.attend_shared(0, q, range(2), 0.08, prefix_slot=2), q, 0.08)
    assert s.rt.health() == 0


def test_calls_on_another_stream():
    gen = _gen(24)
    s = Sessions(gen, [200, 31], 400, hkv=2, d=128)
    for qn in (1, 30):
        q = _q(gen, 2, 8, qn, 128)
        here = s.rt.attend_shared(0, q, range(2), 0.1, prefix_slot=2)
        s.check(here, q, 0.1)
        s.rt.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = s.rt.attend_shared(0, q, range(2), 0.1, prefix_slot=2)
            s.rt.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(here, there)


@pytest.mark.parametrize("d,lens,prefix,layout,window", [(128, [9000, 8000, 7], 20000, "contig", 0),
                                                         (512, [3000, 2500, 1], 5000, "contig", 0),
                                                         (64, [20000, 40000, 33], 17000, "ring", 50000)])
def test_calls_that_outgrow_the_caches(d, lens, prefix, layout, window):
    gen = _gen(25)
    s = Sessions(gen, lens, prefix, hkv=8, d=d, layout=layout, window=window)
    for qn, masked in ((1, False), (1, True)):
        q = _q(gen, 3, 16, qn, d)
        masks = None
        if masked:
            masks = [None, None, None, torch.rand(500, generator=gen, device="cuda") < 0.5]
            s.rt.set_prefix_attention(3, masks[3])
        s.check(s.rt.attend_shared(0, q, range(3), 0.1, prefix_slot=3), q, 0.1, masks=masks)
    assert s.rt.health() == 0
