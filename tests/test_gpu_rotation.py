"""Heads normed and rotated on the GPU against the definition in 64 bits.

Tolerance: the result's rounding, 2^-8 relative, and the error ahead of it: the sum of
squares (21 fp32 roundings, halved by the root), the root (2^-23), three products and the
rotation's two (2^-24 each) stay below 2^-20 relative to the normed pair; sines and
cosines err by 2^-22.9 (the hardware's, over every 2^-24th of a turn) and, from the
angle's rounding to fp32 and 2^-32 of a turn, 2^-22.2. Together below 2^-19 of the pair's
magnitudes; 2^-18 is allowed."""
from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211707")


def _freqs(n: int, base: float = 1e6) -> torch.Tensor:
    return (base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float()


def _reference(x, kind, rot, positions, angle=None):
    """(result, allowed error) of heads x [n, H, Q, D] in 64 bits; positions [A, n, Q]."""
    freq, axes, adjacent, norm, weight, eps, scaling = rot
    y = x.double()
    d = y.shape[-1]
    if kind in {"none": "", "qk": "qk", "qkv": "qkv"}[norm]:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.double()
    slack = y.abs()
    f = freq.numel()
    if kind != "v" and f:
        if angle is None:
            angle = positions.double()[axes].permute(1, 2, 0) * freq.double().to(x.device)
        c, s = (scaling * angle.cos())[:, None], (scaling * angle.sin())[:, None]
        one, two = (slice(0, 2 * f, 2), slice(1, 2 * f, 2)) if adjacent else (slice(0, f), slice(f, 2 * f))
        a, b = y[..., one].clone(), y[..., two].clone()
        y = y.clone()
        y[..., one], y[..., two] = a * c - b * s, b * c + a * s
        slack = slack.clone()
        slack[..., one] = slack[..., two] = abs(scaling) * (a.abs() + b.abs())
    return y, 2.0 ** -8 * y.abs() + 2.0 ** -18 * slack


def _check(got, x, kind, rot, positions):
    want, tol = _reference(x, kind, rot, positions)
    assert got.dtype == BF16 and got.shape == x.shape
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), (kind, float((off - tol).max()))


def _positions(gen, axes, n, q, far):
    return torch.randint(-far, far, (axes, n, q), generator=gen, device="cuda")


CASES = [
    # d, hq, hkv, freqs, axes, order, adjacent, norm, n, q, far
    (128, 16, 8, 64, 1, "sections", False, "qk", 1, 1, 4096),
    (128, 16, 8, 64, 3, "alternate", False, "qk", 4, 1, 4096),
    (256, 8, 1, 128, 1, "sections", False, "qkv", 4, 2, 100000),
    (512, 8, 1, 64, 1, "sections", False, "qkv", 3, 29, 16384),
    (64, 16, 8, 32, 2, "sections", True, "qk", 5, 7, 2 ** 20),
    (128, 12, 4, 24, 4, "alternate", False, "none", 2, 33, 2 ** 31 - 1),
    (512, 5, 3, 256, 3, "sections", True, "qkv", 2, 3, 2 ** 31 - 1),
    (64, 3, 1, 8, 1, "sections", False, "qk", 7, 1, 50),
    (256, 1, 1, 0, 1, "sections", False, "qkv", 3, 5, 5),
    # enough heads that a group of lanes takes several: counts that are no multiple of them
    (128, 16, 8, 64, 3, "sections", False, "qk", 3, 1501, 16384),
    (64, 7, 2, 16, 2, "alternate", True, "qkv", 2, 9001, 9000),
    (256, 9, 3, 40, 1, "sections", False, "qkv", 1, 2113, 2 ** 31 - 1),
    (512, 6, 1, 128, 1, "sections", True, "qk", 1, 2500, 16384),
]


@pytest.mark.parametrize("d,hq,hkv,freqs,axes,order,adjacent,norm,n,q,far", CASES)
@pytest.mark.parametrize("packed", [False, True])
def test_matches_the_definition(d, hq, hkv, freqs, axes, order, adjacent, norm, n, q, far, packed):
    from kvrt import HeadRotation

    gen = torch.Generator(device="cuda").manual_seed(d + hq + q)
    x = torch.randn(n, q, hq + 2 * hkv, d, generator=gen, device="cuda") * torch.exp(
        2 * torch.randn(n, q, hq + 2 * hkv, 1, generator=gen, device="cuda"))
    parts = x.to(BF16).split([hq, hkv, hkv], 2)
    qw, kw = (None, None) if norm == "none" else (torch.randn(d, generator=gen, device="cuda").to(BF16), torch.rand(d) * 2)
    freq = _freqs(freqs)
    which = [f % axes if order == "alternate" else f * axes // max(freqs, 1) for f in range(freqs)]
    rot = HeadRotation(d, freq, axes=which, adjacent=adjacent, norm=norm, q_weight=qw, k_weight=kw, scaling=1.25)
    pos = _positions(gen, axes, n, q, far)
    if packed:
        heads = [p.reshape(n * q, -1, d) for p in parts]
        got = rot.apply(*heads, positions=pos.reshape(axes, n * q).to(torch.int32))
        got = [g.reshape(n, q, -1, d).transpose(1, 2) for g in got]
    else:
        got = rot.apply(*(p.transpose(1, 2) for p in parts), positions=pos)
        assert all(g.is_contiguous() for g in got)
    for g, p, kind, w in zip(got, parts, "qkv", (qw, None if kw is None else kw.cuda(), None)):
        _check(g, p.transpose(1, 2), kind, (freq, which, adjacent, norm, w, 1e-6, 1.25), pos)


def test_far_positions_and_frequencies_past_a_turn():
    from kvrt import HeadRotation

    freq = torch.tensor([1.0, 3.0, 6.5, 700.25, 1e-9, 0.0, -0.5, 2.0])
    rot = HeadRotation(64, freq, norm="none")
    pos = torch.tensor([[2 ** 31 - 1, -2 ** 31, 0, 1, -1, 2 ** 24 + 1, 123456789, -987654321]], device="cuda")
    x = torch.randn(1, 2, 8, 64, device="cuda").to(BF16)
    # whole turns dropped in whole numbers: a product in 64 bits would be off by 2^-13 of a turn
    angle = [[float(Fraction(f) * p / TWO_PI % 1 * TWO_PI) for f in freq.tolist()] for p in pos[0].tolist()]
    angle = torch.tensor(angle, dtype=torch.float64, device="cuda")[None]
    for p in (pos, pos.to(torch.int32)):
        got, _, _ = rot.apply(x, positions=p)
        # (the table's error, 2^-57 of a turn at 111 turns a position, is 2^-26 of one at 2^31)
        want, tol = _reference(x, "q", (freq, [0] * 8, False, "none", None, 0.0, 1.0), pos[None], angle)
        assert bool(((got.double() - want).abs() <= tol).all())
    assert torch.equal(got[..., 5], x[..., 5]) and torch.equal(got[..., 13], x[..., 13])  # a zero frequency
    assert torch.equal(got[..., 16:], x[..., 16:])                                        # dims that do not turn


def test_absent_kinds_and_values_that_pass():
    from kvrt import HeadRotation

    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(2, h, 3, 128, generator=gen, device="cuda").to(BF16) for h in (4, 2, 2))
    rot = HeadRotation(128, _freqs(64))
    pos = _positions(gen, 1, 2, 3, 500)[0]
    all_three = rot.apply(q, k, v, positions=pos)
    assert torch.equal(all_three[2], v)
    assert rot.apply(q, positions=pos)[1:] == (None, None)
    assert torch.equal(rot.apply(q, positions=pos)[0], all_three[0])
    only_k = rot.apply(None, k, positions=pos)
    assert only_k[0] is None and only_k[2] is None and torch.equal(only_k[1], all_three[1])
    empty = rot.apply(q[:, :, :0], k[:, :, :0], positions=pos[:, :0])
    assert empty[0].shape == (2, 4, 0, 128) and empty[1].shape == (2, 2, 0, 128)
    zero = rot.apply(torch.zeros_like(q), positions=pos)[0]
    assert not zero.any()


def test_in_place_and_strided_destinations():
    from kvrt import HeadRotation

    gen = torch.Generator(device="cuda").manual_seed(6)
    rot = HeadRotation(256, _freqs(64), norm="qkv", q_weight=torch.rand(256))
    x = torch.randn(3, 40, 10, 256, generator=gen, device="cuda").to(BF16)
    pos = _positions(gen, 1, 3, 40, 500)[0]
    heads = [t.transpose(1, 2) for t in x.split([8, 1, 1], 2)]
    want = rot.apply(*heads, positions=pos)
    # into a static cache of 64 rows at rows 5 .. 44, the rest untouched
    cache = torch.full((3, 1, 64, 256), 7.0, device="cuda", dtype=BF16)
    got = rot.apply(heads[0], heads[1], positions=pos, out=(torch.empty_like(want[0]), cache[:, :, 5:45], None))
    assert torch.equal(got[0], want[0]) and torch.equal(cache[:, :, 5:45], want[1])
    assert bool((cache[:, :, :5] == 7).all()) and bool((cache[:, :, 45:] == 7).all())
    got = rot.apply(*heads, positions=pos, out=tuple(heads))
    assert all(a is b for a, b in zip(got, heads))
    for h, w in zip(heads, want):
        assert torch.equal(h, w)


def test_positions_of_any_strides():
    from kvrt import HeadRotation

    gen = torch.Generator(device="cuda").manual_seed(7)
    rot = HeadRotation(64, _freqs(32), axes=[0, 1] * 16, norm="none")
    q = torch.randn(4, 2, 6, 64, generator=gen, device="cuda").to(BF16)
    for pos in (torch.arange(6, device="cuda")[None, None].expand(2, 4, 6),
                torch.arange(48, device="cuda", dtype=torch.int32).reshape(6, 4, 2).permute(2, 1, 0),
                torch.arange(96, device="cuda").reshape(2, 4, 12)[..., ::2]):
        got = rot.apply(q, positions=pos)[0]
        assert torch.equal(got, rot.apply(q, positions=pos.contiguous())[0])
        _check(got, q, "q", (_freqs(32), [0, 1] * 16, False, "none", None, 0.0, 1.0), pos)


def test_weights_may_be_written_in_place():
    from kvrt import HeadRotation

    rot = HeadRotation(64, [], q_weight=torch.ones(64), k_weight=torch.ones(64))
    x = torch.randn(1, 1, 1, 64, device="cuda").to(BF16)
    rot.q_weight.fill_(-2.0)
    q, k, _ = rot.apply(x, x)
    assert torch.equal(q, -2.0 * k)


def test_a_captured_call_replays_on_new_inputs():
    from kvrt import HeadRotation

    gen = torch.Generator(device="cuda").manual_seed(8)
    rot = HeadRotation(128, _freqs(64), axes=[0, 1, 2, 0] * 16)
    q = torch.randn(4, 16, 2, 128, generator=gen, device="cuda").to(BF16)
    k = torch.randn(4, 8, 2, 128, generator=gen, device="cuda").to(BF16)
    pos = _positions(gen, 3, 4, 2, 4000)
    rot.apply(q, k, positions=pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rot.apply(q, k, positions=pos)
    for i in range(4):
        pos.add_(i)
        q.mul_(-1.5)
        graph.replay()
        want = rot.apply(q, k, positions=pos)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_calls_on_another_stream():
    from kvrt import HeadRotation

    gen = torch.Generator(device="cuda").manual_seed(9)
    rot = HeadRotation(128, _freqs(64))
    q = torch.randn(4, 16, 300, 128, generator=gen, device="cuda").to(BF16)
    pos = _positions(gen, 1, 4, 300, 4000)
    want = rot.apply(q, positions=pos)[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = rot.apply(q, positions=pos)[0]
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    from kvrt import HeadRotation, KVRTError

    rot = HeadRotation(128, _freqs(64), axes=[0] * 32 + [1] * 32)
    q = torch.randn(2, 4, 3, 128, device="cuda").to(BF16)
    pos = torch.zeros(2, 2, 3, dtype=torch.int64, device="cuda")
    for bad in (dict(positions=None), dict(positions=pos.cpu()), dict(positions=pos, out=(None, q, None)),
                dict(positions=pos, out=(q[:1], None, None))):
        with pytest.raises(ValueError):
            rot.apply(q, **bad)
    for args in ((None,), (q.cpu(),), (q[0, 0],), (q, q[0])):
        with pytest.raises(ValueError):
            rot.apply(*args, positions=pos)
    for bad in (pos[:1], pos[0], pos.float(), pos[:, :1], torch.zeros(3, 2, 3, dtype=torch.int64, device="cuda")):
        with pytest.raises(KVRTError):
            rot.apply(q, positions=bad)
    with pytest.raises(TypeError):  # a type that no descriptor names
        rot.apply(q.half(), positions=pos)
    with pytest.raises(KVRTError):
        rot.apply(q.float(), positions=pos)
    with pytest.raises(KVRTError):
        rot.apply(q, q[:, :, :2], positions=pos)
    with pytest.raises(KVRTError):
        rot.apply(q[..., :64], positions=pos)
    with pytest.raises(KVRTError):  # rows that are not 16-byte aligned
        rot.apply(torch.zeros(2, 4, 3, 132, device="cuda", dtype=BF16)[..., 2:130], positions=pos)
    with pytest.raises(KVRTError):  # destination rows that coincide
        rot.apply(q, positions=pos, out=(torch.zeros(2, 1, 3, 128, device="cuda", dtype=BF16).expand(2, 4, 3, 128), None, None))
    assert math.isfinite(float(rot.apply(q, positions=pos)[0].float().sum()))


@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-6, 1e30])
@pytest.mark.parametrize("d", [64, 512])
def test_magnitudes_whose_squares_leave_fp32(eps, d):
    """Rows of 1e-39 to 3e38 side by side in a wave: the norm's squares would underflow or
    overflow, its quotient does not."""
    from kvrt import HeadRotation

    gen = torch.Generator(device="cuda").manual_seed(5)
    sizes = torch.tensor([1e-39, 1e-30, 1e-22, 1e-19, 3e-18, 1e-15, 1e-6, 1.0, 1e9, 1e15, 2e18, 1e19, 1e25, 2e37],
                         dtype=torch.float64, device="cuda")
    x = torch.randn(2, 14, 9, d, generator=gen, device="cuda", dtype=torch.float64).clamp(-4, 4) * sizes[:, None, None]
    x = x.to(BF16)
    x[0, 3, 2] = 0 if eps else 1
    freq = _freqs(d // 2)
    w = torch.rand(d, generator=gen, device="cuda") + 0.5
    rot = HeadRotation(d, freq, q_weight=w, eps=eps)
    pos = _positions(gen, 1, 2, 9, 5000)
    got = rot.apply(x, positions=pos)[0]
    f32 = torch.tensor(eps, dtype=torch.float32).item()
    want, tol = _reference(x, "q", (freq, [0] * (d // 2), False, "qk", w, f32, 1.0), pos)
    # answers below fp32's normal numbers round to a step of bf16's smallest, 2^-133
    assert bool(((got.double() - want).abs() <= tol + 2.0 ** -133).all())


@pytest.mark.parametrize("d,hq,hkv,tokens,adjacent", [(128, 7, 2, 2400, False), (512, 5, 1, 1000, True),
                                                      (64, 9, 3, 23000, True), (256, 13, 5, 3700, False)])
@pytest.mark.parametrize("in_place", [False, True])
def test_long_prompts_of_any_number_of_heads(d, hq, hkv, tokens, adjacent, in_place):
    """Heads in groups of four with one to three left over, from views of a projection, in
    calls of up to a million lanes and of more."""
    from kvrt import HeadRotation

    gen = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn(1, tokens, hq + 2 * hkv, d, generator=gen, device="cuda").to(BF16)
    q, k, v = (t.transpose(1, 2) for t in x.split([hq, hkv, hkv], 2))
    freq = _freqs(d // 2)
    w = torch.rand(d, generator=gen, device="cuda") + 0.5
    rot = HeadRotation(d, freq, adjacent=adjacent, norm="qkv", q_weight=w, k_weight=w.flip(0))
    pos = _positions(gen, 1, 1, tokens, 100000)
    before = x.clone()
    got = rot.apply(q, k, v, positions=pos, out=(q, k, v) if in_place else None)
    eps = torch.tensor(1e-6, dtype=torch.float32).item()
    for kind, g, src, weight in zip("qkv", got, before.split([hq, hkv, hkv], 2), (w, w.flip(0), None)):
        _check(g, src.transpose(1, 2), kind, (freq, [0] * (d // 2), adjacent, "qkv", weight, eps, 1.0), pos)
    if not in_place:
        assert torch.equal(x, before)
