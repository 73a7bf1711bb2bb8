"""Measured passes of the step around a cache: heads normed and rotated, attention after a shared prefix.

``prepare`` builds what a serving program keeps (a rotation with its tables, a
runtime whose sessions hold their rows) and a step's inputs; ``run`` makes one
pass and returns all it computed.

Kinds:

* ``rotate``  query and key heads (with ``norm`` "qkv" value heads too) normed and
  rotated by their positions along one to three axes, in one pass;
* ``attend``  attention of each session's newest rows over a prefix that all
  sessions share (``prefix`` rows, 0: none) and its own rows behind it, the scores
  plain, capped by a tanh (``cap``) or with a bias by distance (``slopes``).

A session's own length is ``first - gap * i`` for session i; a projection's rows
are views of one [rows, (hq + 2 hkv) * d] product, as a model has them.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PKG = Path(__file__).resolve().parent.parent / "gemma-4-omni_amd"
if str(_PKG) not in sys.path:
    sys.path.insert(0, str(_PKG))

BF16 = torch.bfloat16
EPS = 1e-6
PAGE = 16


def listed() -> list[dict]:
    return [
        # One token of one stream through a thinker layer: the smallest rotation.
        {"name": "rotate_b1", "kind": "rotate", "n": 1, "q": 1, "hq": 8, "hkv": 1, "d": 256, "freqs": 128, "axes": 1,
         "order": "sections", "adjacent": 0, "norm": "qkv", "far": 4096},
        # A talker frame of four sessions: three axes that alternate from frequency to frequency.
        {"name": "rotate_talker_x4", "kind": "rotate", "n": 4, "q": 1, "hq": 16, "hkv": 8, "d": 128, "freqs": 64,
         "axes": 3, "order": "alternate", "adjacent": 0, "norm": "qk", "far": 4096},
        # A text chunk of four streams into a full layer of which a quarter of the dims turn.
        {"name": "rotate_full_q291", "kind": "rotate", "n": 4, "q": 291, "hq": 8, "hkv": 1, "d": 512, "freqs": 64,
         "axes": 1, "order": "sections", "adjacent": 0, "norm": "qkv", "far": 16384},
        # Long prompts of four sessions, positions of time, height and width in sections: the largest rotation.
        {"name": "rotate_prompt", "kind": "rotate", "n": 4, "q": 4096, "hq": 16, "hkv": 8, "d": 128, "freqs": 64,
         "axes": 3, "order": "sections", "adjacent": 0, "norm": "qk", "far": 16384},
        # A talker frame of four sessions that share a voice prompt, one layer.
        {"name": "shared_talker_x4", "kind": "attend", "n": 4, "hq": 16, "hkv": 8, "d": 128, "layout": "contig",
         "window": 0, "prefix": 2048, "first": 610, "gap": 92, "q": 1, "cap": 0.0, "slopes": 0},
        # Sixty-four sessions behind one long prompt: a serving step.
        {"name": "shared_serve_x64", "kind": "attend", "n": 64, "hq": 16, "hkv": 8, "d": 128, "layout": "contig",
         "window": 0, "prefix": 4096, "first": 1500, "gap": 20, "q": 1, "cap": 0.0, "slopes": 0},
        # Two queries of a full layer (head_dim 512), sixteen streams behind one prompt.
        {"name": "shared_full_q2", "kind": "attend", "n": 16, "hq": 8, "hkv": 1, "d": 512, "layout": "contig",
         "window": 0, "prefix": 4096, "first": 400, "gap": 20, "q": 2, "cap": 0.0, "slopes": 0},
        # A sliding layer of sixteen streams: the window still reaches into the prefix of most.
        {"name": "shared_sliding_x16", "kind": "attend", "n": 16, "hq": 8, "hkv": 1, "d": 256, "layout": "ring",
         "window": 512, "prefix": 2048, "first": 600, "gap": 37, "q": 1, "cap": 0.0, "slopes": 0},
        # A text chunk of four sessions behind a shared prompt: the most arithmetic.
        {"name": "shared_chunk", "kind": "attend", "n": 4, "hq": 16, "hkv": 8, "d": 128, "layout": "contig",
         "window": 0, "prefix": 1400, "first": 700, "gap": 41, "q": 512, "cap": 0.0, "slopes": 0},
        # One row of one stream over a short cache, capped scores: the smallest attention call.
        {"name": "capped_b1", "kind": "attend", "n": 1, "hq": 8, "hkv": 1, "d": 256, "layout": "contig", "window": 0,
         "prefix": 0, "first": 512, "gap": 0, "q": 1, "cap": 50.0, "slopes": 0},
        # A text chunk of two streams with capped scores.
        {"name": "capped_chunk", "kind": "attend", "n": 2, "hq": 8, "hkv": 4, "d": 128, "layout": "contig", "window": 0,
         "prefix": 0, "first": 2000, "gap": 100, "q": 291, "cap": 30.0, "slopes": 0},
        # Sixteen paged sessions of unequal length behind a prompt, scores biased by distance.
        {"name": "biased_x16", "kind": "attend", "n": 16, "hq": 16, "hkv": 8, "d": 128, "layout": "paged", "window": 0,
         "prefix": 1024, "first": 2500, "gap": 100, "q": 1, "cap": 0.0, "slopes": 1},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number of [lo, hi], its logarithm uniform."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    if rng.random() < 0.4:
        hq, hkv, d = rng.choice([(16, 8, 128), (16, 8, 128), (8, 1, 256), (8, 1, 512), (8, 4, 128), (16, 8, 64),
                                 (12, 4, 128)])
        rows = _log(rng, 1, 8000)
        n = _log(rng, 1, min(rows, 64))
        return {"kind": "rotate", "n": n, "q": -(-rows // n), "hq": hq, "hkv": hkv, "d": d,
                "freqs": rng.choice([d // 2, d // 2, d // 4, d // 8, 24]), "axes": rng.choice([1, 1, 2, 3]),
                "order": rng.choice(["sections", "alternate"]), "adjacent": rng.choice([0, 0, 1]),
                "norm": rng.choice(["qk", "qk", "qkv", "none"]), "far": _log(rng, 8, 1000000)}
    hq, hkv, d = rng.choice([(16, 8, 128), (16, 8, 128), (8, 1, 256), (8, 1, 512), (8, 8, 128), (8, 4, 128),
                             (12, 4, 128), (16, 8, 64)])
    layout = rng.choice(["contig", "contig", "ring", "paged"])
    window = rng.choice([512, 1000]) if layout == "ring" else rng.choice([0, 0, 0, 700])
    cap, slopes = rng.choice([(0.0, 0), (0.0, 0), (0.0, 0), (30.0, 0), (50.0, 0), (0.0, 1), (20.0, 1)])
    prefix = rng.choice([0, _log(rng, 1, 5000), _log(rng, 100, 5000), _log(rng, 100, 5000)])
    if rng.random() < 0.65:  # a decode step
        n, q = _log(rng, 1, 64), rng.choice([1, 1, 1, 2])
        first = max(q, _log(rng, 1, 4000 if n <= 16 else 1400))
    else:
        n, q, prefix = rng.randint(1, 4), _log(rng, 3, 500), min(prefix, 2500)
        first = q + rng.choice([0, _log(rng, 1, 1500)])
    return {"kind": "attend", "n": n, "hq": hq, "hkv": hkv, "d": d, "layout": layout, "window": window,
            "prefix": prefix, "first": first, "gap": rng.randint(0, (first - q) // n), "q": q, "cap": cap,
            "slopes": slopes}


# ---- shapes and inputs ------------------------------------------------------------------


def _lengths(c: dict) -> list[int]:
    return [c["first"] - c["gap"] * i for i in range(c["n"])]


def _axis_of(c: dict) -> list[int]:
    """The axis whose position turns frequency f, for every f."""
    if c["order"] == "alternate":
        return [f % c["axes"] for f in range(c["freqs"])]
    return [f * c["axes"] // c["freqs"] for f in range(c["freqs"])]


def _slopes(c: dict) -> list[float]:
    return [2.0 ** (-8.0 * (h + 1) / c["hq"]) for h in range(c["hq"])]


def prepare(case: dict, seed: int) -> dict:
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    n, q, hq, hkv, d = c["n"], c["q"], c["hq"], c["hkv"], c["d"]
    s: dict = {"case": c}
    if c["kind"] == "rotate":
        # one projection of all heads; some channels larger than others, as trained ones are
        x = randn(n, q, hq + 2 * hkv, d) * torch.exp(0.5 * randn(hq + 2 * hkv, d))
        x = x.to(BF16)
        s["q"], s["k"], s["v"] = (t.transpose(1, 2) for t in x.split([hq, hkv, hkv], 2))
        s["qw"], s["kw"] = (torch.exp(0.3 * randn(d)).to(BF16) for _ in range(2))
        start = torch.randint(0, c["far"], (c["axes"], n, 1), generator=gen, device="cuda")
        s["positions"] = (start + torch.arange(q, device="cuda") // torch.tensor([1, 7, 3], device="cuda")[
            :c["axes"], None, None]).to(torch.int32)
        s["inv_freq"] = 1.0e6 ** (-torch.arange(c["freqs"], device="cuda", dtype=torch.float64) / c["freqs"])
        s["inv_freq"] = s["inv_freq"].float()
        s["axis"] = torch.tensor(_axis_of(c), device="cuda")
        if own:
            from kvrt import HeadRotation

            s["rotation"] = HeadRotation(d, s["inv_freq"], axes=_axis_of(c), adjacent=bool(c["adjacent"]),
                                         norm=c["norm"], eps=EPS,
                                         **({} if c["norm"] == "none" else {"q_weight": s["qw"], "k_weight": s["kw"]}))
        return s
    lens = _lengths(c)
    s["lengths"] = torch.tensor(lens, device="cuda")
    s["slopes"] = torch.tensor(_slopes(c), dtype=torch.float32, device="cuda") if c["slopes"] else None
    sharp = 3.0 if c["cap"] else 1.0  # scores that the cap bends
    s["q"] = (sharp * randn(n, hq, q, d)).to(BF16)
    channel = torch.exp(0.5 * randn(hkv, 1, d))
    for name, rows in (("p", c["prefix"]), ("o", c["first"])):
        items = 1 if name == "p" else n
        s[name + "k"] = (randn(items, hkv, rows, d) * channel).to(BF16)
        s[name + "v"] = randn(items, hkv, rows, d).to(BF16)
    if own:
        from kvrt import KVRuntime, LayerSpec

        top = max(c["prefix"], c["first"])
        pages = -(-c["prefix"] // PAGE) + sum(-(-x // PAGE) for x in lens)
        ring = c["window"] + q if c["layout"] == "ring" else 0
        spec = LayerSpec(kv_heads=hkv, head_dim=d, layout=c["layout"], window=c["window"], ring_rows=ring)
        rt = KVRuntime([spec], n_slots=n + 1, capacity=top + 16, max_q=min(q, 2), block_size=PAGE,
                       pool_pages=pages + 4 if c["layout"] == "paged" else 0, pool_seed=int(seed) % 10000 + 1)
        for i in range(n):
            rt.import_(i, 0, s["ok"][i:i + 1, :, :lens[i]], s["ov"][i:i + 1, :, :lens[i]])
        if c["prefix"]:
            rt.import_(n, 0, s["pk"], s["pv"])
        s["runtime"] = rt
    return s


# ---- the framework's calls ----------------------------------------------------------------


def run(s: dict):
    c = s["case"]
    if not own:
        return _plain_rotate(s) if c["kind"] == "rotate" else _plain_attend(s)
    if c["kind"] == "rotate":
        return s["rotation"].apply(s["q"], s["k"], s["v"] if c["norm"] == "qkv" else None, positions=s["positions"])
    return s["runtime"].attend_shared(0, s["q"], range(c["n"]), c["d"] ** -0.5,
                                      prefix_slot=c["n"] if c["prefix"] else None, softcap=c["cap"],
                                      slopes=s["slopes"])


# ---- plain forms ----------------------------------------------------------------------------


def _plain_rotate(s: dict):
    c = s["case"]
    f = c["freqs"]
    # angles in 64 bits: far positions times frequencies lose a radian's digits in 32
    angle = s["positions"].double()[s["axis"]].permute(1, 2, 0) * s["inv_freq"].double()  # [n, q, f]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = []
    for name, weight in (("q", s["qw"]), ("k", s["kw"]), ("v", None)):
        if name == "v" and c["norm"] != "qkv":
            out.append(None)
            continue
        x = s[name].float()
        if c["norm"] != "none":
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            if weight is not None:
                x = x * weight.float()
        if name != "v":
            turn, rest = x[..., :2 * f], x[..., 2 * f:]
            a, b = (turn[..., 0::2], turn[..., 1::2]) if c["adjacent"] else (turn[..., :f], turn[..., f:])
            a, b = a * cos - b * sin, b * cos + a * sin
            turn = torch.stack((a, b), -1).flatten(-2) if c["adjacent"] else torch.cat((a, b), -1)
            x = torch.cat((turn, rest), -1)
        out.append(x.to(BF16))
    return tuple(out)


def _plain_attend(s: dict) -> torch.Tensor:
    c = s["case"]
    n, q, hkv, g, d, p = c["n"], c["q"], c["hkv"], c["hq"] // c["hkv"], c["d"], c["prefix"]
    x = s["q"].float().view(n, hkv, g * q, d) * d ** -0.5
    pk, pv, ok, ov = (s[name].float() for name in ("pk", "pv", "ok", "ov"))
    # the prefix's products once for all sessions' rows
    every = x.transpose(0, 1).reshape(hkv, n * g * q, d)
    w = torch.cat((torch.matmul(every, pk[0].transpose(1, 2)).view(hkv, n, g * q, p).transpose(0, 1),
                   torch.matmul(x, ok.transpose(2, 3))), -1).view(n, hkv, g, q, -1)
    if c["cap"]:
        w = c["cap"] * torch.tanh(w / c["cap"])
    key = torch.arange(p + c["first"], device="cuda")
    length = p + s["lengths"][:, None, None]
    pos = length - q + torch.arange(q, device="cuda")[:, None]  # [n, q, 1]
    if s["slopes"] is not None:
        w = w + s["slopes"].view(hkv, g, 1, 1) * (key - pos).float()[:, None, None]
    seen = key <= pos
    if c["window"]:
        seen = seen & (key > pos - c["window"])
    w = w.masked_fill(~seen[:, None, None], float("-inf"))
    w = torch.exp(w - w.amax(-1, keepdim=True))
    total = w.sum(-1, keepdim=True).view(n, hkv, g * q, 1)
    w = w.view(n, hkv, g * q, -1)
    o = torch.matmul(w[..., :p].transpose(0, 1).reshape(hkv, n * g * q, p), pv[0])
    o = o.view(hkv, n, g * q, d).transpose(0, 1) + torch.matmul(w[..., p:], ov)
    return (o / total).reshape(n, hkv * g, q, d).to(BF16)


# ---- the operators' definitions in 64 bits -----------------------------------------------------


def exact(case: dict, seed: int):
    c, s = dict(case), prepare(case, seed)
    f8, n, q, hkv, d = torch.float64, c["n"], c["q"], c["hkv"], c["d"]
    g = c["hq"] // hkv
    if c["kind"] == "rotate":
        f, axis = c["freqs"], _axis_of(c)
        freq, place = s["inv_freq"].to(f8), s["positions"].to(f8)
        out: list = []
        for name, weight in (("q", s["qw"]), ("k", s["kw"]), ("v", None)):
            if name == "v" and c["norm"] != "qkv":
                out.append(None)
                continue
            y = s[name].to(f8).clone()
            if c["norm"] != "none":
                y /= torch.sqrt(y.square().sum(-1, keepdim=True) / d + EPS)
                y *= 1.0 if weight is None else weight.to(f8)
            if name != "v":
                z = y.clone()
                for i in range(f):  # one pair of dims after the other
                    one, two = (2 * i, 2 * i + 1) if c["adjacent"] else (i, i + f)
                    turn = (place[axis[i]] * freq[i])[:, None]
                    z[..., one] = y[..., one] * torch.cos(turn) - y[..., two] * torch.sin(turn)
                    z[..., two] = y[..., one] * torch.sin(turn) + y[..., two] * torch.cos(turn)
                y = z
            out.append(y)
        return tuple(out)
    res = torch.empty((n, c["hq"], q, d), dtype=f8, device="cuda")
    for i, length in enumerate(_lengths(c)):
        at = torch.arange(c["prefix"] + length, device="cuda")
        mine = at[-q:, None]
        hide = at > mine
        if c["window"]:
            hide |= mine - at >= c["window"]
        for h in range(hkv):
            k, v = (torch.cat((s["p" + a][0, h], s["o" + a][i, h, :length])).to(f8) for a in "kv")
            w = s["q"][i, h * g:(h + 1) * g].to(f8) @ k.T / math.sqrt(d)  # [g, q, keys]
            if c["cap"]:
                w = torch.tanh(w / c["cap"]) * c["cap"]
            if c["slopes"]:
                # slopes as the 32-bit numbers that the call is given
                w -= s["slopes"][h * g:(h + 1) * g, None, None].to(f8) * (mine - at)
            res[i, h * g:(h + 1) * g] = torch.softmax(w.masked_fill(hide, float("-inf")), -1) @ v
    return res


def work(case: dict) -> dict:
    c = dict(case)
    n, q, hq, hkv, d = c["n"], c["q"], c["hq"], c["hkv"], c["d"]
    if c["kind"] == "rotate":
        heads = hq + hkv + (hkv if c["norm"] == "qkv" else 0)
        elements = n * q * heads * d
        return {"bytes": 4.0 * elements + 4.0 * c["axes"] * n * q + 4.0 * d + 8.0 * c["freqs"], "flops": 10.0 * elements}
    p, w = c["prefix"], c["window"]
    keys, pairs, low = 0, 0, p
    for length in _lengths(c):
        at = range(p + length - q, p + length)
        pairs += sum(min(x + 1, w) if w else x + 1 for x in at)
        lo = max(0, at[0] - w + 1) if w else 0
        low = min(low, lo)
        keys += p + length - max(lo, p)
    data = 4.0 * (keys + p - low) * hkv * d + 4.0 * n * q * hq * d
    return {"bytes": data, "flops": 4.0 * d * hq * pairs}
