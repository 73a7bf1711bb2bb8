"""Measured passes over a paged KV cache held in 8 bits, one scale a page and KV head.

``prepare`` builds what a serving program keeps (page tables, a pool of coded
pages) and a step's inputs; ``run`` makes one pass and returns all it computed.

Kinds:

* ``tables``  a step's page tables and slot map from request lengths: the rows of
  the turn before are rolled back, then pages for the new rows are mapped;
* ``listen``  new rows coded into their pages, then read back as the zero-padded
  bf16 batch (with its mask) that attention over tensors takes;
* ``attend``  attention of each request's newest rows over its coded pages.

Lengths are ``first - gap * i`` for request i; new rows ``max(1, q - qgap * i)``,
or, with ``every`` > 1, ``q`` for each ``every``-th request and one for the rest.
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
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}  # largest code
LOW, HIGH = 2.0 ** -64, 2.0 ** 32  # range of a scale


def listed() -> list[dict]:
    return [
        # The page tables of a talker step: four sessions, two rows each.
        {"name": "tables_x4", "kind": "tables", "n": 4, "block": 16, "pages": 320, "first": 4159, "gap": 37, "q": 2,
         "qgap": 0, "every": 1, "spare": 0},
        # A serving step over 256 requests: a chunk of 512 rows for every eighth, one row for the others.
        {"name": "tables_serve", "kind": "tables", "n": 256, "block": 16, "pages": 576, "first": 8100, "gap": 30,
         "q": 512, "qgap": 0, "every": 8, "spare": 3872},
        # The listener's frame: two rows of four ragged streams, then the padded batch.
        {"name": "listen_x4", "kind": "listen", "n": 4, "hkv": 1, "d": 256, "code": "int8", "block": 16, "first": 610,
         "gap": 92, "q": 2, "qgap": 0, "every": 1, "pad": 640, "back": 0},
        # Sixteen talker sessions opened with prefixes of 512 rows and fewer: all new rows coded and read back.
        {"name": "open_x16", "kind": "listen", "n": 16, "hkv": 8, "d": 128, "code": "e4m3", "block": 16, "first": 60,
         "gap": 3, "q": 512, "qgap": 11, "every": 1, "pad": 512, "back": 1},
        # One row of one stream over a short cache: the smallest attention call.
        {"name": "decode_b1", "kind": "attend", "n": 1, "hq": 8, "hkv": 1, "d": 256, "code": "int8", "block": 16,
         "first": 512, "gap": 0, "q": 1, "qgap": 0, "every": 1, "window": 0},
        # A talker frame of four sessions at about 4096 positions, one layer.
        {"name": "decode_talker_x4", "kind": "attend", "n": 4, "hq": 16, "hkv": 8, "d": 128, "code": "int8",
         "block": 16, "first": 4159, "gap": 37, "q": 1, "qgap": 0, "every": 1, "window": 0},
        # Two queries of a full layer over long sessions of four streams (head_dim 512).
        {"name": "decode_full_q2", "kind": "attend", "n": 4, "hq": 8, "hkv": 1, "d": 512, "code": "e4m3", "block": 32,
         "first": 8192, "gap": 0, "q": 2, "qgap": 0, "every": 1, "window": 0},
        # Sixty-four sessions of unequal length served from one pool: the largest read of a cache.
        {"name": "decode_serve_x64", "kind": "attend", "n": 64, "hq": 16, "hkv": 8, "d": 128, "code": "e4m3",
         "block": 16, "first": 8100, "gap": 110, "q": 1, "qgap": 0, "every": 1, "window": 0},
        # A text chunk into one session.
        {"name": "chunk_q34", "kind": "attend", "n": 1, "hq": 8, "hkv": 8, "d": 128, "code": "int8", "block": 16,
         "first": 2666, "gap": 0, "q": 34, "qgap": 0, "every": 1, "window": 0},
        # A text chunk into a sliding layer of four streams.
        {"name": "chunk_sliding", "kind": "attend", "n": 4, "hq": 8, "hkv": 1, "d": 256, "code": "e4m3", "block": 16,
         "first": 2339, "gap": 0, "q": 291, "qgap": 0, "every": 1, "window": 512},
        # The talker's prefixes prefilled for four sessions of unequal length.
        {"name": "chunk_talker", "kind": "attend", "n": 4, "hq": 16, "hkv": 8, "d": 128, "code": "int8", "block": 16,
         "first": 1400, "gap": 41, "q": 512, "qgap": 37, "every": 1, "window": 0},
        # A long chunk into a full layer of four streams: the most arithmetic.
        {"name": "chunk_full", "kind": "attend", "n": 4, "hq": 8, "hkv": 1, "d": 512, "code": "int8", "block": 16,
         "first": 4096, "gap": 0, "q": 2048, "qgap": 0, "every": 1, "window": 0},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number of [lo, hi], its logarithm uniform."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["tables", "tables", "listen", "listen", "attend", "attend", "attend", "attend", "attend"])
    block = rng.choice([16, 16, 32, 64])
    if kind == "tables":
        n, first = _log(rng, 1, 256), _log(rng, 1, 8000)
        q, every = _log(rng, 1, 600), rng.choice([1, 4, 8])
        if n * q > 20000:
            every = 8
        return {"kind": kind, "n": n, "block": block, "pages": -(-(first + q) // block) + rng.randint(0, 40),
                "first": first, "gap": rng.randint(0, first // n), "q": q, "qgap": rng.randint(0, max(1, q // n)),
                "every": every, "spare": rng.choice([0, rng.randint(1, 500)])}
    code = rng.choice(["int8", "e4m3"])
    if kind == "listen":
        hkv, d = rng.choice([(1, 256), (1, 512), (8, 128), (4, 128), (2, 64)])
        n, first, q = _log(rng, 1, 16), _log(rng, 1, 1500), _log(rng, 1, 500)
        back = rng.choice([0, 1])
        return {"kind": kind, "n": n, "hkv": hkv, "d": d, "code": code, "block": block, "first": first,
                "gap": rng.randint(0, first // n), "q": q, "qgap": rng.randint(0, q // n), "every": 1,
                "pad": (q if back else first + q) + rng.randint(0, 100), "back": back}
    hq, hkv, d = rng.choice([(16, 8, 128), (16, 8, 128), (8, 1, 256), (8, 1, 512), (8, 8, 128), (8, 4, 128),
                             (12, 4, 128), (16, 8, 64)])
    window = rng.choice([0, 0, 0, 512, 1000])
    if rng.random() < 0.5:  # a decode step
        n = _log(rng, 1, 64)
        first = _log(rng, 1, 8100 if n <= 32 else 4000)
        q = rng.choice([1, 1, 1, 2]) if first > 1 else 1
        gap = rng.randint(0, (first - q) // n)
        qgap, every = 0, 1
    else:
        n, q = rng.randint(1, 6), _log(rng, 3, 1200)
        first = q + rng.choice([0, _log(rng, 16, 3000)])
        gap = rng.randint(0, (first - q) // n)
        qgap, every = rng.randint(0, q // n), rng.choice([1, 1, 2])
    return {"kind": "attend", "n": n, "hq": hq, "hkv": hkv, "d": d, "code": code, "block": block, "first": first,
            "gap": gap, "q": q, "qgap": qgap, "every": every, "window": window}


# ---- shapes and inputs ------------------------------------------------------------------


def _lengths(c: dict) -> list[int]:
    return [c["first"] - c["gap"] * i for i in range(c["n"])]


def _news(c: dict) -> list[int]:
    if c["every"] > 1:
        return [c["q"] if i % c["every"] == 0 else 1 for i in range(c["n"])]
    return [max(1, c["q"] - c["qgap"] * i) for i in range(c["n"])]


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(news: list[int]) -> torch.Tensor:
    s = [0]
    for x in news:
        s.append(s[-1] + x)
    return _i32(s)


def _to_codes(x: torch.Tensor, code: str) -> torch.Tensor:
    """x (fp32, in units of the scale) rounded to codes."""
    x = x.clamp(-TOP[code], TOP[code])
    return x.round().to(torch.int8) if code == "int8" else x.to(torch.float8_e4m3fn)


def _tables_of(counts: list[int], width: int, gen, pool: int) -> torch.Tensor:
    """[n, width] page ids: request i's first counts[i] entries, pages in shuffled order; -1 after."""
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    per = _i32(counts)
    j = torch.arange(width, device="cuda", dtype=torch.int32)
    live = j[None, :] < per[:, None]
    rank = (live.reshape(-1).cumsum(0) - 1).reshape(live.shape).clamp(min=0)
    return torch.where(live, order[rank], torch.full_like(rank, -1, dtype=torch.int32)), order


def _pool(gen, pool: int, c: dict) -> list[torch.Tensor]:
    """Coded pages of K and V as a serving run leaves them, and their scales."""
    shape = (pool, c["hkv"], c["block"], c["d"])
    out = []
    for is_k in (True, False):
        x = torch.randn(shape, generator=gen, device="cuda")
        if is_k:  # keys have channels larger than others
            x *= torch.exp(0.5 * torch.randn((1, c["hkv"], 1, c["d"]), generator=gen, device="cuda"))
        else:
            x *= torch.exp(0.3 * torch.randn((pool, c["hkv"], 1, 1), generator=gen, device="cuda"))
        scale = (x.abs().amax((2, 3)) / TOP[c["code"]]).clamp(LOW, HIGH)
        out += [_to_codes(x / scale[:, :, None, None], c["code"]), scale]
    return out


def prepare(case: dict, seed: int) -> dict:
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    lens, news, b = _lengths(c), _news(c), c["block"]
    s: dict = {"case": c, "starts": _starts(news)}
    if c["kind"] == "tables":
        pool = sum(-(-(x + y) // b) for x, y in zip(lens, news)) + 64
        counts = [-(-x // b) for x in lens]
        s["table"], order = _tables_of(counts, c["pages"], gen, pool)
        s["mapped"] = _i32(counts)
        s["free"] = torch.cat([order[sum(counts):], order[:sum(counts)]]).contiguous()
        s["free_count"] = _i32([pool - sum(counts)])
        s["lengths"], s["new"] = _i32(lens), _i32(news)
        s["none"] = torch.zeros_like(s["new"])
        s["rows"] = sum(news) + c["spare"]
        if own:
            from kvrt import BlockTables

            t = BlockTables(c["n"], c["pages"], pool, block_size=b, device="cuda")
            for name in ("table", "mapped", "free", "free_count"):
                getattr(t, name).copy_(s[name])
            s["tables"] = t
        return s
    full = [x + y for x, y in zip(lens, news)] if c["kind"] == "listen" else lens
    pages = [-(-x // b) for x in full]
    pool = sum(pages) + 3
    s["table"], _ = _tables_of(pages, max(pages), gen, pool)
    s["lengths"] = _i32(full)
    s["k"], s["k_scale"], s["v"], s["v_scale"] = _pool(gen, pool, c)
    rows = sum(news)
    if c["kind"] == "listen":
        seq = torch.repeat_interleave(torch.arange(c["n"], device="cuda"), _i32(news).long())
        pos = _i32(lens).long()[seq] + torch.arange(rows, device="cuda") - s["starts"].long()[seq]
        s["slot_map"] = (s["table"].long()[seq, pos // b] * b + pos % b).to(torch.int32)
        s["from"] = _i32(lens) if c["back"] else torch.zeros_like(s["lengths"])
        shape = (rows, c["hkv"], c["d"])
        s["new_k"] = (torch.randn(shape, generator=gen, device="cuda") * 1.2).to(BF16)
        s["new_v"] = torch.randn(shape, generator=gen, device="cuda").to(BF16)
    else:
        s["q"] = torch.randn((rows, c["hq"], c["d"]), generator=gen, device="cuda").to(BF16)
        s["max_q"] = max(news)
    if own:
        from kvrt import Block8Pool

        s["pool"] = Block8Pool(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


# ---- the framework's calls ----------------------------------------------------------------


def run(s: dict):
    c = s["case"]
    if not own:
        return {"tables": _plain_tables, "listen": _plain_listen, "attend": _plain_attend}[c["kind"]](s)
    if c["kind"] == "tables":
        t = s["tables"]
        t.update(s["lengths"], s["none"], rows=0)
        p = t.update(s["lengths"], s["new"], rows=s["rows"])
        return {"table": t.table, "mapped": t.mapped, "free": t.free, "free_count": t.free_count, "starts": p.starts,
                "slot_map": p.slot_map, "lengths": p.lengths, "granted": p.granted}
    pool = s["pool"]
    if c["kind"] == "listen":
        pool.append(s["new_k"], s["new_v"], s["slot_map"])
        k, v, mask = pool.gather(s["table"], s["lengths"], c["pad"], start_pos=s["from"])
        return {"k": k, "v": v, "mask": mask, "k_scale": pool.k_scale, "v_scale": pool.v_scale}
    return pool.attend(s["q"], s["table"], s["lengths"], s["starts"], c["d"] ** -0.5, max_q=s["max_q"],
                       window=c["window"])


# ---- plain forms ----------------------------------------------------------------------------


def _plain_update(s: dict, new: torch.Tensor, rows: int) -> dict:
    """Tables after keeping ``lengths`` rows of each request and adding ``new``."""
    b, dev = s["case"]["block"], "cuda"
    lens, add, mapped = s["lengths"].long(), new.long(), s["mapped"].long()
    width, pool = s["table"].shape[1], s["free"].numel()
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), add.cumsum(0)])
    need = (lens + add + b - 1) // b
    fits = (lens >= 0) & (add >= 0) & (need <= width) & (lens <= mapped * b) & (starts[1:] <= rows)
    gone = torch.where(fits, (mapped - need).clamp(min=0), torch.zeros_like(need))
    want = torch.where(fits, (need - mapped).clamp(min=0), torch.zeros_like(need))
    top = s["free_count"].long() + gone.sum()
    ok = fits & ((want == 0) | (want.cumsum(0) <= top))
    want = torch.where(ok, want, torch.zeros_like(want))
    now = torch.where(ok, need, mapped)
    j = torch.arange(width, device=dev)[None, :]
    lost = (j >= now[:, None]) & (j < mapped[:, None])
    got = (j >= mapped[:, None]) & (j < now[:, None])
    # the k-th released page goes to free[top - 1 - k]; the k-th new one comes from there
    at = torch.where(lost, top - 1 - (lost.reshape(-1).cumsum(0) - 1).reshape(lost.shape), pool)
    free = torch.cat([s["free"], s["free"][:1]]).scatter(0, at.reshape(-1), s["table"].reshape(-1))[:pool]
    at = (top - 1 - (got.reshape(-1).cumsum(0) - 1).reshape(got.shape)).clamp(0, pool - 1)
    table = torch.where(got, free[at], s["table"])
    table = torch.where(lost, torch.full_like(table, -1), table)
    s["table"].copy_(table)
    s["mapped"].copy_(now)
    s["free"].copy_(free)
    s["free_count"].copy_(top - want.sum())
    granted = torch.where(ok, add, torch.zeros_like(add))
    t = torch.arange(rows, device=dev)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=lens.numel() - 1)
    pos = lens[seq] + t - starts[seq]
    live = (t < starts[-1]) & ok[seq]
    page = table[seq, (pos // b).clamp(0, width - 1)].long()
    slot = torch.where(live, page * b + pos % b, torch.full_like(pos, -1))
    i32 = torch.int32
    return {"table": s["table"], "mapped": s["mapped"], "free": s["free"], "free_count": s["free_count"],
            "starts": starts.clamp(max=rows).to(i32), "slot_map": slot.to(i32), "lengths": (lens + granted).to(i32),
            "granted": granted.to(i32)}


def _plain_tables(s: dict) -> dict:
    _plain_update(s, s["none"], 0)
    return _plain_update(s, s["new"], s["rows"])


def _plain_append(codes: torch.Tensor, scale: torch.Tensor, x: torch.Tensor, slots: torch.Tensor, code: str) -> None:
    """Rows x [T, H, D] into the pages of their slots, in place. A page's scale grows with
    its new rows, and the rows before them are coded anew; a page begun at its first row
    takes the new rows' scale."""
    b = codes.shape[2]
    page, off = (slots // b).long(), (slots % b).long()
    x = x.float()
    new = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(2), "amax")
    new = (new / TOP[code]).clamp(LOW, HIGH)
    first = torch.full((scale.shape[0],), b, device=x.device).index_reduce_(0, page, off, "amin")
    after = torch.where((first > 0)[:, None], torch.maximum(scale, new), new)
    touched = page[torch.cat([page[:1] * 0 == 0, page[1:] != page[:-1]])]
    old = codes[touched].float() * (scale[touched] / after[touched])[:, :, None, None]
    keep = (torch.arange(b, device=x.device)[None, :] < first[touched][:, None])[:, None, :, None]
    codes[touched] = torch.where(keep, _to_codes(old, code).float(), codes[touched].float()).to(codes.dtype)
    codes[page, :, off] = _to_codes(x * (1.0 / after[page])[:, :, None], code)
    scale[touched] = after[touched]


def _plain_rows(codes: torch.Tensor, scale: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """fp32 rows [n, H, pages * block, D] of the tables' pages (page 0's where unmapped)."""
    t = table.clamp(min=0).long()
    x = codes[t].float() * scale[t][..., None, None]
    n, p, h, b, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(n, h, p * b, d)


def _plain_listen(s: dict) -> dict:
    c = s["case"]
    out: dict = {}
    j = s["from"][:, None].long() + torch.arange(c["pad"], device="cuda")[None, :]
    mask = j < s["lengths"][:, None]
    for name in ("k", "v"):
        _plain_append(s[name], s[name + "_scale"], s["new_" + name], s["slot_map"], c["code"])
        x = _plain_rows(s[name], s[name + "_scale"], s["table"])
        at = j.clamp(max=x.shape[2] - 1)[:, None, :, None].expand(-1, x.shape[1], -1, x.shape[3])
        out[name] = (x.gather(2, at) * mask[:, None, :, None]).to(BF16)
    return {**out, "mask": mask, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _plain_attend(s: dict) -> torch.Tensor:
    c, q, starts = s["case"], s["q"], s["starts"].long()
    n, hkv, g, d, most = c["n"], c["hkv"], c["hq"] // c["hkv"], c["d"], s["max_q"]
    lens = s["lengths"].long()
    count = starts[1:] - starts[:-1]
    r = torch.arange(most, device="cuda")
    at = (starts[:-1, None] + r).clamp(max=q.shape[0] - 1)  # [n, most]
    x = q[at].float().reshape(n, most, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, g * most, d)
    k, v = (_plain_rows(s[a], s[a + "_scale"], s["table"]) for a in ("k", "v"))
    pos = (lens - count)[:, None] + r  # [n, most]
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key[None, None, :] <= pos[:, :, None]) & (key[None, None, :] < lens[:, None, None])
    if c["window"]:
        seen &= key[None, None, :] > pos[:, :, None] - c["window"]
    w = torch.matmul(x, k.transpose(2, 3)).mul_(d ** -0.5).view(n, hkv, g, most, -1)
    w.masked_fill_(~seen[:, None, None], float("-inf"))
    top = w.amax(-1, keepdim=True)
    w.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(n, hkv, g * most, -1), v).view(n, hkv, g, most, d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(n * most, hkv * g, d).to(BF16)
    # row starts[i] + r of the answer is row i * most + r here
    row = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return o[seq * most + row - starts[seq]]


# ---- the operators' definitions in 64 bits -----------------------------------------------------


def _exact_codes(x: torch.Tensor, code: str) -> torch.Tensor:
    """The code nearest to each x, ties to the even one, as float64 values."""
    if code == "int8":
        return torch.round(x).clamp(-127, 127)
    x = x.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case: dict, seed: int):
    if case["kind"] == "tables":
        return None  # whole numbers
    c, s = dict(case), prepare(case, seed)
    f8, b, dev = torch.float64, c["block"], "cuda"
    lens, news = s["lengths"].tolist(), _news(c)
    if c["kind"] == "attend":
        g, d, at, outs = c["hq"] // c["hkv"], c["d"], 0, []
        for i, (length, m) in enumerate(zip(lens, news)):
            pages = s["table"][i, :-(-length // b)].long()
            q = s["q"][at:at + m].to(f8)
            at += m
            pos = torch.arange(length - m, length, device=dev)
            key = torch.arange(length, device=dev)
            hide = key[None, :] > pos[:, None]
            if c["window"]:
                hide |= key[None, :] <= pos[:, None] - c["window"]
            heads = []
            for h in range(c["hkv"]):
                kv = [(s[a][pages, h].to(torch.float32).to(f8) * s[a + "_scale"][pages, h].to(f8)[:, None, None])
                      .reshape(-1, d)[:length] for a in ("k", "v")]
                for e in range(g):
                    w = (q[:, h * g + e] @ kv[0].T) * d ** -0.5
                    heads.append(torch.softmax(w.masked_fill(hide, float("-inf")), 1) @ kv[1])
            outs.append(torch.stack(heads, 1))
        return torch.cat(outs)
    out: dict = {}
    for a in ("k", "v"):
        val = s[a].to(torch.float32).to(f8)
        scale = s[a + "_scale"].to(f8).clone()
        at, x = 0, s["new_" + a].to(f8)
        rows = torch.zeros((c["n"], c["hkv"], c["pad"], c["d"]), dtype=f8, device=dev)
        for i, (length, m) in enumerate(zip(lens, news)):
            pages = s["table"][i, :-(-length // b)].long()
            first = length - m
            # this request's touched pages, rows outside [first, length) of them as zeros
            p0, p1 = first // b, -(-length // b)
            some = torch.zeros(((p1 - p0) * b, c["hkv"], c["d"]), dtype=f8, device=dev)
            some[first - p0 * b:length - p0 * b] = x[at:at + m]
            at += m
            some = some.reshape(p1 - p0, b, c["hkv"], c["d"]).transpose(1, 2)
            pg = pages[p0:p1]
            new = (some.abs().amax((2, 3)) / TOP[c["code"]]).clamp(LOW, HIGH)
            was = scale[pg].clone()
            if first % b:
                new[0] = torch.maximum(new[0], was[0])
                val[pg[0], :, :first % b] = _exact_codes(val[pg[0], :, :first % b] * (was[0] / new[0])[:, None, None],
                                                         c["code"])
            scale[pg] = new
            fresh = _exact_codes(some / new[:, :, None, None], c["code"])
            p = torch.arange(p0 * b, p1 * b, device=dev).reshape(p1 - p0, 1, b, 1)
            val[pg] = torch.where((p >= first) & (p < length), fresh, val[pg])
            whole = (val[pages] * scale[pages][:, :, None, None]).transpose(0, 1).reshape(c["hkv"], -1, c["d"])
            lo = first if c["back"] else 0
            rows[i, :, :length - lo] = whole[:, lo:length]
        out[a], out[a + "_scale"] = rows, scale
    return {"k": out["k"], "v": out["v"], "mask": None, "k_scale": out["k_scale"], "v_scale": out["v_scale"]}


def work(case: dict) -> dict:
    c = dict(case)
    lens, news, b = _lengths(c), _news(c), c["block"]
    if c["kind"] == "tables":
        moved = sum(-(-(x + y) // b) - -(-x // b) for x, y in zip(lens, news))
        # lengths, new, mapped in and out, starts, granted; each new page's id out of the list, into the table and
        # back; the slot map
        return {"bytes": 4.0 * (9 * c["n"] + 4 * moved + sum(news) + c["spare"]), "flops": 0}
    if c["kind"] == "listen":
        width, rows = c["hkv"] * c["d"], sum(news)
        read = sum(y if c["back"] else x for x, y in zip(lens, news))  # stored rows that only the batch reads
        touched = sum(-(-(x + y) // b) - x // b for x, y in zip(lens, news))
        data = 2 * (2 * rows * width + rows * width + (read if not c["back"] else 0) * width
                    + 2 * c["n"] * c["pad"] * width)
        return {"bytes": float(data + 4 * rows + c["n"] * c["pad"] + 16 * touched * c["hkv"]), "flops": 0}
    hq, hkv, d, w = c["hq"], c["hkv"], c["d"], c["window"]
    keys = pairs = 0
    for length, m in zip(lens, news):
        lo = max(0, length - m - w + 1) if w else 0
        keys += length - lo
        if w:
            pairs += sum(min(p + 1, w) for p in range(length - m, length))
        else:
            pairs += m * (length - m) + m * (m + 1) // 2
    data = 2 * keys * hkv * d + 8 * (keys // b + c["n"]) * hkv + 4 * sum(news) * hq * d
    return {"bytes": float(data), "flops": 4.0 * d * hq * pairs}
