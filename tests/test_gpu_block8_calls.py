"""The native calls of 8-bit pages against the general path: the same answers and
the same refusals for every form of argument either takes; and what the Python
layer refuses."""
from __future__ import annotations

import pytest
import torch

from tests.helpers import randn_bf16

pytestmark = pytest.mark.gpu


class _General:
    """Stands in for the native module: every call takes the general path."""

    def __getattr__(self, name):
        return lambda *a: 1


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _outcome(fn):
    try:
        r = fn()
        return [t for t in (r if isinstance(r, tuple) else (r,)) if t is not None]
    except Exception as e:  # noqa: BLE001 - the refusal itself is compared
        return (type(e), str(e))


def _both(make, call):
    """Outcomes of call(objects) on the native and on the general path."""
    got = []
    for general in (False, True):
        objs = make()
        if general:
            for o in objs:
                o._call = _General()
        got.append(_outcome(lambda: call(*objs)))
    return got


def _same(a, b):
    if isinstance(a, tuple) or isinstance(b, tuple):
        assert a == b
        return
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)


def _make():
    from kvrt import Block8Pool, BlockTables

    t = BlockTables(2, 5, 12)
    p = Block8Pool.zeros(12, 2, 64, dtype="e4m3")
    plan = t.update(_i32([0, 0]), _i32([20, 9]), rows=29)
    gen = torch.Generator().manual_seed(1)
    x = randn_bf16(gen, (29, 2, 64)).cuda()
    p.append(x, x * 2, plan.slot_map)
    return t, p


Q = lambda: randn_bf16(torch.Generator().manual_seed(2), (4, 6, 64)).cuda()  # noqa: E731

UPDATES = {
    "plain": {}, "int64 lengths": {"lengths": "int64"}, "cpu new": {"new": torch.tensor([1, 1], dtype=torch.int32)},
    "too few": {"new": [1]}, "strided": {"lengths": "strided"}, "negative rows": {"rows": -1}, "no rows": {"rows": 0, "new": [0, 0]},
    "table": {"table": True}, "list": {"new": "list"},
}


@pytest.mark.parametrize("form", list(UPDATES))
def test_update(form):
    kw = dict(UPDATES[form])

    def call(t, p):
        lengths, new = kw.get("lengths", [20, 9]), kw.get("new", [1, 2])
        forms = {"strided": lambda: _i32([20, 0, 9, 0])[::2], "int64": lambda: _i32([20, 9]).long()}
        lengths = forms[lengths]() if isinstance(lengths, str) else _i32(lengths)
        new = [1, 2] if isinstance(new, str) else new if torch.is_tensor(new) else _i32(new)
        if kw.get("table"):
            t.table = t.table.long()
        return (*t.update(lengths, new, rows=kw.get("rows", 3)), t.table, t.free, t.mapped)

    _same(*_both(_make, call))


APPENDS = {
    "plain": {}, "strided": {"k": lambda k: k.transpose(0, 1).contiguous().transpose(0, 1)}, "fp32": {"k": lambda k: k.float()},
    "cpu": {"k": lambda k: k.cpu()}, "heads": {"k": lambda k: k[:, :1]}, "rows": {"k": lambda k: k[:2]}, "odd": {"k": lambda k: k[..., 1:]},
    "slots": {"slots": lambda s: s.long()}, "few slots": {"slots": lambda s: s[:2]}, "parameter": {"k": lambda k: torch.nn.Parameter(k)},
    "4 dims": {"k": lambda k: k[None]},
}


@pytest.mark.parametrize("form", list(APPENDS))
def test_append(form):
    kw = APPENDS[form]

    def call(t, p):
        k = randn_bf16(torch.Generator().manual_seed(3), (3, 2, 64)).cuda()
        slots = t.update(_i32([20, 9]), _i32([1, 2]), rows=3).slot_map
        p.append(kw.get("k", lambda x: x)(k), k * 3, kw.get("slots", lambda x: x)(slots))
        return p.k.view(torch.int8), p.v.view(torch.int8), p.k_scale, p.v_scale

    _same(*_both(_make, call))


GATHERS = {
    "plain": {}, "fp32": {"dtype": torch.float32}, "fp16": {"dtype": torch.float16}, "no mask": {"mask_dtype": None},
    "fp32 mask": {"mask_dtype": torch.float32}, "int mask": {"mask_dtype": torch.int32}, "start": {"start_pos": [3, 0]},
    "no lmax": {"lmax": None}, "negative": {"lmax": -2}, "empty": {"lmax": 0}, "out": {"out": 2}, "out mask": {"out": 3},
    "out lmax": {"out": 2, "lmax": 7}, "int64": {"lengths": torch.int64}, "table": {"table": torch.int64},
}


@pytest.mark.parametrize("form", list(GATHERS))
def test_gather(form):
    kw = dict(GATHERS[form])

    def call(t, p):
        args = dict(kw)
        table, lengths = t.table.to(args.pop("table", torch.int32)), _i32([20, 9]).to(args.pop("lengths", torch.int32))
        lmax = args.pop("lmax", 22)
        if "start_pos" in args:
            args["start_pos"] = _i32(args["start_pos"])
        if "out" in args:
            n = args["out"]
            out = [torch.zeros((2, 2, 22, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
            args["out"] = tuple(out + [torch.zeros((2, 22), dtype=torch.bool, device="cuda")] * (n - 2))
            lmax = kw.get("lmax")
        return p.gather(table, lengths, lmax, **args)

    _same(*_both(_make, call))


ATTENDS = {
    "plain": {}, "int scale": {"scale": 1}, "nan": {"scale": float("nan")}, "window": {"window": 5}, "negative window": {"window": -1},
    "granted": {"granted": [1, 2]}, "long granted": {"granted": [1, 2, 3]}, "max_q": {"max_q": 2}, "large max_q": {"max_q": 10 ** 6},
    "negative max_q": {"max_q": -1}, "no max_q": {"max_q": 0}, "fp32": {"q": lambda q: q.float()}, "heads": {"q": lambda q: q[:, :3]},
    "cpu": {"q": lambda q: q.cpu()}, "4 dims": {"q": lambda q: q[None]}, "strided": {"q": lambda q: q.transpose(0, 1).contiguous().transpose(0, 1)},
    "out": {"out": lambda q: torch.zeros_like(q)}, "short out": {"out": lambda q: torch.zeros_like(q)[:2]},
    "parameter": {"q": lambda q: torch.nn.Parameter(q, requires_grad=False)}, "grad": {"q": lambda q: q.requires_grad_()},
    "starts": {"starts": [0, 1]}, "no rows": {"q": lambda q: q[:0], "starts": [0, 0, 0]},
}


@pytest.mark.parametrize("form", list(ATTENDS))
def test_attend(form):
    kw = ATTENDS[form]

    def call(t, p):
        q = kw.get("q", lambda x: x)(Q())
        granted = kw.get("granted")
        out = kw["out"](q) if "out" in kw else None
        got = p.attend(q, t.table, _i32([20, 9]), _i32(kw.get("starts", [0, 1, 4])), kw.get("scale", 0.125),
                       max_q=kw.get("max_q", 3), window=kw.get("window", 0), granted=None if granted is None else _i32(granted), out=out)
        assert out is None or got is out
        # rows that no request was granted, or past max_q, are nobody's: a new tensor's are undefined
        rows = 0 if kw.get("max_q") == 0 else 3 if granted or kw.get("max_q") == 2 else got.shape[0]
        return got[:rows]

    _same(*_both(_make, call))


def test_pools_are_checked():
    from kvrt import Block8Pool

    codes = torch.zeros((4, 2, 16, 64), dtype=torch.int8, device="cuda")
    scale = torch.zeros((4, 2), device="cuda")
    Block8Pool(codes, codes.clone(), scale, scale.clone())
    for bad in ((codes.float(), codes, scale, scale), (codes[0], codes, scale, scale), (codes, codes[:3], scale, scale),
                (codes, codes.view(torch.float8_e4m3fn), scale, scale), (codes, codes, scale[:3], scale), (codes, codes, scale.double(), scale),
                (codes[:, :, :8].contiguous(), codes, scale, scale), (codes[..., :32].contiguous(), codes, scale, scale),
                (codes, codes.cpu(), scale, scale), (codes.transpose(0, 1), codes, scale, scale)):
        with pytest.raises(ValueError):
            Block8Pool(*bad)
