"""Head rotation without a GPU: the struct's layout against the header, the table of
turns against whole-number arithmetic, and every refusal that is made before anything is
launched. Pointers here are host memory that no call reads."""
from __future__ import annotations

import ctypes
import json
import math
import shutil
import subprocess
from fractions import Fraction
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


def _lib():
    from kvrt import _lib as L

    if not L.LIB_PATH.exists():
        pytest.fail("libkvrt.so is not built; run __graft_entry__.build() first")
    return L, L.load()


FIELDS = ("turns", "axis", "q_weight", "k_weight", "head_dim", "n_freq", "adjacent", "norm", "n_axes", "eps", "scaling",
          "reserved")


def test_struct_matches_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    L, lib = _lib()
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    body = "".join(f'printf("\\"{f}\\": [%zu, %zu],", offsetof(kvrt_rotation, {f}), sizeof(((kvrt_rotation *)0)->{f}));'
                   for f in FIELDS)
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "kvrt.h"\nint main(void) { printf("{");' + body +
                   'printf("\\"size\\": %zu}", sizeof(kvrt_rotation)); return 0; }')
    subprocess.run([gcc, "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = json.loads(subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout)
    assert got.pop("size") == ctypes.sizeof(L.KvrtRotation)
    for f, where in got.items():
        d = getattr(L.KvrtRotation, f)
        assert [d.offset, d.size] == where, f
    assert [f for f, _ in L.KvrtRotation._fields_] == list(FIELDS)
    assert lib.kvrt_capabilities() & L.CAP_ROTATE_HEADS


# 2 pi to 80 digits
TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211707")


def test_turns_are_the_fraction_of_a_turn():
    L, lib = _lib()
    freqs = [1.0, 0.5, 1e-6, 3e-8, 7.0, 100.25, -0.25, -9.0, 0.0, float(torch.tensor(1e6) ** -0.37), 6.283185307179586]
    out = (ctypes.c_uint64 * len(freqs))()
    assert lib.kvrt_rotation_turns((ctypes.c_double * len(freqs))(*freqs), len(freqs), out) == 0
    for f, got in zip(freqs, out):
        want = Fraction(f) / TWO_PI
        want = (want - math.floor(want)) * 2 ** 64
        # 64 bits of mantissa in the division and its reduction: 2^-64 of the whole turns too
        off = abs(Fraction(got) - want)
        off = min(off, 2 ** 64 - off)
        assert off <= 4 * max(1.0, abs(f)), f
    assert lib.kvrt_rotation_turns(None, 0, None) == 0
    assert lib.kvrt_rotation_turns(None, 1, out) == L.KVRT_EINVAL
    assert lib.kvrt_rotation_turns((ctypes.c_double * 1)(1.0), -1, out) == L.KVRT_EINVAL
    for bad in (math.inf, -math.inf, math.nan):
        assert lib.kvrt_rotation_turns((ctypes.c_double * 2)(1.0, bad), 2, out) == L.KVRT_EINVAL


HERE = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(HERE) + 255) & ~255


def _tensor(L, dtype, dims, strides=None, data=AT):
    t = L.KvrtTensor()
    t.data, t.dtype, t.ndim = data, dtype, len(dims)
    if strides is None:
        strides, s = [], 1
        for d in reversed(dims):
            strides.insert(0, s)
            s *= max(1, d)
    for i, (d, s) in enumerate(zip(dims, strides)):
        t.dims[i], t.strides[i] = d, s
    return t


def _rotation(L, **kw):
    r = L.KvrtRotation()
    r.turns, r.axis, r.head_dim, r.n_freq, r.norm, r.n_axes, r.eps, r.scaling = AT, AT, 128, 64, 3, 1, 1e-6, 1.0
    for name, value in kw.items():
        setattr(r, name, value)
    return r


def _call(lib, rot, q, k, v, pos, oq, ok, ov):
    ref = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731
    return lib.kvrt_rotate_heads_async(ref(rot), ref(q), ref(k), ref(v), ref(pos), ref(oq), ref(ok), ref(ov), None)


def test_empty_calls_launch_nothing():
    L, lib = _lib()
    for dims in ((0, 4, 3, 128), (2, 4, 0, 128), (2, 0, 3, 128)):
        q = _tensor(L, L.DT_BF16, dims, data=None)
        pos = _tensor(L, L.DT_INT32, (1, dims[0], dims[2]))
        assert _call(lib, _rotation(L), q, None, None, pos, q, None, None) == 0


@pytest.mark.parametrize("change", [
    {"head_dim": 96}, {"head_dim": 0}, {"n_freq": -8}, {"n_freq": 12}, {"n_freq": 72}, {"n_axes": 0}, {"n_axes": 5},
    {"norm": 8}, {"norm": -1}, {"adjacent": 2}, {"eps": -1e-6}, {"eps": math.nan}, {"eps": math.inf},
    {"scaling": math.nan}, {"scaling": math.inf}, {"turns": None}, {"turns": AT + 4}, {"axis": AT + 4},
    {"axis": None, "n_axes": 2}, {"q_weight": AT + 4}, {"k_weight": AT + 8},
])
def test_rotations_that_are_refused(change):
    L, lib = _lib()
    q = _tensor(L, L.DT_BF16, (2, 4, 3, 128))
    pos = _tensor(L, L.DT_INT32, (max(1, change.get("n_axes", 1)), 2, 3))
    assert _call(lib, _rotation(L, **change), q, None, None, pos, q, None, None) == L.KVRT_EINVAL


def test_arguments_that_are_refused():
    L, lib = _lib()
    rot = _rotation(L)
    q = _tensor(L, L.DT_BF16, (2, 4, 3, 128))
    pos = _tensor(L, L.DT_INT32, (1, 2, 3))
    bad = L.KVRT_EINVAL
    assert _call(lib, None, q, None, None, pos, q, None, None) == bad
    assert _call(lib, rot, None, None, None, pos, None, None, None) == bad
    assert _call(lib, rot, q, None, None, pos, None, None, None) == bad   # no destination
    assert _call(lib, rot, q, None, None, pos, q, q, None) == bad         # a destination without heads
    assert _call(lib, rot, q, None, None, None, q, None, None) == bad     # no positions
    for t in (_tensor(L, L.DT_FP32, (2, 4, 3, 128)), _tensor(L, L.DT_BF16, (2, 4, 128)),
              _tensor(L, L.DT_BF16, (2, 4, 3, 64)), _tensor(L, L.DT_BF16, (2, 4, 3, 128), data=None),
              _tensor(L, L.DT_BF16, (2, 4, 3, 128), data=AT + 8),
              _tensor(L, L.DT_BF16, (2, 4, 3, 128), (1536, 384, 128, 2)),
              _tensor(L, L.DT_BF16, (2, 4, 3, 128), (1536, 384, 132, 1)),
              _tensor(L, L.DT_BF16, (2, 4, 3, 128), (1536, -384, 128, 1)),
              _tensor(L, L.DT_BF16, (2, 4, -3, 128))):
        assert _call(lib, rot, t, None, None, pos, q, None, None) == bad
        assert _call(lib, rot, q, None, None, pos, t, None, None) == bad
    # a destination whose rows coincide; other shapes
    assert _call(lib, rot, q, None, None, pos, _tensor(L, L.DT_BF16, (2, 4, 3, 128), (1536, 0, 128, 1)), None, None) == bad
    assert _call(lib, rot, q, None, None, pos, _tensor(L, L.DT_BF16, (2, 5, 3, 128)), None, None) == bad
    k = _tensor(L, L.DT_BF16, (2, 1, 4, 128))
    assert _call(lib, rot, q, k, None, pos, q, k, None) == bad
    k = _tensor(L, L.DT_BF16, (3, 1, 3, 128))
    assert _call(lib, rot, q, k, None, pos, q, k, None) == bad
    for p in (_tensor(L, L.DT_FP32, (1, 2, 3)), _tensor(L, L.DT_INT32, (2, 3)), _tensor(L, L.DT_INT32, (2, 2, 3)),
              _tensor(L, L.DT_INT32, (1, 3, 3)), _tensor(L, L.DT_INT32, (1, 2, 2)),
              _tensor(L, L.DT_INT32, (1, 2, 3), data=None), _tensor(L, L.DT_INT32, (1, 2, 3), data=AT + 2),
              _tensor(L, L.DT_INT64, (1, 2, 3), data=AT + 4), _tensor(L, L.DT_INT32, (1, 2, 3), (6, -3, 1))):
        assert _call(lib, rot, q, None, None, p, q, None, None) == bad
    # more threads than 32 bits count: 2^24 * 3 rows of 16 heads of 8 lanes, and counts past 32 bits
    for dims in ((1 << 24, 16, 3, 128), (1 << 20, 4, 1 << 20, 128), (1 << 31, 4, 3, 128), (2, 1 << 30, 3, 128)):
        big = _tensor(L, L.DT_BF16, dims)
        p = _tensor(L, L.DT_INT32, (1, dims[0], dims[2]))
        assert _call(lib, rot, big, None, None, p, big, None, None) == bad


def test_python_refusals():
    from kvrt import HeadRotation

    f = [0.1] * 64
    for args, kw in (((96, f), {}), ((128, f), {"norm": "k"}), ((128, [0.1] * 12), {}), ((128, [0.1] * 72), {}),
                     ((128, torch.zeros(8, 8)), {}), ((128, f), {"axes": [0] * 63}), ((128, f), {"axes": [4] * 64}),
                     ((128, f), {"axes": [-1] * 64}), ((128, f), {"eps": -1.0}), ((128, f), {"eps": math.nan}),
                     ((128, f), {"scaling": math.inf}), ((128, f), {"q_weight": torch.ones(64)}),
                     ((128, f), {"k_weight": torch.ones(128, 1)}),
                     ((128, f), {"norm": "none", "q_weight": torch.ones(128)})):
        with pytest.raises(ValueError):
            HeadRotation(*args, **kw)
    from kvrt import KVRTError

    with pytest.raises(KVRTError):
        HeadRotation(128, [math.nan] * 8)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError):
            HeadRotation(128, f)
