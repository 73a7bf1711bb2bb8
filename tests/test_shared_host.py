"""Shared-prefix attention's entry points without a GPU: refusals ahead of a context, and the
native call module's own error handling (tensors are GPU tensors in name only)."""
from __future__ import annotations

import ctypes
import subprocess
import sys
import textwrap
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

PROGRAM = """
import ctypes, sys, threading
sys.path.insert(0, {pkg!r})
import torch
from kvrt import TalkerMask, _lib

mod = _lib.load_calls()
host = torch.zeros(4096, dtype=torch.uint8)
storage = torch._C._construct_storage_from_data_pointer(host.data_ptr(), torch.device("cuda", 0), 4096)

def gpu(size, stride, dtype=torch.bfloat16):
    return torch._C._construct_CUDA_Tensor_From_Storage_And_Metadata(
        dict(size=size, stride=stride, dtype=dtype, storage_offset=0), storage)

P = ctypes.c_void_p
seen = []
bind = ctypes.CFUNCTYPE(ctypes.c_int, P, P)(lambda c, s: 0)
no = ctypes.CFUNCTYPE(ctypes.c_int, P, P)(lambda c, s: -2)

def call(ctx, layer, n, slots, prefix, q, out, scale, cap, slopes):
    seen.append((ctx, layer, n, list(ctypes.cast(slots, ctypes.POINTER(ctypes.c_int32))[:n]), prefix, scale, cap, slopes))
    return 0

entry = ctypes.CFUNCTYPE(ctypes.c_int, P, ctypes.c_int32, ctypes.c_int32, P, ctypes.c_int32, P, P, ctypes.c_float,
                         ctypes.c_float, P)(call)
addr = lambda f: ctypes.cast(f, P).value
other = addr(bind)
t = gpu((1, 2, 1, 64), (128, 64, 64, 1))
apart = gpu((1, 2, 1, 64), (256, 128, 128, 1))
slopes = gpu((2,), (1,), torch.float32)
run = lambda slots=[3], scale=0.5, q=t, out=t, prefix=1, cap=0.25, bias=slopes: mod.attend_shared(
    8, 0, 4, slots, scale, q, out, prefix, cap, bias)
mod.connect(TalkerMask, addr(bind), other, other, other, other, other, other)
mod.connect_shared(addr(entry))
assert run() == 0 and run(bias=None, prefix=-1) == 0
assert seen == [(8, 4, 1, [3], 1, 0.5, 0.25, host.data_ptr()), (8, 4, 1, [3], -1, 0.5, 0.25, None)], seen
# what it does not read itself goes to the general path, and nothing ran
for kw in (dict(slots=(3.0,)), dict(scale=1), dict(q=apart), dict(q=torch.zeros(1, 2, 1, 64)), dict(out=torch.zeros(1)),
           dict(prefix=None), dict(prefix=1 << 40), dict(cap=0), dict(bias=1.0), dict(q=None), dict(slots=7)):
    assert run(**kw) == 1, kw
mod.connect(TalkerMask, addr(no), other, other, other, other, other, other)
assert run() == 1 and len(seen) == 2
mod.connect(TalkerMask, addr(bind), other, other, other, other, other, other)
cxx = ctypes.CDLL("libstdc++.so.6")
for thrown in ("_ZSt17__throw_bad_allocv", "_ZSt16__throw_bad_castv"):
    mod.connect_shared(addr(getattr(cxx, thrown)))
    assert run() == -3
    got = []
    th = threading.Thread(target=lambda: got.append(run()))
    th.start()
    th.join()
    assert got == [-3]
for args in ((), (0,), (1, 2), ("x",)):
    try:
        mod.connect_shared(*args)
    except TypeError:
        continue
    raise AssertionError(args)
print("done")
"""


def test_the_native_call():
    prog = textwrap.dedent(PROGRAM.format(pkg=str(ROOT / "gemma-4-omni_amd")))
    res = subprocess.run([sys.executable, "-c", prog], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip().endswith("done"), (res.returncode, res.stderr[-2000:])


def test_refusals_without_a_context():
    from kvrt import _lib as L

    lib = L.load()
    assert lib.kvrt_capabilities() >> 16 & 1
    slots = (ctypes.c_int32 * 1)(0)
    t = L.KvrtTensor()
    call = lib.kvrt_attend_shared_async
    assert call(None, 0, 1, slots, -1, ctypes.byref(t), ctypes.byref(t), 1.0, 0.0, None) == -1
