"""Numbers that 32 bits do not hold as arguments of attention behind a shared prefix: none of
them is taken for the number that its low word is (no GPU: tensors are GPU tensors in name
only, the library's calls a recorder)."""
from __future__ import annotations

import subprocess
import sys
import textwrap
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

PROGRAM = """
import ctypes, sys, threading, types
sys.path.insert(0, {pkg!r})
import torch
from kvrt import KVRTError, KVRuntime, runtime

host = torch.zeros(4096, dtype=torch.uint8)
storage = torch._C._construct_storage_from_data_pointer(host.data_ptr(), torch.device("cuda", 0), 4096)
q = torch._C._construct_CUDA_Tensor_From_Storage_And_Metadata(
    dict(size=(2, 2, 1, 64), stride=(128, 64, 64, 1), dtype=torch.bfloat16, storage_offset=0), storage)
seen = []

def shared(ctx, layer, n, slots, prefix, *rest):
    args = ctypes.c_int32(layer).value, tuple(slots), ctypes.c_int32(prefix).value  # (as the library sees them)
    seen.append(args)
    return 0 if args == (0, (0, 1), 2) else -1

rt = KVRuntime.__new__(KVRuntime)
rt.device = torch.device("cuda", 0)
rt._owner_thread = threading.get_ident()
rt._ctx = ctypes.c_void_p(8)
rt.lib = types.SimpleNamespace(kvrt_attend_shared_async=shared, kvrt_bind_stream=lambda c, s: 0,
                               kvrt_strerror=lambda c: b"refused")
rt._call = types.SimpleNamespace(attend_shared=lambda *a: 1)  # the general path
runtime.current_stream_handle = lambda d: 0

def call(layer=0, slots=(0, 1), prefix=2):
    return rt.attend_shared(layer, q, slots, 0.1, prefix_slot=prefix, out=q)

assert call() is q
for kw in (dict(prefix=2 ** 32 + 2), dict(prefix=2 ** 32 - 1), dict(prefix=2 ** 31), dict(prefix=2 ** 64 + 2), dict(layer=2 ** 32),
           dict(layer=-2 ** 32), dict(slots=(2 ** 32, 1)), dict(slots=(0, 2 ** 32 + 1)), dict(slots=[0, -2 ** 32 + 1])):
    try:
        call(**kw)
    except (KVRTError, ValueError):
        continue
    raise AssertionError((kw, seen[-1]))
print("done")
"""


def test_numbers_past_32_bits_are_refused():
    prog = textwrap.dedent(PROGRAM.format(pkg=str(ROOT / "gemma-4-omni_amd")))
    res = subprocess.run([sys.executable, "-c", prog], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip().endswith("done"), (res.returncode, res.stderr[-2000:])
