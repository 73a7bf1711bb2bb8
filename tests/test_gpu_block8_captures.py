"""Decode attention over 8-bit pages gives the same bits whatever calls the process
made before: as its first call, captured, and after more captured calls than there
are arrival counters for the joining of partials."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

CHILD = Path(__file__).with_name("block8_capture_child.py")


def _run(what: str) -> None:
    r = subprocess.run([sys.executable, "-u", str(CHILD), what], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), (r.returncode, r.stdout[-2000:], r.stderr[-3000:])


@pytest.mark.parametrize("what", ["first", "many", "layers"])
def test_captured_calls_give_the_eager_bits(what):
    _run(what)


def test_calls_on_every_threads_own_stream_keep_apart():
    """hipStreamPerThread is one handle for a stream of each thread: calls of two threads
    overlap on the GPU and give what they give alone."""
    import ctypes
    import threading

    import torch

    from kvrt import _lib as L
    from kvrt.runtime import tensor_desc
    from tests.block8_capture_child import SHAPES, served

    lib, per_thread = L.load(), ctypes.c_void_p(2)
    made = [served(SHAPES[0], seed) for seed in (1, 2)]
    want = [pool.attend(*args, max_q=1) for pool, args in made]
    torch.cuda.synchronize()
    outs = [[torch.zeros_like(w) for _ in range(20)] for w in want]
    works = []
    for pool, (q, table, *_) in made:
        size = lib.kvrt_block8_attend_work(pool._c(), *table.shape, q.shape[0], q.shape[1], 1)
        works.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    codes = [[], []]

    def run(i):
        pool, (q, table, lengths, starts, scale) = made[i]
        for out in outs[i]:  # one after the other on the thread's stream
            codes[i].append(lib.kvrt_block8_attend_async(
                pool._c(), tensor_desc(q), tensor_desc(table), lengths.data_ptr(), starts.data_ptr(), None, tensor_desc(out),
                scale, 0, 1, works[i].data_ptr(), works[i].numel(), per_thread))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    for i in range(2):
        assert codes[i] == [L.KVRT_OK] * 20
        assert all(torch.equal(out, want[i]) for out in outs[i]), i
        assert made[i][0].status() == 0
