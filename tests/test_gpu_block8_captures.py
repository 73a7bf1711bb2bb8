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


@pytest.mark.parametrize("name,hq,heads,dim", [("int8", 4, 2, 64), ("e4m3", 8, 1, 256), ("int8", 2, 1, 512)])
def test_a_captured_chunk_step_follows_the_lengths(name, hq, heads, dim):
    """Tables of so many rows that they take two launches, append, chunk attention and the
    padded batch in one graph; chunks of other lengths at each replay, some refused."""
    import torch

    from kvrt import Block8Pool, BlockTables
    from tests.helpers import randn_bf16

    gen = torch.Generator().manual_seed(dim)
    n, rows, block, pages = 3, 4400, 16, 330
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k, v = (torch.zeros((rows, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros((rows, hq, dim), dtype=torch.bfloat16, device="cuda")
    keep, new = i32([0] * n), i32([0] * n)

    def make():
        return (BlockTables(n, 300, pages, block_size=block), Block8Pool.zeros(pages, heads, dim, block_size=block, dtype=name),
                torch.full_like(q, 5.0))

    def step(tables, pool, out):
        plan = tables.update(keep, new, rows=rows)
        pool.append(k, v, plan.slot_map)
        pool.attend(q, tables.table, plan.lengths, plan.starts, dim ** -0.5, max_q=rows, granted=plan.granted, out=out)
        return (*plan, *pool.gather(tables.table, plan.lengths, 500, dtype=torch.float32))

    eager, graphed = make(), make()
    step(*make())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(*graphed)
    for lens, adds in (([0, 0, 0], [1400, 37, 1]), ([1400, 30, 1], [1, 2900, 33]), ([700, 0, 34], [4000, 100, 260]),
                       ([701, 100, 290], [64, 65, 4200]), ([0, 3, 0], [0, 4000, 400])):
        for t, x in ((keep, lens), (new, adds)):
            t.copy_(i32(x))
        for t in (k, v, q):
            t.copy_(randn_bf16(gen, t.shape))
        want = step(*eager)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), lens
        assert torch.equal(eager[2], graphed[2]), lens
        assert eager[0].status() == graphed[0].status() and eager[1].status() == graphed[1].status()
        for a, b in zip((eager[0].table, eager[0].free_count, eager[1].k.view(torch.int8), eager[1].v_scale),
                        (graphed[0].table, graphed[0].free_count, graphed[1].k.view(torch.int8), graphed[1].v_scale)):
            assert torch.equal(a, b), lens
