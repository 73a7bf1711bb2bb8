"""8-bit pages without a GPU: struct layouts against the header, and every refusal of
the C entry points that is made before anything is launched. Pointers here are
host memory that no call reads."""
from __future__ import annotations

import ctypes
import json
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def _lib():
    from kvrt import _lib as L

    if not L.LIB_PATH.exists():
        pytest.fail("libkvrt.so is not built; run __graft_entry__.build() first")
    return L, L.load()


_PROBE = r"""
#include <stddef.h>
#include <stdio.h>
#include "kvrt.h"
#define F(S, m) printf("\"%s.%s\": [%zu, %zu],\n", #S, #m, offsetof(S, m), sizeof(((S *)0)->m))
int main(void) {
  printf("{\n");
  F(kvrt_block8, k); F(kvrt_block8, v); F(kvrt_block8, k_scale); F(kvrt_block8, v_scale); F(kvrt_block8, status);
  F(kvrt_block8, dtype); F(kvrt_block8, pages); F(kvrt_block8, kv_heads); F(kvrt_block8, block);
  F(kvrt_block8, head_dim); F(kvrt_block8, reserved);
  F(kvrt_block_tables, table); F(kvrt_block_tables, mapped); F(kvrt_block_tables, free_pages);
  F(kvrt_block_tables, free_count); F(kvrt_block_tables, work); F(kvrt_block_tables, status);
  F(kvrt_block_tables, n); F(kvrt_block_tables, max_pages); F(kvrt_block_tables, pool_pages);
  F(kvrt_block_tables, block);
  printf("\"sizes\": [%zu, %zu], \"bits\": [%d, %d], \"more\": [%d, %d], \"work\": [%d, %d]\n}\n", sizeof(kvrt_block8),
         sizeof(kvrt_block_tables), KVRT_BLOCK_BAD_INDEX, KVRT_BLOCK_NO_PAGES, KVRT_BLOCK_NOT_FINITE, KVRT_E4M3,
         (int)KVRT_BLOCK_TABLES_WORK(7), (int)(KVRT_CAP_BLOCK8 >> 14));
  return 0;
}
"""


def test_structs_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    L, lib = _lib()
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text(_PROBE)
    subprocess.run([gcc, "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = json.loads(subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout)
    assert got.pop("sizes") == [ctypes.sizeof(L.KvrtBlock8), ctypes.sizeof(L.KvrtBlockTables)]
    assert got.pop("bits") == [L.BLOCK_BAD_INDEX, L.BLOCK_NO_PAGES]
    assert got.pop("more") == [L.BLOCK_NOT_FINITE, L.DT_E4M3]
    assert got.pop("work") == [L.block_tables_work(7), 1]
    for key, where in got.items():
        name, field = key.split(".")
        desc = getattr({"kvrt_block8": L.KvrtBlock8, "kvrt_block_tables": L.KvrtBlockTables}[name], field)
        assert [desc.offset, desc.size] == where, key
    assert lib.kvrt_capabilities() & L.CAP_BLOCK8


HERE = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(HERE) + 255) & ~255


def _pages(L, **kw):
    p = L.KvrtBlock8()
    p.k = p.v = p.k_scale = p.v_scale = p.status = AT
    p.dtype, p.pages, p.kv_heads, p.block, p.head_dim = L.DT_INT8, 8, 2, 16, 128
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def _tensor(L, dtype, dims, strides=None, data=AT):
    t = L.KvrtTensor()
    t.data, t.dtype, t.ndim = data, dtype, len(dims)
    if strides is None:
        strides, at = [], 1
        for d in reversed(dims):
            strides.insert(0, at)
            at *= max(d, 1)
    for i, (d, s) in enumerate(zip(dims, strides)):
        t.dims[i], t.strides[i] = d, s
    return t


BAD_PAGES = [dict(dtype=0), dict(dtype=2), dict(pages=0), dict(pages=1 << 27), dict(kv_heads=0), dict(kv_heads=65),
             dict(block=8), dict(block=24), dict(block=256), dict(head_dim=96), dict(head_dim=1024), dict(k=None),
             dict(v=AT + 8), dict(k_scale=None), dict(v_scale=AT + 2), dict(status=None)]


@pytest.mark.parametrize("bad", BAD_PAGES)
def test_pages_are_checked(bad):
    L, lib = _lib()
    p = _pages(L, **bad)
    k = _tensor(L, L.DT_BF16, (3, p.kv_heads, p.head_dim))
    assert lib.kvrt_block8_append_async(p, k, k, AT, None) == L.KVRT_EINVAL
    table = _tensor(L, L.DT_INT32, (2, 4))
    o = _tensor(L, L.DT_BF16, (2, p.kv_heads, 5, p.head_dim))
    assert lib.kvrt_block8_gather_async(p, table, AT, None, o, o, None, None) == L.KVRT_EINVAL
    q = _tensor(L, L.DT_BF16, (2, 2 * p.kv_heads, p.head_dim))
    assert lib.kvrt_block8_attend_async(p, q, table, AT, AT, None, q, 1.0, 0, 1, AT, 1 << 30, None) == L.KVRT_EINVAL
    assert lib.kvrt_block8_attend_work(p, 2, 4, 2, 4, 1) == 0


def test_append_refusals():
    L, lib = _lib()
    p = _pages(L)
    good = _tensor(L, L.DT_BF16, (3, 2, 128))
    call = lambda k, v, slots=AT: lib.kvrt_block8_append_async(p, k, v, slots, None)  # noqa: E731
    for bad in (_tensor(L, L.DT_FP32, (3, 2, 128)), _tensor(L, L.DT_BF16, (3, 1, 128)), _tensor(L, L.DT_BF16, (3, 2, 64)),
                _tensor(L, L.DT_BF16, (2, 2, 128)), _tensor(L, L.DT_BF16, (1, 3, 2, 128)),
                _tensor(L, L.DT_BF16, (3, 2, 128), (256, 128, 2)), _tensor(L, L.DT_BF16, (3, 2, 128), (260, 128, 1)),
                _tensor(L, L.DT_BF16, (3, 2, 128), (-256, 128, 1)), _tensor(L, L.DT_BF16, (3, 2, 128), data=AT + 8),
                _tensor(L, L.DT_BF16, (3, 2, 128), data=None)):
        assert call(good, bad) == L.KVRT_EINVAL and call(bad, good) == L.KVRT_EINVAL
    assert lib.kvrt_block8_append_async(p, None, good, AT, None) == L.KVRT_EINVAL
    assert lib.kvrt_block8_append_async(None, good, good, AT, None) == L.KVRT_EINVAL
    assert call(good, good, None) == L.KVRT_EINVAL and call(good, good, AT + 2) == L.KVRT_EINVAL
    empty = _tensor(L, L.DT_BF16, (0, 2, 128), data=None)
    assert call(empty, empty, None) == L.KVRT_OK  # nothing to do, nothing launched


def test_gather_refusals():
    L, lib = _lib()
    p = _pages(L)
    table = _tensor(L, L.DT_INT32, (2, 4))
    o = _tensor(L, L.DT_BF16, (2, 2, 5, 128))

    def call(t=table, lens=AT, start=None, k=o, v=o, mask=None):
        return lib.kvrt_block8_gather_async(p, t, lens, start, k, v, mask, None)

    for bad in (_tensor(L, L.DT_INT64, (2, 4)), _tensor(L, L.DT_INT32, (2,)), _tensor(L, L.DT_INT32, (3, 4)),
                _tensor(L, L.DT_INT32, (2, 1 << 28)), _tensor(L, L.DT_INT32, (2, 4), data=None),
                _tensor(L, L.DT_INT32, (2, 4), (8, 2)), None):
        assert call(t=bad) == L.KVRT_EINVAL
    for bad in (_tensor(L, L.DT_FP32, (2, 2, 5, 128)), _tensor(L, L.DT_BF16, (2, 2, 6, 128)), _tensor(L, L.DT_BF16, (2, 1, 5, 128)),
                _tensor(L, L.DT_BF16, (2, 2, 5, 64)), _tensor(L, L.DT_BF16, (2, 2, 5, 128), (1280, 640, 0, 1)),
                _tensor(L, L.DT_BF16, (2, 2, 5, 128), (1280, 320, 128, 1)), _tensor(L, L.DT_INT8, (2, 2, 5, 128)), None):
        assert call(v=bad) == L.KVRT_EINVAL
    for bad in (_tensor(L, L.DT_INT32, (2, 5)), _tensor(L, L.DT_BOOL, (2, 6)), _tensor(L, L.DT_BOOL, (1, 5)),
                _tensor(L, L.DT_BOOL, (2, 5), (0, 1))):
        assert call(mask=bad) == L.KVRT_EINVAL
    assert call(lens=None) == L.KVRT_EINVAL and call(start=AT + 1) == L.KVRT_EINVAL
    none = _tensor(L, L.DT_BF16, (2, 2, 0, 128), data=None)
    assert call(k=none, v=none) == L.KVRT_OK


def test_attend_refusals():
    L, lib = _lib()
    p = _pages(L)
    table = _tensor(L, L.DT_INT32, (2, 400))
    q = _tensor(L, L.DT_BF16, (2, 4, 128))
    size = lib.kvrt_block8_attend_work(p, 2, 400, 2, 4, 1)
    assert size > 0

    def call(t=table, x=q, o=q, lens=AT, starts=AT, granted=None, scale=1.0, window=0, max_q=1, work=AT, nbytes=size):
        return lib.kvrt_block8_attend_async(p, x, t, lens, starts, granted, o, scale, window, max_q, work, nbytes, None)

    for bad in (_tensor(L, L.DT_FP32, (2, 4, 128)), _tensor(L, L.DT_BF16, (2, 3, 128)), _tensor(L, L.DT_BF16, (2, 4, 64)),
                _tensor(L, L.DT_BF16, (2, 0, 128)), _tensor(L, L.DT_BF16, (2, 130, 128)), _tensor(L, L.DT_BF16, (1, 2, 4, 128)),
                _tensor(L, L.DT_BF16, (2, 4, 128), (516, 128, 1)), None):
        assert call(x=bad, o=bad) == L.KVRT_EINVAL
    for bad in (_tensor(L, L.DT_BF16, (1, 4, 128)), _tensor(L, L.DT_BF16, (2, 4, 128), (128, 128, 1)), None):
        assert call(o=bad) == L.KVRT_EINVAL
    for kw in (dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(max_q=-1), dict(max_q=1 << 30),
               dict(lens=None), dict(starts=AT + 2), dict(granted=AT + 1), dict(work=None), dict(work=AT + 8),
               dict(nbytes=size - 1), dict(t=_tensor(L, L.DT_INT32, (2, 1 << 28)))):
        assert call(**kw) == L.KVRT_EINVAL, kw
    none = _tensor(L, L.DT_BF16, (0, 4, 128), data=None)
    assert call(x=none, o=none) == L.KVRT_OK and call(max_q=0) == L.KVRT_OK


def test_tables_refusals():
    L, lib = _lib()

    def call(rows=8, lens=AT, new=AT, starts=AT, slots=AT, out=AT, granted=AT, **kw):
        t = L.KvrtBlockTables()
        t.table = t.mapped = t.free_pages = t.free_count = t.work = t.status = AT
        t.n, t.max_pages, t.pool_pages, t.block = 4, 10, 40, 16
        for name, value in kw.items():
            setattr(t, name, value)
        return lib.kvrt_block_tables_update_async(t, lens, new, rows, starts, slots, out, granted, None)

    for kw in (dict(n=0), dict(n=65537), dict(max_pages=0), dict(max_pages=1 << 29), dict(pool_pages=0), dict(pool_pages=1 << 27),
               dict(block=0), dict(block=17), dict(block=256), dict(rows=-1), dict(rows=(1 << 30) + 1), dict(n=65536, max_pages=1 << 15),
               dict(table=None), dict(mapped=None), dict(free_pages=AT + 1), dict(free_count=None), dict(work=None),
               dict(status=None), dict(lens=None), dict(new=None), dict(starts=AT + 2), dict(slots=None), dict(out=None),
               dict(granted=None)):
        assert call(**kw) == L.KVRT_EINVAL, kw
    assert lib.kvrt_block_tables_update_async(None, AT, AT, 0, AT, AT, AT, AT, None) == L.KVRT_EINVAL


def test_python_objects_need_a_gpu():
    import torch

    from kvrt import Block8Pool, BlockTables

    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    with pytest.raises(RuntimeError, match="GPU"):
        BlockTables(2, 4, 8)
    with pytest.raises(ValueError, match="block_size"):
        BlockTables(2, 4, 8, block_size=24)
    with pytest.raises(ValueError, match="32 bits"):
        BlockTables(2, 1 << 27, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        Block8Pool.zeros(4, 1, 128)
    with pytest.raises(ValueError, match="dtype"):
        Block8Pool.zeros(4, 1, 128, dtype="bf16")
    t = torch.zeros((4, 1, 16, 128), dtype=torch.int8)
    with pytest.raises(ValueError, match="GPU"):
        Block8Pool(t, t, t, t)


def test_tables_hold_at_most_two_to_the_thirty_positions():
    L, lib = _lib()
    p = _pages(L)
    wide = _tensor(L, L.DT_INT32, (2, (1 << 30) // p.block + 1))
    o, q = _tensor(L, L.DT_BF16, (2, 2, 5, 128)), _tensor(L, L.DT_BF16, (2, 4, 128))
    assert lib.kvrt_block8_gather_async(p, wide, AT, None, o, o, None, None) == L.KVRT_EINVAL
    assert lib.kvrt_block8_attend_async(p, q, wide, AT, AT, None, q, 1.0, 0, 1, AT, 1 << 40, None) == L.KVRT_EINVAL


WORKED = [(n, width, rows, hq, max_q, dim, block) for n in (1, 3, 70) for width in (0, 1, 9, 400) for rows in (1, 5, 900)
          for hq, max_q in ((2, 1), (16, 2), (16, 5), (64, 300)) for dim, block in ((64, 16), (512, 128))]


@pytest.mark.parametrize("dim,block", [(64, 16), (512, 128)])
def test_attend_takes_the_workspace_it_asks_for(dim, block):
    """Every size that attend_work answers is accepted (the launch itself then fails here),
    and one byte less is refused; tables without columns among them."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the calls would launch on host memory")
    L, lib = _lib()
    p = _pages(L, head_dim=dim, block=block)
    for n, width, rows, hq, max_q, *shape in WORKED:
        if shape != [dim, block]:
            continue
        size = lib.kvrt_block8_attend_work(p, n, width, rows, hq, max_q)
        table = _tensor(L, L.DT_INT32, (n, width), data=AT if width else None)
        q = _tensor(L, L.DT_BF16, (rows, hq, dim))
        call = lambda work, nbytes: lib.kvrt_block8_attend_async(p, q, table, AT, AT, None, q, 1.0, 0, max_q, work,  # noqa: E731
                                                                 nbytes, None)
        assert call(AT if size else None, size) == L.KVRT_EDEVICE, (n, width, rows, hq, max_q)
        if size:
            assert call(AT, size - 1) == L.KVRT_EINVAL
    assert lib.kvrt_block8_attend_work(p, 2, -1, 2, 4, 1) == 0


def test_tables_that_update_takes_are_tables_that_attention_reads():
    """One limit of requests (65535) and of positions (2^30) for all calls."""
    import torch

    from kvrt import BlockTables

    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the calls would launch on host memory")
    L, lib = _lib()

    def update(n, max_pages, block):
        t = L.KvrtBlockTables()
        t.table = t.mapped = t.free_pages = t.free_count = t.work = t.status = AT
        t.n, t.max_pages, t.pool_pages, t.block = n, max_pages, 8, block
        return lib.kvrt_block_tables_update_async(t, AT, AT, 1, AT, AT, AT, AT, None)

    def read(n, width, block):
        p, table = _pages(L, block=block), _tensor(L, L.DT_INT32, (n, width))
        o, q = _tensor(L, L.DT_BF16, (n, 2, 5, 128)), _tensor(L, L.DT_BF16, (2, 4, 128))
        return (lib.kvrt_block8_gather_async(p, table, AT, None, o, o, None, None),
                lib.kvrt_block8_attend_async(p, q, table, AT, AT, None, q, 1.0, 0, 1, AT, 1 << 40, None))

    for block in (16, 128):
        most = (1 << 30) // block
        for n, width in ((1, most), (65535, 9)):
            assert update(n, width, block) == L.KVRT_EDEVICE and read(n, width, block) == (L.KVRT_EDEVICE,) * 2
            with pytest.raises(RuntimeError, match="GPU"):
                BlockTables(n, width, 8, block_size=block)
        for n, width in ((1, most + 1), (65536, 9), (65537, 9)):
            assert update(n, width, block) == L.KVRT_EINVAL and read(n, width, block) == (L.KVRT_EINVAL,) * 2
            with pytest.raises(ValueError, match="65535|positions"):
                BlockTables(n, width, 8, block_size=block)


def test_decode_divides_over_the_workgroups_that_run_at_a_time():
    """A unit of work per place: waves a SIMD as the build reports them for the kernel
    (a workgroup of four waves takes one on each), 256 CUs."""
    L, lib = _lib()
    report = L.LIB_PATH.parent / "kernel_resources.json"
    if not report.exists():
        pytest.skip("the build left no report")
    built = json.loads(report.read_text())
    for dim in (64, 128, 256, 512):
        waves = [int(v["Occupancy"]) for k, v in built.items() if "block8_attend_kernel" in k and f"ELi{dim}E" in k]
        assert len(waves) == 2  # int8, e4m3
        p = _pages(L, head_dim=dim, kv_heads=8)
        size = lib.kvrt_block8_attend_work(p, 64, 500, 64, 8, 1)
        assert size == 256 * min(waves) * 2 * 16 * (4 * dim + 8), dim


def test_launches_of_more_threads_than_32_bits_count_are_refused():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the calls would launch on host memory")
    L, lib = _lib()
    for heads, most in ((1, (1 << 29) - 32), (8, (1 << 26) - 16)):  # a wave for 16 rows of each head of K and V
        p = _pages(L, kv_heads=heads, head_dim=64)
        for rows, want in ((most, L.KVRT_EDEVICE), (2 * most, L.KVRT_EINVAL)):
            x = _tensor(L, L.DT_BF16, (rows, heads, 64))
            assert lib.kvrt_block8_append_async(p, x, x, AT, None) == want, (heads, rows)
    table = _tensor(L, L.DT_INT32, (1, 4))
    for dim, rows in ((128, 32), (512, 8)):  # rows a workgroup of 256 threads
        p, most = _pages(L, kv_heads=1, head_dim=dim), ((1 << 24) - 1) * rows
        for lmax, want in ((most, L.KVRT_EDEVICE), (most + 1, L.KVRT_EINVAL)):
            o = _tensor(L, L.DT_BF16, (1, 1, lmax, dim))
            assert lib.kvrt_block8_gather_async(p, table, AT, None, o, o, None, None) == want, (dim, lmax)
