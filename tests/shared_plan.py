"""Divisions of calls behind a shared prefix (csrc/kvrt_shared_plan.h), computed on the host."""
from __future__ import annotations

import shutil
import subprocess
import tempfile
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
LAYOUTS = {"contig": 0, "ring": 1, "paged": 2}

PROGRAM = r"""
#include <cstdio>
#include "kvrt_shared_plan.h"
using namespace kvrt;
int main() {
    int D, hkv, group, n, q, layout, window, tiles_ok;
    long long pre, room, x;
    while (std::scanf("%d %d %d %d %d %d %d %d %lld %lld", &D, &hkv, &group, &n, &q, &layout, &window, &tiles_ok, &pre, &room) == 10) {
        int64_t rows[64];
        for (int i = 0; i < n; ++i) {
            if (std::scanf("%lld", &x) != 1) return 1;
            rows[i] = x;
        }
        SharedArgs a{};
        SharedChunkArgs p{};
        a.kv.kv_heads = p.kv.kv_heads = hkv;
        a.kv.layout = p.kv.layout = layout;
        a.group = p.group = group;
        a.qn = p.qn = q;
        a.n_items = p.n_items = n;
        a.window = p.window = window;
        a.prefix_slot = p.prefix_slot = pre >= 0 ? n : -1;
        const bool tiles = plan_shared_call(a, p, D, tiles_ok != 0, pre > 0 ? pre : 0, rows, (size_t)room);
        const size_t bytes = shared_part_bytes((int64_t)n * hkv * group * q, tiles ? p.n_ksplit : a.parts, D);
        std::printf("%d %d %d %d %d %d %d %d %d %d %d %d %zu\n", tiles, p.row_waves, p.key_parts, p.n_ksplit, a.joined, a.pre_tiles,
                    a.pre_splits, a.own_tiles, a.own_splits, a.own_per, a.own_wgs, a.parts, bytes);
    }
    return 0;
}
"""
FIELDS = ("tiles", "row_waves", "key_parts", "ranges", "joined", "pre_tiles", "pre_splits", "own_tiles", "own_splits",
          "own_per", "own_wgs", "parts", "bytes")

_exe: Path | None = None
_dir: tempfile.TemporaryDirectory | None = None  # (gone with the process)


def _program() -> Path | None:
    """The compiled program, once a process; None without a host compiler or HIP's headers."""
    global _exe, _dir
    if _exe is None:
        gxx = shutil.which("g++")
        if gxx is None or not Path("/opt/rocm/include/hip/hip_runtime.h").exists():
            return None
        _dir = tempfile.TemporaryDirectory(prefix="kvrt_plan_")
        where = Path(_dir.name)
        (where / "plan.cpp").write_text(PROGRAM)
        subprocess.run([gxx, "-std=c++17", "-O2", "-w", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{ROOT / 'include'}",
                        f"-I{ROOT / 'gemma-4-omni_amd' / 'csrc'}", str(where / "plan.cpp"), "-o", str(where / "plan")], check=True)
        _exe = where / "plan"
    return _exe


def plans(calls: list[dict]) -> list[dict] | None:
    """The division of each call: head_dim d, hkv, hq, q, own (rows seen of each session), prefix
    (rows seen; None: no prefix), and optionally layout, window, tiles (False: masks), room."""
    exe = _program()
    if exe is None:
        return None
    text = []
    for c in calls:
        prefix = c.get("prefix")
        text.append(" ".join(map(str, (c["d"], c["hkv"], c["hq"] // c["hkv"], len(c["own"]), c["q"], LAYOUTS[c.get("layout", "contig")],
                                       c.get("window", 0), int(c.get("tiles", True)), -1 if prefix is None else prefix,
                                       c.get("room", 1 << 30), *c["own"]))))
    got = subprocess.run([str(exe)], input="\n".join(text) + "\n", capture_output=True, text=True, check=True)
    return [dict(zip(FIELDS, map(int, line.split()))) for line in got.stdout.splitlines()]


def forms(c: dict, p: dict) -> set[tuple]:
    """The kernels of a call and what they run as: ("chunk", d, layout, row waves, key parts,
    split), ("unit", d, layout, 16-row blocks a wave, whose keys, past the caches) and ("join", d,
    groups of a row's parts), as csrc/kvrt_shared_kernel.h and kvrt_shared_chunk.hip choose them."""
    d, layout, n, rows = c["d"], c.get("layout", "contig"), len(c["own"]), c["hq"] // c["hkv"] * c["q"]
    if p["tiles"]:
        return {("chunk", d, layout, p["row_waves"], p["key_parts"], p["ranges"] > 1)}
    tile = 128 if d <= 128 else 64
    prefix = c.get("prefix") or 0
    large = (sum(c["own"]) + prefix) * c["hkv"] * d * 4 > 128 << 20 and layout != "paged"

    def blocks(total, tiles):
        sizes = {min(total - tile * t, tile) for t in {0, tiles - 1}}
        return {0 if s <= 16 else 1 if tile == 64 or s <= 64 else 2 for s in sizes}

    got = set()
    if p["pre_tiles"]:
        got |= {("unit", d, layout, b, "prefix", large and p["pre_tiles"] == 1) for b in blocks(n * rows, p["pre_tiles"])}
    whose = "both" if p["joined"] else "own"
    got |= {("unit", d, layout, b, whose, large and p["own_tiles"] == 1 and not p["joined"]) for b in blocks(rows, p["own_tiles"])}
    if p["parts"] > 1:
        groups = 2 if d == 512 else 4 if d == 256 else 8
        while groups > 1 and p["parts"] <= 8 * (groups // 2):
            groups //= 2
        got.add(("join", d, groups))
    return got


def every_form() -> set[tuple]:
    """All that the kernels are compiled as (a chunk's key ranges and units past the caches apart)."""
    out = set()
    for d in (64, 128, 256, 512):
        for layout in LAYOUTS:
            shapes = [(4, 1)] + ([(2, 2)] if d <= 256 else []) + ([(2, 4)] if d <= 128 else [])
            if d <= 128 and layout != "paged":
                shapes.append((1, 4))
            out |= {("chunk", d, layout, *s, split) for s in shapes for split in (False, True)}
            for b in range(3 if d <= 128 else 2):
                out |= {("unit", d, layout, b, whose, False) for whose in ("prefix", "own", "both")}
                if layout != "paged":
                    out |= {("unit", d, layout, b, whose, True) for whose in ("prefix", "own")}
        out |= {("join", d, g) for g in (1, 2, 4, 8) if g <= (2 if d == 512 else 4 if d == 256 else 8)}
    return out
