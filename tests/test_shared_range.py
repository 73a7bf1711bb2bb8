"""Key ranges of chunks behind a shared prefix (csrc/kvrt_range.h, compiled for the host):
the ranges of a tile are whole blocks, cover every key that one of its queries sees, once,
and the rows that a block fetches lie in one slot."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "gemma-4-omni_amd" / "csrc"

PROGRAM = r"""
#include <algorithm>
#include <cstdio>
#include <set>
#include "kvrt_range.h"
using namespace kvrt;
int main() {
    const int block = 32;
    long n = 0;
    for (int P : {0, 1, 31, 32, 33, 64, 100, 257})
        for (int len : {0, 1, 3, 31, 32, 40, 129, 300})
            for (int Q : {1, 2, 33, 129, 200})
                for (int window : {0, 1, 5, 32, 100, 1000})
                    for (int qf = 0; qf < Q; qf += 1 + qf / 2)
                        for (int ql : {qf, std::min(Q - 1, qf + 31), Q - 1})
                            for (int nks : {1, 2, 3, 16}) {
                                const int own0 = (P + block - 1) / block * block, gap = own0 - P, base = own0 + len - Q;
                                std::multiset<int> got;
                                for (int ks = 0; ks < nks; ++ks, ++n) {
                                    const KeyRange r = shared_range(base, qf, ql, window, nks, ks, block, P, own0);
                                    if (r.kend > r.kstart && r.kstart % block) return std::printf("start %d\n", r.kstart), 1;
                                    for (int k = r.kstart; k < r.kend; ++k) got.insert(k);
                                    for (int kt = r.kstart; r.kend > r.kstart && kt < r.kend + 5 * block; kt += block) {
                                        // the fetch of the block at kt, as the kernel makes it
                                        const int t0 = std::min(kt, r.kend - 1);
                                        const bool own = t0 >= own0;
                                        const int key = own ? t0 - own0 : std::min(t0, P - 1);
                                        const int last = own ? r.kend - 1 - t0 : std::min(r.kend, P) - 1 - key;
                                        const int rows = own ? len : P;
                                        // (rows from the first key on, which one of the queries sees)
                                        const int first = std::max(0, shared_first_key(base + qf, window, P, own0) - t0);
                                        if (first > last) return std::printf("first %d > %d\n", first, last), 1;
                                        if (key < 0 || last < 0 || key + std::min(last, block - 1) >= rows)
                                            return std::printf("rows %d + %d of %d (P %d len %d Q %d kt %d)\n", key, last, rows, P, len, Q, kt), 1;
                                    }
                                }
                                for (int q = qf; q <= ql; ++q) {
                                    const int pos = P + len - Q + q;  // real
                                    for (int k = 0; k < P + len; ++k) {
                                        if (k > pos || (window > 0 && k <= pos - window)) continue;
                                        const int number = k < P ? k : k + gap;
                                        if (got.count(number) != 1)
                                            return std::printf("key %d seen by %d: %ld times\n", k, pos, (long)got.count(number)), 1;
                                        if (number < shared_first_key(base + q, window, P, own0)) return std::printf("first key\n"), 1;
                                    }
                                }
                            }
    std::printf("ok %ld\n", n);
    return 0;
}
"""


def test_ranges_cover_what_the_queries_see(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    src, exe = tmp_path / "probe.cpp", tmp_path / "probe"
    src.write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-O1", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.startswith("ok "), got.stdout
