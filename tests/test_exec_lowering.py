"""The build's check that no register is saved to the other register file while the
lanes of a divergent region are off, without a GPU: listings with and without the
pattern."""
from __future__ import annotations

from kvrt import _build as B

GOOD = """
_ZN4kvrt1kE:
\ts_and_saveexec_b64 s[4:5], vcc
\ts_cbranch_execz .LBB0_2
; %bb.1:
\tglobal_load_dword v1, v[2:3], off
\tv_accvgpr_write_b32 a0, v1
.LBB0_2:
\tv_writelane_b32 v255, s9, 3
\ts_or_b64 exec, exec, s[4:5]
\tv_accvgpr_write_b32 a19, v30
\ts_endpgm
"""


def test_copies_inside_a_region_and_behind_it_pass():
    assert B.exec_errors(GOOD) == []


def test_a_copy_before_the_lanes_are_back_is_refused():
    lines = GOOD.splitlines()
    at = lines.index("\ts_or_b64 exec, exec, s[4:5]")
    for copy in ("v_accvgpr_write_b32 a19, v30", "v_accvgpr_read_b32 v30, a19", "scratch_store_dword off, v1, off"):
        bad = "\n".join(lines[:at] + ["\t" + copy + "  ; spill"] + lines[at:])
        assert B.exec_errors(bad) == [f"_ZN4kvrt1kE: {copy}"]


def test_each_kernel_is_named():
    lines = GOOD.splitlines()
    at = lines.index("\ts_or_b64 exec, exec, s[4:5]")
    bad = "\n".join(lines[:at] + ["\tv_accvgpr_mov_b32 a1, a2"] + lines[at:])
    both = bad + "\n" + bad.replace("_ZN4kvrt1kE", "kvrt_other").replace("LBB0", "LBB1")
    assert B.exec_errors(both) == ["_ZN4kvrt1kE: v_accvgpr_mov_b32 a1, a2", "kvrt_other: v_accvgpr_mov_b32 a1, a2"]
