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


@pytest.mark.parametrize("what", ["first", "many"])
def test_captured_calls_give_the_eager_bits(what):
    _run(what)
