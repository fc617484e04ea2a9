"""Flat scoring's C entries (csrc/flat.cc) over 2^32 - 1 rows, on the host with launches that only count
(tests/native/flat_rows.cc): every row is launched once, and the loops over blocks of rows end."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_entries_launch_every_row_once(tmp_path):
    exe = tmp_path / "flat_rows"
    inc = ROOT / "dm-hnsw-reference_amd" / "csrc"
    build = subprocess.run(["g++", "-O1", "-std=c++20", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{inc}",
                            str(ROOT / "tests" / "native" / "flat_rows.cc"), str(inc / "flat.cc"), "-o", str(exe)],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-2000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "rows ok" in run.stdout, run.stdout + run.stderr
