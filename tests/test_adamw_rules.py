"""What AdamW, its 8-bit states and the clipping promise besides the step itself, as far as no GPU is
needed."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_codes_at_every_exponent_byte(tmp_path):
    exe = tmp_path / "state8_range_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", str(ROOT / "flash_muon_b200" / "csrc"), "-x", "c++",
                    str(ROOT / "tests" / "state8_range_check.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
