"""What AdamW, its 8-bit states and the clipping promise besides the step itself, as far as no GPU is
needed."""
import shutil
import subprocess
from pathlib import Path

import pytest

from flash_muon_b200 import _lib
from flash_muon_b200._lib import lib

ROOT = Path(__file__).resolve().parents[1]
INVALID = -1


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_codes_at_every_exponent_byte(tmp_path):
    exe = tmp_path / "state8_range_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", str(ROOT / "flash_muon_b200" / "csrc"), "-x", "c++",
                    str(ROOT / "tests" / "state8_range_check.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr


@pytest.mark.parametrize("dtype, size", [(_lib.FM_BF16, 2), (_lib.FM_F16, 2), (_lib.FM_F32, 4)])
def test_misaligned_values_are_refused(dtype, size):
    """By the host, ahead of the launch: on the GPU such an access is a fault."""
    for off in range(1, size):
        assert lib.fm_adamw8_values(0x1000, 0x2000, 32, 1, 0x3000 + off, dtype, None) == INVALID
        assert b"misaligned" in lib.fm_last_error()
        assert lib.fm_adamw8_encode(0x1000 + off, dtype, 32, 2, 0x2000, 0x3000, None) == INVALID
        assert b"misaligned" in lib.fm_last_error()
