"""The quotient that e4m3 codes are the roundings of, against division, on the host."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_no_quotient_is_on_the_wrong_side_of_a_midpoint(tmp_path):
    """Every seventh mantissa of the scale, next to every midpoint of two e4m3 values (all of them: argument 1)."""
    exe = tmp_path / "quotient_codes"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I", str(ROOT / "roost_amd" / "csrc"),
                    str(ROOT / "tests" / "quotient_codes.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe), "7"], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stdout
