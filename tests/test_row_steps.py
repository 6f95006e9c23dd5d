"""The copies that GemmLora's wavefronts count on, over every width, on the host."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_no_step_is_used_before_its_copies_have_landed(tmp_path):
    """Issued against awaited copies. Rows of 8 bits take two copies of an adapter's rows a step, and a last step of 64 bytes or
    less issues only the first: a wait that counts on both would return while the step before is still on its way."""
    exe = tmp_path / "row_steps_count"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I", str(ROOT / "roost_amd" / "csrc"),
                    str(ROOT / "tests" / "row_steps_count.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout
