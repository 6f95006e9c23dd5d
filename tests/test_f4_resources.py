"""Registers, LDS and scratch of the 4-bit attention's kernels as the build reports them, held to what their source counts on."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROCM = Path("/opt/rocm/llvm/bin")
CSRC = Path(__file__).resolve().parent.parent / "roost_amd" / "csrc"
OBJECT = CSRC.parent / "_build" / "paged_attention_f4.o"
LDS, REGISTERS = 160 * 1024, 512  # of a CU; of a lane in all wavefronts of a SIMD


@pytest.fixture(scope="module")
def kernels_built(tmp_path_factory):
    """{(kernel, head_dim, ...): {property: number}}"""
    if not OBJECT.exists() or not all((ROCM / t).exists() for t in ("llvm-objcopy", "clang-offload-bundler", "llvm-readobj")):
        pytest.skip("no objects of a build, or no tools to read them with")
    tmp = tmp_path_factory.mktemp("co")
    shutil.copy(OBJECT, tmp / "in.o")
    subprocess.run([ROCM / "llvm-objcopy", f"--dump-section=.hip_fatbin={tmp / 'fat.bin'}", tmp / "in.o", tmp / "out.o"], check=True)
    subprocess.run([ROCM / "clang-offload-bundler", "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
                    f"--input={tmp / 'fat.bin'}", f"--output={tmp / 'gpu.co'}"], check=True)
    notes = subprocess.run([ROCM / "llvm-readobj", "--notes", tmp / "gpu.co"], check=True, capture_output=True, text=True).stdout
    found, numbers = {}, {}
    for line in notes.splitlines():
        m = re.match(r"    \.(\w+): +(\S+)$", line)  # a kernel's own, in the order of their names
        if m is None:
            continue
        if m[1] == "group_segment_fixed_size":
            numbers = {}
        if m[1] == "name":
            n = re.search(r"\d\d([A-Z]\w+Kernel)I((?:Li\d+E)+)E", m[2])
            found[(n[1], *map(int, re.findall(r"Li(\d+)E", n[2])))] = numbers
        elif m[2].isdigit():
            numbers[m[1]] = int(m[2])
    return found


def test_every_kernel_is_there(kernels_built):
    names = [k[0] for k in kernels_built]
    assert (names.count("RowAttentionKernel"), names.count("TileAttentionKernel")) == (15, 9)  # three caps each


def _holds(k, waves):
    """Workgroups of `waves` wavefronts a SIMD that a CU holds."""
    return min(REGISTERS // (8 * -(-k["vgpr_count"] // 8)) // waves, LDS // k["group_segment_fixed_size"])


def test_the_row_kernels_fit_as_often_as_keys_are_dealt_for(kernels_built):
    """RowsResident: the launch bounds ask for it and the host deals to it."""
    text = (CSRC / "paged_attention_f4.hip").read_text()
    assert "tiles == 2 || d == 256 ? 2 : d == 128 ? 3 : 4" in text
    for (name, d, *more), k in kernels_built.items():
        if name != "RowAttentionKernel":
            continue
        want = 2 if more[0] == 2 or d == 256 else 3 if d == 128 else 4
        assert _holds(k, 1) == want, (d, more, k)
        assert k["vgpr_spill_count"] == 0 and k["private_segment_fixed_size"] == 0, (d, more, k)


def test_the_tile_kernels(kernels_built):
    """No lane's values in scratch but at head_dim 256, where a few are, in front of and behind the loop over the keys; two
    workgroups a CU at head_dim 64, one of the far caps'."""
    for (name, d, *more), k in kernels_built.items():
        if name != "TileAttentionKernel":
            continue
        assert k["vgpr_spill_count"] <= (16 if d == 256 else 0), (d, more, k)
        assert _holds(k, 2) == (2 if d == 64 and more[0] < 2 else 1), (d, more, k)
