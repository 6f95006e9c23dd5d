"""The copies from memory straight into LDS that are written in inline assembly."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROCM = Path("/opt/rocm/llvm/bin")
CSRC = Path(__file__).resolve().parent.parent / "roost_amd" / "csrc"
BUILD = CSRC.parent / "_build"


def test_m0_is_written_a_wait_state_before_the_copy_that_reads_it():
    """A copy takes its LDS address from M0, and an instruction that does so needs one wait state after a scalar write of M0.
    The compiler keeps to that for its own instructions and does not look into inline assembly."""
    found = 0
    for source in sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.h")]):
        for text in re.findall(r'asm volatile\("([^"]*global_load_lds[^"]*)"', source.read_text()):
            lines = [line.strip().split()[0] for line in text.split("\\n\\t")]
            copy = next(i for i, op in enumerate(lines) if op.startswith("global_load_lds"))
            write = max(i for i, line in enumerate(text.split("\\n\\t")[:copy]) if re.match(r"s_\w+ m0,", line))
            assert "s_nop" in lines[write + 1:copy], f"{source.name}: {text}"
            found += 1
    assert found >= 1


def _scalars(operand):
    """The scalar registers that an operand names."""
    m = re.match(r"s\[(\d+):(\d+)\]|s(\d+)$", operand.strip())
    if m is None:
        return set()
    return set(range(int(m[1]), int(m[2]) + 1)) if m[1] else {int(m[3])}


def _functions(text):
    """The disassembly's functions as lists of (address, opcode, operands, address of a branch's target)."""
    code = []
    start = 0
    for line in text.splitlines():
        head = re.match(r"([0-9a-f]+) <\S+>:", line)
        if head:
            if code:
                yield code
            code, start = [], int(head[1], 16)
            continue
        m = re.match(r"\t(\S+) ?(.*?)\s*// ([0-9A-F]+):(.*)", line)
        if m:
            target = re.search(r"<\S+?(?:\+0x([0-9a-f]+))?>", m[4]) if m[1].startswith(("s_branch", "s_cbranch")) else None
            code.append((int(m[3], 16), m[1], m[2], None if target is None else start + int(target[1] or "0", 16)))
    if code:
        yield code


def _hazards(code):
    """Copies into LDS whose scalar base a vector instruction wrote fewer than five wait states before, on any way to them."""
    at = {ins[0]: i for i, ins in enumerate(code)}
    before = [[] for _ in code]
    for i, (_, op, _, target) in enumerate(code):
        if i + 1 < len(code) and op not in ("s_branch", "s_endpgm"):
            before[i + 1].append(i)
        if target in at:
            before[at[target]].append(i)
    copies, found = 0, []
    for i, (address, op, operands, _) in enumerate(code):
        if not op.startswith("global_load_lds"):
            continue
        copies += 1
        needs = _scalars(operands.split(",")[1].split(" offset")[0].split(" nt")[0])
        ways = [(j, 0) for j in before[i]]
        while ways:
            j, states = ways.pop()
            _, earlier, its, _ = code[j]
            written = its.split(",")[:2 if "_co_" in earlier else 1]  # a carry is a second result
            if earlier.startswith("v_") and any(_scalars(w) & needs for w in written):
                found.append(f"{address:x}: {op} {operands} after {earlier} {its}, {states} wait states")
            states += int(its) + 1 if earlier == "s_nop" else 1
            if states < 5:
                ways += [(k, states) for k in before[j]]
    return copies, found


@pytest.mark.parametrize("name", ["gemm_lora", "gated_delta_rule", "paged_attention"])
def test_no_copy_reads_a_scalar_base_too_early(name, tmp_path):
    """A memory instruction may read a scalar register five wait states after a vector instruction wrote it. The compiler keeps to
    that for its own instructions; whether it put such a write in front of an assembly block is read from the objects that
    the build made of these sources."""
    obj = BUILD / f"{name}.o"
    if not obj.exists() or not all((ROCM / t).exists() for t in ("llvm-objcopy", "clang-offload-bundler", "llvm-objdump")):
        pytest.skip("no objects of a build, or no tools to read them with")
    fat, co = tmp_path / "fat.bin", tmp_path / "gpu.co"
    shutil.copy(obj, tmp_path / "in.o")
    subprocess.run([ROCM / "llvm-objcopy", f"--dump-section=.hip_fatbin={fat}", tmp_path / "in.o", tmp_path / "out.o"], check=True)
    subprocess.run([ROCM / "clang-offload-bundler", "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
                    f"--input={fat}", f"--output={co}"], check=True)
    text = subprocess.run([ROCM / "llvm-objdump", "-d", co], check=True, capture_output=True, text=True).stdout
    copies, found = 0, []
    for code in _functions(text):
        n, bad = _hazards(code)
        copies, found = copies + n, found + bad
    assert copies > 0 and not found, found[:5]


def test_the_scan_finds_what_it_looks_for():
    """Straight before, behind a loop's edge, and far enough away."""
    straight = [(0, "v_readfirstlane_b32", "s8, v1", None), (4, "s_mov_b32", "m0, s3", None), (8, "s_nop", "0", None),
                (12, "global_load_lds_dwordx4", "v2, s[8:9]", None), (20, "s_endpgm", "", None)]
    assert _hazards(straight)[0] == 1 and len(_hazards(straight)[1]) == 1
    far = [straight[0], (4, "s_nop", "4", None), (8, "global_load_lds_dwordx4", "v2, s[8:9]", None)]
    assert _hazards(far) == (1, [])
    loop = [(0, "s_mov_b32", "m0, s3", None), (4, "global_load_lds_dwordx4", "v2, s[8:9]", None),
            (8, "v_readlane_b32", "s9, v1, 3", None), (12, "s_cbranch_scc1", "0", 0)]
    assert len(_hazards(loop)[1]) == 1
    text = "0000000000000100 <f>:\n\ts_nop 0    // 000000000100: BF800000\n\ts_cbranch_scc1 7   // 000000000104: BF850007 <f+0x20>\n"
    assert list(_functions(text)) == [[(0x100, "s_nop", "0", None), (0x104, "s_cbranch_scc1", "7", 0x120)]]
