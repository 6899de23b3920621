"""The 8-bit products' kernels as the compiler leaves them for gfx950 (no GPU): the order of LDS reads, waits and
meetings, on which their sums rest."""
import re
import shutil
import subprocess

import pytest

from yoda_scheduler_amd.ops import build

SOURCE = build.NATIVE / "hip" / "fp8_matmul.hip"


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    """{kernel's mangled name: its lines}"""
    if not (shutil.which("hipcc") or (build.ROCM / "bin" / "hipcc").exists()):
        pytest.skip("no hipcc")
    out = tmp_path_factory.mktemp("asm") / "fp8_matmul.s"
    subprocess.run([build.hipcc(), f"--offload-arch={build.ARCH}", "-O3", "-std=c++17", "-Xclang", "-target-feature",
                    "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S", str(SOURCE), "-o", str(out)],
                   check=True, capture_output=True, timeout=300)
    kernels, lines = {}, None
    for line in out.read_text().splitlines():
        if m := re.match(r"(_ZN\w+):", line):
            lines = kernels.setdefault(m[1], [])
        elif "s_endpgm" in line:
            lines = None
        elif lines is not None:
            lines.append(line.strip())
    return kernels


def _events(lines):
    """'read' of LDS, 'wait' for all LDS reads that the source itself asks for, 'meet', in the order of the text"""
    inline = False
    for line in lines:
        if "#ASMSTART" in line or "#ASMEND" in line:
            inline = "#ASMSTART" in line
        elif line.startswith("ds_read"):
            yield "read"
        elif inline and line.startswith("s_waitcnt") and "lgkmcnt(0)" in line:
            yield "wait"
        elif line.startswith("s_barrier"):
            yield "meet"


@pytest.mark.parametrize("kernel,meetings", [("k_eight", 2), ("k_mid", None)])
def test_no_read_of_lds_is_left_where_waves_meet(assembly, kernel, meetings):
    """What lies behind a meeting fills what was read before it, so each meeting of the loop has a wait of its own for
    all reads, and not one that the compiler happens to need for something else."""
    found = {n: ls for n, ls in assembly.items() if kernel in n}
    assert found
    for name, lines in found.items():
        events = list(_events(lines))
        loop = events[events.index("read"):]         # from the operands of the first step on
        at = [i for i, e in enumerate(loop) if e == "meet"]
        assert len(at) == meetings if meetings else at, (name, loop)
        for i in at:
            before = loop[:i]
            last = max((j for j, e in enumerate(before) if e != "wait"), default=-1)
            assert "wait" in before[last + 1:], (name, loop)


def test_inline_assembly_names_the_register_it_writes():
    """m0, the direct loads' place in LDS, belongs to the compiler: a statement that sets it says so."""
    found = 0
    for path in sorted((build.NATIVE / "hip").glob("*.h*")):
        for statement in re.findall(r"\basm\s+volatile\s*\((.*?)\);", path.read_text(), re.S):
            if re.search(r"\bm0, ", statement.partition("\n")[0]):
                found += 1
                assert '"m0"' in statement.rpartition(":")[2], (path.name, statement)
    assert found
