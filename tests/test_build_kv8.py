"""The cache kernels' code object: no kernel has a private (scratch) segment,
which is memory traffic in loops that are bound by registers and issue."""
import re
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HSACO = ROOT / "_build" / "er_kv8.hsaco"
LLVM = Path("/opt/rocm/llvm/bin")


def test_no_private_segment(tmp_path):
    bundler, readobj = LLVM / "clang-offload-bundler", LLVM / "llvm-readobj"
    if not HSACO.exists() or not bundler.exists() or not readobj.exists():
        pytest.skip("built code object or ROCm LLVM tools not present")
    elf = tmp_path / "kv8.elf"
    subprocess.run([str(bundler), "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
                    f"--input={HSACO}", f"--output={elf}"], check=True)
    notes = subprocess.run([str(readobj), "--notes", str(elf)], check=True, capture_output=True, text=True).stdout
    kernels, name = {}, None
    for line in notes.splitlines():
        m = re.match(r"\s+\.name:\s+(\S+)", line)
        if m:
            name = m.group(1)
        m = re.match(r"\s+\.private_segment_fixed_size:\s+(\d+)", line)
        if m:
            kernels[name] = int(m.group(1))
    # three head widths: norm, append, two joins; and for three page sizes and two output types both attention kernels
    assert len(kernels) == 3 * (4 + 3 * 2 * 2)
    assert not {k: v for k, v in kernels.items() if v}
