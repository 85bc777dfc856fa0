"""The draft kernels' code object: every kernel that the host asks for is there,
and none spills vector registers or touches scratch memory, which is memory
traffic in loops that are bound by registers and issue."""
import re
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HSACO = ROOT / "_build" / "er_draft.hsaco"
LLVM = Path("/opt/rocm/llvm/bin")


@pytest.fixture(scope="module")
def elf(tmp_path_factory):
    bundler = LLVM / "clang-offload-bundler"
    if not HSACO.exists() or not all((LLVM / t).exists() for t in ("clang-offload-bundler", "llvm-readobj", "llvm-objdump")):
        pytest.skip("built code object or ROCm LLVM tools not present")
    out = tmp_path_factory.mktemp("draft") / "draft.elf"
    subprocess.run([str(bundler), "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--input={HSACO}",
                    f"--output={out}"], check=True)
    return out


def test_kernels_and_spills(elf):
    notes = subprocess.run([str(LLVM / "llvm-readobj"), "--notes", str(elf)], check=True, capture_output=True, text=True).stdout
    spills, name = {}, None
    for line in notes.splitlines():
        m = re.match(r"\s+\.symbol:\s+(\S+)\.kd", line)
        name = m.group(1) if m else name
        m = re.match(r"\s+\.vgpr_spill_count:\s+(\d+)", line)
        if m:
            spills[name] = int(m.group(1))
    # three head widths: the acceptance and two joins of wide pieces; for three page sizes and two output types the wide
    # kernel and that of 16 columns, of 32 too below width 256; and these with their own two joins
    assert len(spills) == 3 * (3 + 3 * 2 * 2) + 2 * (3 * 2) + 5 * 2 + len([n for n in spills if n.startswith("er_choose")])
    assert {"er_choose_join", "er_kv8_accept_d64", "er_kv8_masked_attend_wide_d256_p16_f32"} <= set(spills)
    assert not {k: v for k, v in spills.items() if v}


def test_no_scratch_memory(elf):
    text = subprocess.run([str(LLVM / "llvm-objdump"), "-d", "--no-show-raw-insn", str(elf)], check=True, capture_output=True,
                          text=True).stdout
    assert "v_mfma" in text and not re.search(r"\bscratch_(load|store)", text)
