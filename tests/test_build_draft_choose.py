"""The kernels of rules on logits that the built code object has, by name and number."""
import re
import subprocess

from test_build_draft import LLVM
from test_build_draft import elf  # noqa: F401  (fixture)


def test_choose_kernels(elf):  # noqa: F811
    notes = subprocess.run([str(LLVM / "llvm-readobj"), "--notes", str(elf)], check=True, capture_output=True, text=True).stdout
    names = re.findall(r"\.symbol:\s+(\S+)\.kd", notes)
    assert sorted(n for n in names if n.startswith("er_choose")) == ["er_choose_join", "er_choose_s1", "er_choose_s2"]
    assert len(names) == len(set(names)) == 3 * (3 + 3 * 2 * 2) + 2 * (3 * 2) + 5 * 2 + 3
