"""CPU: kernels that are launched while the kernel before them drains read nothing as constant memory: what that kernel writes
changes during their life, and a read-only load may be moved ahead of the wait for it."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "fast_polynomial_transcendentals_b200" / "csrc"
EARLY = [p.name for p in sorted(CSRC.glob("*.cu")) if "griddepcontrol.wait" in p.read_text()]


def test_there_are_some():
    assert {"fpt_linear.cu", "fpt_qk_rope.cu"} <= set(EARLY)


@pytest.mark.parametrize("name", EARLY)
def test_no_read_only_loads(name):
    code = re.sub(r"//[^\n]*|/\*.*?\*/", "", (CSRC / name).read_text(), flags=re.S)
    assert not re.findall(r"__ldg\s*\(|__restrict__|ld\.global\.nc", code)
