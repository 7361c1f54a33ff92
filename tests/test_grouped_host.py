"""Host side of the bucketed and 8-bit operators, without a GPU: what the C entries are called with, and rules on the sources."""

import re
from pathlib import Path


def test_waits_for_tensor_memory_name_their_registers():
    """A wait without operands orders memory only: arithmetic on the registers that a read fills may move before it."""
    csrc = Path(__file__).parent.parent / "nnue_pytorch_b200" / "csrc"
    for name in ("tc.cuh", "grouped_tc.cuh", "grouped_linear.cu", "fp8_linear.cu"):
        source = (csrc / name).read_text()
        for wait in re.finditer(r'asm volatile\(\s*"tcgen05\.wait::ld[^;]*;"([^;]*);', source):
            named = wait.group(1).count('"+r"')
            assert named == 32, f"{name}: the wait for a read of 32 registers names {named}"
        assert "tmem_wait_ld()" not in source, name
