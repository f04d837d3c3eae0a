"""Guards on the sources and the compiler's output of kernels that address LDS copies through m0 and count their
outstanding vector memory operations."""
import re

import pytest

from sparse_amd import build


def test_inline_assembly_that_writes_m0_says_so():
    """The compiler keeps what it put into m0 unless a statement that writes it lists it as overwritten."""
    seen = 0
    for path in sorted(build.CSRC.glob("*.hip")) + sorted(build.CSRC.glob("*.h")):
        for statement in re.findall(r"asm\s+volatile\s*\((.*?)\)\s*;", path.read_text(), flags=re.S):
            if re.search(r"s_mov_b32 m0\b", statement):
                seen += 1
                assert '"m0"' in statement.rsplit(":", 1)[-1], (path.name, statement)
    assert seen >= 3
