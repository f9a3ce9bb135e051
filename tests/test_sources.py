"""Rules of the hardware that the compiler does not see to inside inline asm,
checked in the sources' text."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _copies_to_lds():
    """(file, the copy, the instructions of its asm block before it)"""
    for path in sorted(glob.glob(os.path.join(ROOT, "proxima_amd", "csrc", "*.h*"))):
        for text in re.findall(r'asm volatile\(((?:\s*"[^"]*")+)', open(path).read()):
            lines = "".join(re.findall(r'"([^"]*)"', text)).replace("\\t", "").split("\\n")
            for i, line in enumerate(lines):
                if re.search(r"\blds\b|_load_lds_", line):
                    yield os.path.basename(path), line, lines[:i]


def test_m0_has_its_wait_state_before_a_copy_to_lds():
    # SALU write of m0, then a load to LDS that takes its address from it: one wait state between them
    copies = list(_copies_to_lds())
    assert len(copies) >= 6
    for name, line, before in copies:
        assert before and not re.search(r"\bm0\b", before[-1]), f"{name}: {before}; {line}"


def test_copies_through_a_resource_have_its_wait_states():
    # VALU write of an SGPR (v_readfirstlane of a part of the resource or of the scalar offset), then a vector memory
    # instruction that reads it: five wait states, an instruction being one and s_nop n being n + 1
    copies = [c for c in _copies_to_lds() if c[1].startswith("buffer_")]
    assert len(copies) >= 4
    for name, line, before in copies:
        states = sum(1 + (int(b.split()[1]) if b.startswith("s_nop") else 0) for b in before)
        assert states >= 5, f"{name}: {before}; {line}"
