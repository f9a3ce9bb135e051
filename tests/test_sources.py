"""Rules of the hardware that the compiler does not see to inside inline asm,
checked in the sources' text."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_m0_has_its_wait_state_before_a_copy_to_lds():
    # SALU write of m0, then a load to LDS that takes its address from it: one wait state between them
    copies = 0
    for path in sorted(glob.glob(os.path.join(ROOT, "proxima_amd", "csrc", "*.h*"))):
        for text in re.findall(r'asm volatile\(((?:\s*"[^"]*")+)', open(path).read()):
            lines = "".join(re.findall(r'"([^"]*)"', text)).replace("\\t", "").split("\\n")
            for before, line in zip([""] + lines, lines):
                if re.search(r"\blds\b|_load_lds_", line):
                    copies += 1
                    assert not re.search(r"\bm0\b", before), f"{os.path.basename(path)}: {before}; {line}"
    assert copies >= 6
