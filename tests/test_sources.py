"""Rules of the hardware that the compiler does not see to inside inline asm,
checked in the sources' text and in the instructions of the built library."""
import glob
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "proxima_amd", "libproxima_hip.so")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def test_m0_has_its_wait_state_before_a_copy_to_lds():
    # SALU write of m0, then a load to LDS that takes its address from it: one wait state between them
    copies = 0
    for path in sorted(glob.glob(os.path.join(ROOT, "proxima_amd", "csrc", "*.h*"))):
        for text in re.findall(r'asm volatile\(((?:\s*"[^"]*")+)', open(path).read()):
            lines = "".join(re.findall(r'"([^"]*)"', text)).replace("\\t", "").split("\\n")
            for before, line in zip([""] + lines, lines):
                if re.search(r"\blds\b|_load_lds_", line):
                    copies += 1
                    assert before and not re.search(r"\bm0\b", before), f"{os.path.basename(path)}: {before}; {line}"
    assert copies >= 6


def _sgprs(text):
    found = set()
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        found |= set(range(int(a), int(b) + 1))
    return found | {int(a) for a in re.findall(r"\bs(\d+)\b", text)} | ({"vcc"} if "vcc" in text else set())


VMEM = ("buffer_", "global_", "flat_", "scratch_")


def too_near(lines):
    """(copies to LDS, [violations]) of a listing: a vector memory instruction needs five wait states after a vector
    instruction that wrote one of its scalar registers, a copy to LDS one after a write of m0. An instruction is one
    state, s_nop n is n + 1; a taken branch is longer than any of them."""
    copies, bad, recent = 0, [], []  # recent: (instruction, scalar registers that a vector instruction wrote, states)
    for line in lines:
        line = line.split("//")[0].strip()
        if not line or line.endswith(":"):
            continue
        op, _, args = line.partition(" ")
        if op.startswith(VMEM):
            needs, states = _sgprs(args), 0
            for before, wrote, length in reversed(recent):
                if states >= 5:
                    break
                if wrote & needs:
                    bad.append((before, line))
                states += length
            if args.endswith(" lds") or "_load_lds_" in op:
                copies += 1
                if recent and re.match(r"s_\w+ m0,", recent[-1][0]):
                    bad.append((recent[-1][0], line))
        wrote = set()
        if op.startswith(("v_readfirstlane", "v_readlane", "v_cmp")):
            wrote = _sgprs(args.split(",")[0])
        elif op.startswith("v_") and ("_co_" in op or op.startswith("v_div_scale")):
            wrote = _sgprs(args.split(",")[1])
        recent = recent[-6:] + [(line, wrote, int(args, 0) + 1 if op == "s_nop" else 1)]
    return copies, bad


def test_the_check_finds_what_is_too_near():
    copy = "buffer_load_dwordx4 v75, s[12:15], s46 offen lds"
    near = ["v_readfirstlane_b32 s14, v73", "s_mov_b32 s15, s23", "s_or_b32 s1, s0, 1", "s_mov_b32 m0, s20", "s_nop 0"]
    assert too_near(near + [copy]) == (1, [(near[0], copy)])
    assert too_near(near[:1] + ["s_nop 0"] + near[1:] + [copy]) == (1, [])
    assert too_near(near[:3] + ["s_nop 1"] + near[3:4] + [copy]) == (1, [(near[3], copy)])
    assert too_near(["v_cmp_gt_f32_e64 s[46:47], v0, v1", copy])[1]
    assert too_near(["v_add_co_u32 v0, s[12:13], v1, v2", copy])[1]
    assert not too_near(["v_readfirstlane_b32 s16, v73", copy])[1]


def test_instructions_of_the_built_library_keep_their_distances(tmp_path):
    if not os.path.exists(LIB) or not os.path.exists(OBJDUMP):
        pytest.skip("no library, or no llvm-objdump")
    shutil.copy(LIB, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", os.path.basename(LIB)], cwd=tmp_path, check=True, capture_output=True)
    copies = 0
    for code in sorted(glob.glob(str(tmp_path / "*gfx950"))):
        listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", code], check=True,
                                 capture_output=True, text=True).stdout
        more, bad = too_near(listing.splitlines())
        assert not bad, bad[:5]
        copies += more
    assert copies > 1000
