"""How groups are divided into parts (proxima_amd/csrc/groups.hpp), compiled
for the host and compared with whole-number arithmetic of any size."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROWS_MAX = 2 ** 31 - 1024

PROGRAM = r"""
#include <cstdio>
#include "groups.hpp"
int main() {
  long long size, limit;
  while (scanf("%lld %lld", &size, &limit) == 2) {
    const int parts = pxg::group_parts((int)size, (int)limit);
    printf("%d %d %llu %llu\n", parts, parts > 1 ? pxg::group_part_length((int)size, parts) : (int)size,
           (unsigned long long)pxg::group_parts_max(size, 1, limit),
           (unsigned long long)pxg::group_slots_max(size, 1, limit));
  }
}
"""


@pytest.fixture(scope="module")
def divide(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    at = tmp_path_factory.mktemp("groups")
    source, program = at / "groups.hip", at / "groups"
    source.write_text(PROGRAM)
    # as the device computes: whole numbers wrap
    subprocess.run([hipcc, "-O0", "-fwrapv", "-std=c++17", "--offload-host-only", "-I",
                    os.path.join(ROOT, "proxima_amd", "csrc"), str(source), "-o", str(program)],
                   check=True, capture_output=True)

    def run(pairs):
        text = subprocess.run([str(program)], input="\n".join(f"{a} {b}" for a, b in pairs), text=True, check=True,
                              capture_output=True).stdout
        return [tuple(int(v) for v in line.split()) for line in text.splitlines()]

    return run


def test_parts_of_any_length(divide):
    sizes = [1, 2, 63, 64, 65, 1000, 16_384, 10 ** 6, 1_500_000_000, 2_090_000_000, ROWS_MAX - 1, ROWS_MAX]
    limits = [0, 128, 192, 4096, 999_936, 65_312_512, 750_000_000, 2 ** 30, ROWS_MAX // 64 * 64]
    pairs = [(s, m) for s in sizes for m in limits]
    got = divide(pairs)
    assert len(got) == len(pairs)
    for (size, limit), (parts, length, most, slots) in zip(pairs, got):
        want = -(-size // limit) if limit and size > limit else 1
        assert parts == want, (size, limit)
        if parts > 1:
            each = -(-size // parts)
            assert length == -(-each // 64) * 64, (size, limit)
            assert parts * length >= size          # every row is in a part
            assert parts <= most and parts <= slots  # and every part has a place and a slot
