"""The table that tells the 8-bit decode's joining kernel which warps have shares of a unit: an entry that was never written becomes
neither an address nor a number of turns.  No GPU needed."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda_ltc_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "kv8_shares.h"
int main() {
    const int32_t odd[] = {INT32_MIN, INT32_MIN + 1, -2000000000, -3, -1, 0, 1, 2, 5, 6, 7, 8, 100, 2367, 2368, 2369, 1 << 20, 0x3f800000,
                           0x7fc00000, INT32_MAX - 1, INT32_MAX};
    const int32_t sizes[] = {0, 1, 2, 7, 8, 2368, INT32_MAX};
    int wrong = 0, taken = 0;
    for (int32_t first : odd)
        for (int32_t more : odd)
            for (int32_t warps : sizes) {
                // in 64 bits: both are numbers of warps, and the last of them is one
                const bool want = first >= 0 && more >= 0 && (int64_t)first + more < warps;
                const bool got = ltca::shares_are_there(first, more, warps);
                wrong += want != got;
                taken += got;
            }
    printf("%d %d\n", wrong, taken);
}
"""


def test_only_warps_that_there_are(tmp_path):
    src = tmp_path / "s.cpp"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-fsanitize=undefined", "-I", CSRC, str(src), "-o", str(tmp_path / "s")])
    wrong, taken = map(int, subprocess.check_output([str(tmp_path / "s")]).split())
    assert wrong == 0 and taken > 50


def test_the_join_asks_before_it_forms_an_address():
    with open(os.path.join(CSRC, "kv8_decode.cu")) as f:
        text = f.read()
    join = text[text.index("kv8_decode_join_kernel("):text.index("struct Plan")]
    read, asked = join.index("a.shares["), join.index("shares_are_there(who.x, who.y, a.warps)")
    used = [m.start() for m in re.finditer(r"who\.[xy]", join) if not asked <= m.start() <= asked + 60]
    assert read < asked < min(used)
