"""Room of the epilogue groups of the gate/up product (csrc/token_slots.h), compiled for the host: no two tokens of a tile share
a slot, and a group in one tile shares none with the other group in a tile of any other size, which it may still be working on."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascend_kernel_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "token_slots.h"
using namespace b200moe;

int main() {
    for (int n = 32; n <= kTileTokens; n += 32)      // tokens of the first group's tile
        for (int m = 32; m <= kTileTokens; m += 32)  // and of the second's
            for (int i = 0; i < n / 2; ++i) {
                const int at = token_slot(0, i);
                if (at < 0 || at >= kTileTokens) return std::printf("token %d of %d has no slot\n", i, n), 1;
                if (i && at <= token_slot(0, i - 1)) return std::printf("two tokens of %d share a slot\n", n), 1;
                for (int j = 0; j < m / 2; ++j) {
                    const int other = token_slot(1, j);
                    if (other < 0 || other >= kTileTokens) return std::printf("token %d of %d has no slot\n", j, m), 1;
                    if (other == at) return std::printf("tiles of %d and %d tokens meet in slot %d\n", n, m, at), 1;
                }
            }
    return 0;
}
"""


def test_the_groups_never_meet(tmp_path):
    src, exe = tmp_path / "slots.cpp", tmp_path / "slots"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_the_kernel_numbers_its_tokens_so():
    text = open(os.path.join(CSRC, "grouped_gemm_fp8_block.cu")).read()
    assert "const int slots = token_slot(wg, 0);" in text
    used = re.findall(r"(?:e\.tops\[\(|\(e\.tops\)\[|\(e\.quantizers\)\[)(\w+)", text)
    assert len(used) == 4 and set(used) == {"slots"}
