"""CPU: the rule that shares the backward pass of norm and rotation out over blocks, compiled by itself: the blocks of both sides
together are never more than the workspace has rows for, and their tiles hold every token."""
import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "fast_polynomial_transcendentals_b200" / "csrc"
PROGRAM = r"""
#include <cstdio>
#include "fpt_qk_rope_plan.h"
using namespace fpt;
int main() {
    const uint32_t heads[] = {0, 1, 2, 3, 8, 32, 40, 130, 511, 512, 700, 1024, 2592, 65535};
    const uint32_t tokens[] = {1, 2, 3, 31, 147, 148, 149, 295, 296, 297, 591, 593, 1021, 4096, 8192, 100003, 131072, 780000, 2000003, 16777216, 1u << 30};
    long cases = 0;
    for (uint32_t groups : {8u, 16u, 32u, 64u})
        for (uint32_t pairs : {4u, 32u, 64u, 128u})
            for (uint32_t total : {2u, 264u, 296u, 304u})
                for (uint32_t q : heads)
                    for (uint32_t k : heads)
                        for (uint32_t t : tokens)
                            for (int far = 0; far < 2; ++far) {
                                if (!q && !k) continue;
                                BwdShare a{}, b{};
                                share_blocks(a, q, b, k, t, groups, pairs, total, [&](int, uint32_t n) { return !far || n == 1; });
                                ++cases;
                                bool good = (q ? a.blocks : 0) + (k ? b.blocks : 0) <= total;
                                const BwdShare* sides[2] = {&a, &b};
                                for (int s = 0; s < 2; ++s) {
                                    if (!(s ? k : q)) continue;
                                    const BwdShare& d = *sides[s];
                                    const uint32_t n = d.tile_tokens;
                                    good = good && d.blocks >= 1 && d.blocks <= d.tiles && n >= 1 && n <= groups && (n & (n - 1)) == 0 && n * pairs <= kBwdTrig &&
                                           uint64_t(d.tiles) * n >= t && uint64_t(d.tiles - 1) * n < t;
                                }
                                if (!good) {
                                    printf("groups %u pairs %u total %u heads %u + %u tokens %u: blocks %u + %u tiles %u + %u of %u, %u\n", groups, pairs, total, q, k,
                                           t, a.blocks, b.blocks, a.tiles, b.tiles, a.tile_tokens, b.tile_tokens);
                                    return 1;
                                }
                            }
    printf("%ld\n", cases);
}
"""


def test_blocks_fit_the_workspace(tmp_path):
    source, binary = tmp_path / "plan.cpp", tmp_path / "plan"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", f"-I{CSRC}", str(source), "-o", str(binary)], check=True, capture_output=True, text=True)
    ran = subprocess.run([str(binary)], capture_output=True, text=True, timeout=300)
    assert ran.returncode == 0, ran.stdout
    assert int(ran.stdout) > 100000
