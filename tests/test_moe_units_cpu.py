"""How many thread blocks a pass of a mixture-of-experts layer takes (csrc/qx_moe_units.h), against its units counted one by
one: one for each of the up projection at least, no more than there are units, and no phase with more than two of its units
to a block for want of blocks."""

import os
import random
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "quixicore-cpu_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include "qx_moe_units.h"
int main() {
  long long tokens, places, dim, inner;
  while (std::scanf("%lld %lld %lld %lld", &tokens, &places, &dim, &inner) == 4) {
    std::printf("%lld\n", qx::moe::pass_blocks(tokens, places, dim, inner));
  }
}
"""


def test_no_phase_wants_for_blocks(tmp_path):
    source, program = tmp_path / "units.cpp", tmp_path / "units"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(source), "-o", str(program)], check=True)
    rng = random.Random(4)
    # (narrow experts among them, where the down projection has the most units)
    cases = [(1, 8, 2048, 768), (1, 8, 1536, 512), (1, 1, 4096, 256), (1, 1, 65536, 32), (1, 8, 2048, 1024), (64, 8, 4096, 1536)]
    for _ in range(500):
        dim, inner = (32 * int(2 ** rng.uniform(0, 11)) for _ in range(2))
        cases.append((rng.randint(1, 128), rng.randint(1, 64), dim, inner))
    lines = "".join("%d %d %d %d\n" % case for case in cases)
    done = subprocess.run([str(program)], input=lines, capture_output=True, text=True, check=True)
    for (tokens, places, dim, inner), blocks in zip(cases, map(int, done.stdout.split())):
        up, down = (tokens * places * len(range(0, width, step)) for width, step in ((inner, 32), (dim, 64)))
        combine = tokens * len(range(0, dim, 1024))
        assert up <= blocks <= up + down + combine and 2 * blocks >= max(down, combine), (tokens, places, dim, inner, blocks)
