"""How many heads a thread of the rotary positions turns (csrc/rotary_rule.hpp), compiled for the host: on the faster side of what was measured."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = r"""
#include <cstdio>
#include <cstdlib>
#include "rotary_rule.hpp"
int main(int argc, char** argv) {
    for (int i = 1; i + 4 < argc; i += 5)
        printf("%d ", fattn::rotary_heads_per_thread(atof(argv[i]), atoi(argv[i + 1]), atoi(argv[i + 2]), atoi(argv[i + 3]), atoi(argv[i + 4])));
}
"""


def test_rule(tmp_path):
    src, exe = tmp_path / "rule.cpp", tmp_path / "rule"
    src.write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-I" + os.path.join(ROOT, "flame_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    # rows, chunks of a head, heads; wide, near, fp32, bounds; heads per thread.  D = 128, 40 heads where nothing else is said
    cases = [(512, 16, 40, 1, 1, 0, 0, 1), (1024, 16, 40, 1, 1, 0, 0, 4), (65536, 16, 40, 1, 1, 0, 1, 4),             # neighbours, bf16
             (512, 32, 40, 1, 1, 1, 0, 4), (512, 32, 20, 1, 1, 1, 0, 1), (1024, 32, 20, 1, 1, 1, 1, 4),               # fp32
             (1024, 36, 40, 0, 0, 0, 0, 4), (4096, 67, 20, 0, 1, 1, 1, 4), (100, 84, 40, 0, 0, 0, 0, 1),              # narrow
             (2500, 8, 40, 1, 0, 0, 0, 1), (12593, 8, 40, 1, 0, 0, 0, 1), (32768, 8, 40, 1, 0, 0, 0, 1),              # halves, bf16, positions
             (1024, 8, 40, 1, 0, 0, 1, 1), (12593, 8, 40, 1, 0, 0, 1, 4), (131072, 8, 40, 1, 0, 0, 1, 4),             # bounds
             (13000, 16, 40, 1, 0, 1, 0, 1), (13000, 16, 40, 1, 0, 1, 1, 1)]                                          # halves, fp32
    args = [str(x) for rows, chunks, heads, *form, _ in cases for x in (rows * chunks * heads, *form)]
    out = subprocess.run([str(exe), *args], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in out] == [c[-1] for c in cases]
