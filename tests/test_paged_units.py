"""The search for the unit that a place of the row lies in (csrc/paged_pieces.h, paged_find_unit), compiled for the host, against looking at
every unit in turn."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparseattention_amd", "csrc")
PROGRAM = r"""
#include "paged_pieces.h"
#include <cstdio>
#include <random>
#include <vector>
int main() {
    std::mt19937 rng(1);
    long looked = 0;
    for (int U : {1, 2, 63, 64, 65, 127, 128, 129, 257, 300, 4095, 4096, 4097, 16384, 65537, 300000}) {
        std::vector<unsigned> first(U);
        unsigned at = 0;
        for (unsigned &x : first) {
            x = at;
            at += 1 + rng() % (U > 5000 ? 9 : 700);
        }
        for (unsigned M : {1u, 3u, 56u}) {
            for (int t = 0; t < 3000; t++) {
                const int u = rng() % U;  // a place in unit u: its first, its last or any
                const unsigned end = (u + 1 < U ? first[u + 1] : at) * M, begin = first[u] * M;
                const unsigned x0 = t % 3 == 0 ? begin : t % 3 == 1 ? end - 1 : begin + rng() % (end - begin);
                const int got = sa::paged_find_unit(U, [&](int from, int step, int left) {
                    int n = 0;
                    for (int lane = 0; lane < 64; lane++) {
                        const int i = from + lane * step < U - 1 ? from + lane * step : U - 1;
                        if (i < 0 || i >= U) return 1 << 20;
                        n += lane * step < left && first[i] * M <= x0;
                        looked++;
                    }
                    return n;
                });
                if (got != u) {
                    printf("U %d M %u x0 %u: %d, not %d\n", U, M, x0, got, u);
                    return 1;
                }
            }
        }
    }
    printf("%ld looked at\n", looked);
}
"""


def test_every_place_is_found(tmp_path):
    (tmp_path / "p.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}", str(tmp_path / "p.cpp"), "-o", str(tmp_path / "p")], check=True)
    out = subprocess.run([str(tmp_path / "p")], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr
