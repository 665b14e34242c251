"""How verify_drafts cuts rows up (csrc/verify_plan.h), compiled for the host: parts, quarters and runs hold every value once, four at a time from multiples of four on."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparseattention_amd", "csrc")
PROGRAM = r"""
#include "verify_plan.h"
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>
using namespace sa;
#define CHECK(x) if (!(x)) { printf("B %d, V %d, parts %d, each %d, run %d: %s\n", B, V, p.parts, p.each, run, #x); return 1; }
// a: vocabularies, with every batch up to 1100 and some beyond
int main(int n, char **a) {
    for (int i = 1; i < n; i++) {
        const int V = atoi(a[i]);
        std::set<int> seen;
        for (int j = 1; j <= 1104; j++) {
            const int B = j <= 1100 ? j : j == 1101 ? 4096 : j == 1102 ? 200000 : j == 1103 ? 1 << 30 : 0x7fffffff;
            const VerifyPlan p = verify_plan(B, V);
            const int quarter = p.each / kVerifyWaves, run = verify_run(quarter);
            CHECK(p.parts >= 1 && p.parts <= kVerifyMostParts && p.each > 0 && p.each <= kVerifyMostEach);
            CHECK((int64_t)p.parts * p.each >= V && (int64_t)(p.parts - 1) * p.each < V);
            CHECK(p.each % kVerifyStep == 0 && quarter * kVerifyWaves == p.each && quarter % 4 == 0 && run % 4 == 0);
            if (!seen.insert(p.each).second) continue;
            std::vector<int> summed(V), searched(V);
            for (int part = 0; part < p.parts; part++)
                for (int k = 0; k < kVerifyWaves; k++) {
                    const int from = part * p.each, q0 = from + k * quarter, q1 = std::min(q0 + quarter, V);
                    for (int lane = 0; lane < 64; lane++)  // a wave's sum
                        for (int v = q0 + 4 * lane; v < q1; v += 256) {
                            CHECK((v - from) % 4 == 0);
                            for (int e = v; e < std::min(v + 4, V); e++) { CHECK(e < q1); summed[e]++; }
                        }
                    for (int t = 0; t < kVerifyThreads; t++)  // the search, a run a thread
                        for (int v = q0 + t * run; v < std::min(q0 + t * run + run, q1); v += 4) {
                            CHECK((v - from) % 4 == 0);
                            for (int e = v; e < std::min(v + 4, V); e++) { CHECK(e < q1); searched[e]++; }
                        }
                }
            for (int v = 0; v < V; v++) CHECK(summed[v] == 1 && searched[v] == 1);
        }
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "p.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(d / "p.cpp"), "-o", str(d / "p")], check=True)
    return str(d / "p")


@pytest.mark.parametrize("V", [1, 3, 1024, 2049, 5000, 9300, 31000, 32000, 50257, 65537, 90001, 100000, 100352, 128256, 131072, 151936, 200064, 1 << 20, (1 << 21) - 1, 1 << 21])
def test_every_value_once(program, V):
    r = subprocess.run([program, str(V)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
