"""Who takes which chunks of a batch in the paged attention (csrc/paged_pieces.h), compiled for the host: every chunk of every plane once, by
segments that workgroups can hand over and add up."""
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparseattention_amd", "csrc")
PROGRAM = r"""
#include "paged_pieces.h"
#include <cstdio>
#include <cstdlib>
#include <vector>
// a: compute units, rows, D, chunks of the table, planes of a unit, then T of every unit.  Out: groups, cuts; a line per segment
int main(int n, char **a) {
    const int cus = atoi(a[1]), R = atoi(a[2]), D = atoi(a[3]), chunks = atoi(a[4]), M = atoi(a[5]);
    std::vector<unsigned> T;
    unsigned total = 0, longest = 0;
    for (int i = 6; i < n; i++) {
        T.push_back(atoi(a[i]) > 1 ? atoi(a[i]) : 1);
        total += T.back() * M;
        if (T.back() > longest) longest = T.back();
    }
    const sa::PagedDecodePlan plan = sa::paged_decode_plan((int64_t)T.size() * M, R, D, chunks, cus);
    const sa::PagedShare s = sa::paged_share(total, T.size() * M, plan.groups, longest, plan.parts);
    unsigned row = 0;
    for (unsigned t : T) row += sa::paged_row_length(s, t) * M;
    printf("%d %d %u %u\n", plan.groups, (int)s.cuts, row, s.share);
    for (unsigned block = 0; block < (unsigned)plan.groups; block++) {
        const int me = sa::paged_piece(block, s.cuts ? row : plan.groups);
        if (me < 0) continue;
        const unsigned piece = s.cuts ? 1 : s.share, x0 = piece * me;
        const unsigned x1 = x0 + piece < row ? x0 + piece : row;
        for (unsigned x = x0; x < x1;) {
            unsigned base = 0, u = 0;
            while (x >= base + sa::paged_row_length(s, T[u]) * M) base += sa::paged_row_length(s, T[u++]) * M;
            const unsigned row_T = sa::paged_row_length(s, T[u]), m = (x - base) / row_T;
            x += sa::paged_coming(s, x - base - m * row_T);
            if (x >= x1) break;
            const unsigned at = x - base - m * row_T;
            const sa::PagedSegment g = sa::paged_segment(s, T[u], row_T, at, x1 - x);
            const sa::PagedRange r = sa::paged_range(s, x - at, row_T);
            printf("%d %u %u %d %d %d %d\n", me, u, m, g.off, g.n, r.first, r.parts);
            x += s.cuts ? 1 : g.n;
        }
    }
}
"""


@pytest.fixture(scope="module")
def pieces(tmp_path_factory):
    d = tmp_path_factory.mktemp("pieces")
    (d / "p.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(d / "p.cpp"), "-o", str(d / "p")], check=True)

    def of(*args):
        out = subprocess.run([str(d / "p"), *map(str, args)], check=True, capture_output=True, text=True).stdout
        rows = [tuple(map(int, ln.split())) for ln in out.splitlines()]
        return rows[0], rows[1:]
    return of


def check(pieces, cus, R, D, chunks, M, T):
    (groups, cuts, row, share), segments = pieces(cus, R, D, chunks, M, *T)
    assert groups % 8 == 0 and (not cuts or row <= groups)
    planes, of_group, slots, words = {}, {}, set(), set()
    for me, u, m, off, n, first, parts in segments:
        t = max(T[u], 1)
        assert 0 <= off and 1 <= n <= t - off
        planes.setdefault((u, m), []).append((off, n, me))
        of_group[me] = of_group.get(me, 0) + n
        if n < t:  # a part: two at most of a workgroup, each in a place of its own, its word in the plane's row of words
            slot = 2 * me + (off == 0)
            assert 0 <= me - first < parts <= 128 and slot not in slots
            slots.add(slot)
            word = u * M + m + me
            assert word not in words and word < len(T) * M + groups
            words.add(word)
            assert slot == 2 * first + 1 if me == first else slot == 2 * (first + (me - first))
        else:
            assert parts == 1
    for u, t in enumerate(T):
        for m in range(M):
            got = sorted(planes.pop((u, m)))
            at = 0
            for off, n, _ in got:
                assert off == at
                at += n
            assert at == max(t, 1)
            assert [g for _, _, g in got] == list(range(got[0][2], got[0][2] + len(got)))
    assert not planes and max(of_group.values()) <= share


@pytest.mark.parametrize("cus,R,D,chunks,M,T", [
    (256, 1, 64, 1, 1, [0]), (256, 4, 128, 63, 8, [63]), (256, 4, 128, 4096, 8, [4096]), (256, 32, 64, 512, 4, [129] * 16),
    (256, 1, 128, 32768, 1, [32768]), (256, 16, 128, 1024, 1, [1024] * 16), (256, 224, 128, 400, 56, [400, 3, 0, 150]),
    (256, 8, 256, 2, 8, [1, 2] * 150), (1, 1, 64, 100, 1, [100, 7]), (7, 33, 128, 64, 3, [64, 0, 1, 5] * 9), (256, 4, 128, 1024, 8, [1024, 700] * 16)])
def test_every_chunk_once(pieces, cus, R, D, chunks, M, T):
    check(pieces, cus, R, D, chunks, M, T)


@pytest.mark.parametrize("seed", range(40))
def test_drawn_batches(pieces, seed):
    rng = random.Random(seed)
    top = round(2 ** rng.uniform(0, 11))
    T = [rng.randint(0, top) for _ in range(round(2 ** rng.uniform(0, 8)))]
    R = rng.choice([1, 4, 8, 16, 17, 32, 64, 200])
    check(pieces, rng.choice([1, 8, 64, 256, 256, 304]), R, rng.choice([64, 128, 256]), max(T + [1]) + rng.randint(0, 50), rng.choice([1, 2, 8, 12]) * -(-R // 32), T)
