// How verify.hip cuts a row of V probabilities up.  Plain C++, so that it can be looked at on the host.
//
// A row is `parts` parts of `each` values, a workgroup each, in quarters, a wave each.  Where the next token is looked for a quarter is in runs, a thread each.  Values are
// read four at a time, and so are the bits of rejected tokens, of which 32 are in a word: parts, quarters and runs begin at multiples of 4 of their part and nobody goes beyond
// the end of their own but for a row's last values, behind which there are none.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define SA_VERIFY_FN __host__ __device__ __forceinline__
#else
#define SA_VERIFY_FN inline
#endif

namespace sa {

constexpr int kVerifyThreads = 256, kVerifyWaves = kVerifyThreads / 64;
constexpr int kVerifyStep = 4 * kVerifyThreads;  // parts are multiples of: four values a thread
constexpr int kVerifyMostParts = 64;             // of a row, which one wave adds up
constexpr int kVerifyMostEach = 1 << 15;         // values of a part, which have a bit in LDS each
static_assert(kVerifyMostEach % kVerifyStep == 0 && kVerifyStep / kVerifyWaves % 4 == 0, "quarters of a part begin at multiples of 4");

struct VerifyPlan {
    int parts, each;
};
// Parts of 2048 values at least (and no more than have a bit in LDS), as many as make 1024 workgroups of all rows.
inline VerifyPlan verify_plan(int B, int V) {
    const int64_t wanted = ((int64_t)B + 1023) / B, want = wanted < kVerifyMostParts ? wanted : kVerifyMostParts, least = 2048;
    int64_t each = (V + want - 1) / want;
    each = each < least ? least : each < kVerifyMostEach ? each : kVerifyMostEach;
    each = (each + kVerifyStep - 1) / kVerifyStep * kVerifyStep;
    return {(int)((V + each - 1) / each), (int)each};
}

// Values of a thread's run of a quarter: a multiple of 4, so the last threads may have fewer or none.
SA_VERIFY_FN int verify_run(int quarter) { return ((quarter + kVerifyThreads - 1) / kVerifyThreads + 3) / 4 * 4; }

}  // namespace sa
