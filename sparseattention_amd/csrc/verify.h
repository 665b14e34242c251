// Parameters of the kernel that verifies drafted tokens (verify.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sa {

constexpr int kVerifyMostParts = 64;      // of a row, which one wave adds up
constexpr int kVerifyMostEach = 1 << 15;  // values of a part, which have a bit in LDS each

struct VerifyParams {
    const void *target, *draft;  // [B, n, V]; draft or null
    int64_t target_s[2], draft_s[2];
    const void *tokens;  // [B, n] int32 or int64
    int64_t tokens_s[2];
    const float *uniforms;  // [B, n]
    int64_t uniforms_s[2];
    const int32_t *parents;  // [B, n], or null: a chain
    int64_t parents_s[2];
    const int32_t *counts;  // [B], or null: n
    int B, n, V, tokens_64;
    int32_t *path, *accepted;  // [B, n], [B]
    void *next;                // [B], of the tokens' type
    int parts, each;           // workgroups of a row, and its values for each
    double *sums;              // [B, parts, 4]
    uint64_t *arrivals;        // [B, parts] words (all_arrived)
    uint64_t tag;
};
// Sets parts and each.
void verify_plan(VerifyParams &p);
hipError_t launch_verify(const VerifyParams &p, int dtype, hipStream_t stream);

}  // namespace sa
