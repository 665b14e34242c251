// Parameters of the kernel that verifies drafted tokens (verify.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "verify_plan.h"

namespace sa {

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
    int parts, each;           // workgroups of a row, and its values for each (verify_plan.h)
    double *sums;              // [B, parts, 4]
    uint64_t *arrivals;        // [B, parts] words (all_arrived)
    uint64_t tag;
};
hipError_t launch_verify(const VerifyParams &p, int dtype, hipStream_t stream);

}  // namespace sa
