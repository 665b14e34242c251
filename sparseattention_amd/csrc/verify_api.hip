// C ABI of the verification of drafted tokens: argument validation and dispatch.  The declarations and their contracts live in
// include/sparseattn.h.
#include <hip/hip_runtime.h>

#include "api_common.h"
#include "sparseattn.h"
#include "verify.h"

namespace {

using sa::fail;

constexpr size_t kWordBytes = 5 * 8;  // four sums and an arrival of each workgroup
constexpr int kNodes = 64, kMostTokens = sa::kVerifyMostParts * sa::kVerifyMostEach;

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
bool fits(int B, int n, int V) { return B > 0 && n > 0 && n <= kNodes && V > 0 && V <= kMostTokens; }
int64_t words(int B, int V) { return (int64_t)B * sa::verify_plan(B, V).parts; }

}  // namespace

extern "C" {

size_t sa_verify_drafts_workspace_bytes(int B, int n, int V) { return fits(B, n, V) ? (size_t)words(B, V) * kWordBytes : 0; }

int sa_verify_drafts(const void *target_probs, const int64_t target_strides[3], const void *draft_probs, const int64_t draft_strides[3], const void *tokens,
                     const int64_t tokens_strides[2], int tokens_64, const float *uniforms, const int64_t uniforms_strides[2], const int32_t *parents,
                     const int64_t parents_strides[2], const int32_t *counts, int32_t *path, int32_t *accepted, void *next_token, int B, int n, int V, int dtype,
                     void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "sa_verify_drafts";
    if (!target_probs || !target_strides || !tokens || !tokens_strides || !uniforms || !uniforms_strides || !path || !accepted || !next_token)
        return fail(SA_ERR_INVALID_ARGUMENT, "%s: null argument", who);
    if ((draft_probs && !draft_strides) || (parents && !parents_strides)) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null strides", who);
    if (B <= 0 || n <= 0 || V <= 0) return fail(SA_ERR_INVALID_ARGUMENT, "%s: sizes must be positive (got B %d, n %d, V %d)", who, B, n, V);
    if (!fits(B, n, V)) return fail(SA_ERR_UNSUPPORTED, "%s: at most %d nodes and %d tokens (got n %d, V %d)", who, kNodes, kMostTokens, n, V);
    if (draft_probs && parents) return fail(SA_ERR_INVALID_ARGUMENT, "%s: the draft's probabilities go with chains (no parents)", who);
    if (dtype != SA_DTYPE_BF16 && dtype != SA_DTYPE_FP16 && dtype != SA_DTYPE_FP32)
        return fail(SA_ERR_UNSUPPORTED, "%s: dtype %d not supported (bf16, fp16 and float32 are)", who, dtype);
    const size_t size = dtype == SA_DTYPE_FP32 ? 4 : 2;
    if (target_strides[2] != 1 || (draft_probs && draft_strides[2] != 1) || !aligned(target_probs, size) || !aligned(draft_probs, size) ||
        !aligned(tokens, tokens_64 ? 8 : 4) || !aligned(next_token, tokens_64 ? 8 : 4))
        return fail(SA_ERR_UNSUPPORTED, "%s: probabilities need a contiguous last dimension, all tensors alignment to their elements", who);
    sa::VerifyParams p{};
    p.target = target_probs;
    p.draft = draft_probs;
    p.tokens = tokens;
    p.tokens_64 = tokens_64 != 0;
    p.uniforms = uniforms;
    p.parents = parents;
    for (int i = 0; i < 2; i++) {
        p.target_s[i] = target_strides[i];
        p.draft_s[i] = draft_probs ? draft_strides[i] : 0;
        p.tokens_s[i] = tokens_strides[i];
        p.uniforms_s[i] = uniforms_strides[i];
        p.parents_s[i] = parents ? parents_strides[i] : 0;
    }
    p.counts = counts;
    p.path = path;
    p.accepted = accepted;
    p.next = next_token;
    p.B = B;
    p.n = n;
    p.V = V;
    const sa::VerifyPlan plan = sa::verify_plan(B, V);
    p.parts = plan.parts;
    p.each = plan.each;
    const int64_t count = (int64_t)B * p.parts;
    if (count > sa::kMostGroups256) return fail(SA_ERR_UNSUPPORTED, "%s: more than 2^24 - 1 workgroups", who);
    const size_t need = (size_t)count * kWordBytes;
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
        return fail(SA_ERR_WORKSPACE, "%s: workspace of %zu bytes required, 16-byte aligned (got %zu)", who, need, workspace ? workspace_bytes : (size_t)0);
    p.sums = static_cast<double *>(workspace);
    p.arrivals = reinterpret_cast<uint64_t *>(p.sums + 4 * count);
    p.tag = sa::next_launch_tag() | 1;
    const hipError_t e = sa::launch_verify(p, dtype, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? SA_OK : fail(SA_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
}

}  // extern "C"
