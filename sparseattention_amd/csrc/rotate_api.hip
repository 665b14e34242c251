// C ABI of the norms and position rotation of queries and keys: argument validation and dispatch.  The declarations and their contracts live in
// include/sparseattn.h.
#include <hip/hip_runtime.h>

#include "rotation_api.h"

namespace {

using sa::fail;

// Rows of runs of 4 elements: unit last stride, the others and the address multiples of 16 bytes.
int head_rows(const char *who, const char *name, const void *p, const int64_t *s, int dtype, int64_t (&out)[3]) {
    if (!p || !s) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null %s", who, name);
    const int per16 = dtype == SA_DTYPE_FP32 ? 4 : 8;
    if (s[3] != 1 || s[0] % per16 || s[1] % per16 || s[2] % per16 || !sa::rotation_aligned(p, 16))
        return fail(SA_ERR_UNSUPPORTED, "%s: %s needs a contiguous last dimension, strides of multiples of 16 bytes and 16-byte alignment", who, name);
    for (int i = 0; i < 3; i++) out[i] = s[i];
    return SA_OK;
}

int sizes(const char *who, int B, int Hq, int H, int S, int D, int dtype) {
    if (B <= 0 || Hq <= 0 || H <= 0 || S <= 0) return fail(SA_ERR_INVALID_ARGUMENT, "%s: sizes must be positive (got B %d, heads %d and %d, S %d)", who, B, Hq, H, S);
    if ((int64_t)B * S > 0x7fffffff || Hq > (1 << 20) || H > (1 << 20))
        return fail(SA_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens or 2^20 heads", who);
    if (dtype != SA_DTYPE_BF16 && dtype != SA_DTYPE_FP16 && dtype != SA_DTYPE_FP32)
        return fail(SA_ERR_UNSUPPORTED, "%s: dtype %d not supported (bf16, fp16 and float32 are)", who, dtype);
    if (D <= 0 || D > 256 || D % 8) return fail(SA_ERR_UNSUPPORTED, "%s: head dim %d not supported (multiples of 8 up to 256 are)", who, D);
    return SA_OK;
}

int launched(const char *who, hipError_t e) {
    return e == hipSuccess ? SA_OK : fail(SA_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
}

#define SA_TRY(x)                            \
    do {                                     \
        if (const int rc_ = (x)) return rc_; \
    } while (0)

}  // namespace

extern "C" {

int sa_rotate_heads(const void *q, const int64_t q_strides[4], const void *k, const int64_t k_strides[4], void *q_out, const int64_t q_out_strides[4],
                    void *k_out, const int64_t k_out_strides[4], const sa_rotation *rotation, int B, int Hq, int H, int S, int D, int dtype, void *stream) {
    const char *who = "sa_rotate_heads";
    sa::RotateParams p{};
    SA_TRY(sizes(who, B, Hq, H, S, D, dtype));
    SA_TRY(sa::rotation_of(who, rotation, D, dtype, false, p.r));
    SA_TRY(head_rows(who, "q", q, q_strides, dtype, p.q.xs));
    SA_TRY(head_rows(who, "k", k, k_strides, dtype, p.k.xs));
    SA_TRY(head_rows(who, "q_out", q_out, q_out_strides, dtype, p.q.ys));
    SA_TRY(head_rows(who, "k_out", k_out, k_out_strides, dtype, p.k.ys));
    p.q.x = q, p.q.y = q_out, p.q.H = Hq;
    p.k.x = k, p.k.y = k_out, p.k.H = H;
    p.B = B, p.S = S, p.D = D;
    if (sa::rotate_groups(B, S, Hq + H, D) > sa::kMostGroups256) return fail(SA_ERR_UNSUPPORTED, "%s: more than 2^24 - 1 workgroups", who);
    return launched(who, sa::launch_rotate(p, dtype, static_cast<hipStream_t>(stream)));
}

size_t sa_rotate_heads_bwd_workspace_bytes(int B, int Hq, int H, int S, int D) {
    if (B <= 0 || Hq <= 0 || H <= 0 || S <= 0 || D <= 0 || D > 256 || Hq > (1 << 20) || H > (1 << 20) || (int64_t)B * S > 0x7fffffff) return 0;
    return (size_t)sa::rotate_backward_groups(B, S, Hq + H, D) * 2 * D * sizeof(float);
}

int sa_rotate_heads_bwd(const void *dq_out, const int64_t dq_out_strides[4], const void *dk_out, const int64_t dk_out_strides[4], const void *q,
                        const int64_t q_strides[4], const void *k, const int64_t k_strides[4], void *dq, const int64_t dq_strides[4], void *dk,
                        const int64_t dk_strides[4], void *dq_weight, void *dk_weight, const sa_rotation *rotation, void *workspace, size_t workspace_bytes,
                        int B, int Hq, int H, int S, int D, int dtype, void *stream) {
    const char *who = "sa_rotate_heads_bwd";
    sa::RotateParams p{};
    SA_TRY(sizes(who, B, Hq, H, S, D, dtype));
    SA_TRY(sa::rotation_of(who, rotation, D, dtype, false, p.r));
    SA_TRY(head_rows(who, "dq_out", dq_out, dq_out_strides, dtype, p.q.dys));
    SA_TRY(head_rows(who, "dk_out", dk_out, dk_out_strides, dtype, p.k.dys));
    SA_TRY(head_rows(who, "dq", dq, dq_strides, dtype, p.q.ys));
    SA_TRY(head_rows(who, "dk", dk, dk_strides, dtype, p.k.ys));
    if (p.r.q_weight) SA_TRY(head_rows(who, "q", q, q_strides, dtype, p.q.xs));
    if (p.r.k_weight) SA_TRY(head_rows(who, "k", k, k_strides, dtype, p.k.xs));
    if ((dq_weight && !p.r.q_weight) || (dk_weight && !p.r.k_weight)) return fail(SA_ERR_INVALID_ARGUMENT, "%s: gradient of a weight that is not there", who);
    const size_t align = p.r.weight_dtype == SA_DTYPE_FP32 ? 4 : 2;
    if (!sa::rotation_aligned(dq_weight, align) || !sa::rotation_aligned(dk_weight, align))
        return fail(SA_ERR_UNSUPPORTED, "%s: gradients of weights must be aligned to their elements", who);
    p.q.x = q, p.q.dy = dq_out, p.q.y = dq, p.q.dw = dq_weight, p.q.H = Hq;
    p.k.x = k, p.k.dy = dk_out, p.k.y = dk, p.k.dw = dk_weight, p.k.H = H;
    p.B = B, p.S = S, p.D = D;
    if (dq_weight || dk_weight) {
        const size_t need = sa_rotate_heads_bwd_workspace_bytes(B, Hq, H, S, D);
        if (!workspace || workspace_bytes < need || !sa::rotation_aligned(workspace, 4))
            return fail(SA_ERR_WORKSPACE, "%s: workspace of %zu bytes required (got %zu)", who, need, workspace ? workspace_bytes : (size_t)0);
        p.parts = static_cast<float *>(workspace);
    }
    return launched(who, sa::launch_rotate_backward(p, dtype, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
