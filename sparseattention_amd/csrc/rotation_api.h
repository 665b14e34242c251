// Checks of the C ABI's sa_rotation, for the entry points that take one.
#pragma once
#include "api_common.h"
#include "rotation.h"
#include "sparseattn.h"

namespace sa {
namespace {

bool rotation_aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// D columns of rows of `dtype`; B, S as the positions have them, which `own_positions` calls can do without.
int rotation_of(const char *who, const sa_rotation *r, int D, int dtype, bool own_positions, Rotation &out) {
    if (!r || !r->frequencies) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null rotation or frequencies", who);
    if (D <= 0 || D > 256 || D % 8) return fail(SA_ERR_UNSUPPORTED, "%s: head dim %d not supported (multiples of 8 up to 256 are)", who, D);
    if (r->R <= 0 || r->R > D || r->R % 8)
        return fail(SA_ERR_UNSUPPORTED, "%s: the rotated columns must be a multiple of 8 up to the head dim %d (got %d)", who, D, r->R);
    if (!(r->eps >= 0.f) || r->eps > 3e38f) return fail(SA_ERR_INVALID_ARGUMENT, "%s: eps must be finite and not negative", who);
    if (!r->positions && !own_positions) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null positions", who);
    if (r->num_axes <= 0) return fail(SA_ERR_INVALID_ARGUMENT, "%s: at least one axis of positions (got %d)", who, r->num_axes);
    if ((r->q_weight || r->k_weight) && r->weight_dtype != dtype && r->weight_dtype != SA_DTYPE_FP32)
        return fail(SA_ERR_UNSUPPORTED, "%s: weights must be of the rows' type or float32", who);
    if (!rotation_aligned(r->frequencies, 8) || !rotation_aligned(r->axes, 4) || !rotation_aligned(r->positions, r->positions_64 ? 8 : 4) ||
        !rotation_aligned(r->q_weight, r->weight_dtype == SA_DTYPE_FP32 ? 4 : 2) || !rotation_aligned(r->k_weight, r->weight_dtype == SA_DTYPE_FP32 ? 4 : 2))
        return fail(SA_ERR_UNSUPPORTED, "%s: rotation tensors must be aligned to their elements", who);
    out = {r->frequencies, r->axes, r->positions, {r->position_strides[0], r->position_strides[1], r->position_strides[2]},
           r->positions_64 != 0, r->num_axes, r->R, r->interleaved != 0, r->q_weight, r->k_weight, r->weight_dtype, r->eps};
    return SA_OK;
}

}  // namespace
}  // namespace sa
