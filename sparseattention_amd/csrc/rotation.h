// Parameters of the kernels that norm and rotate the rows of heads (rotate.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sa {

struct Rotation {
    const double *frequencies;  // [R / 2], radians per position
    const int32_t *axes;        // [R / 2], or null: 0
    const void *positions;      // [axes, B, S] int32 or int64
    int64_t position_strides[3];
    int positions_64, num_axes;
    int R, interleaved;
    const void *q_weight, *k_weight;  // [D], or null: no norm
    int weight_dtype;
    float eps;
};

struct RotateRows {
    const void *x;   // rows, or null (backward without a norm)
    const void *dy;  // backward: gradients of the outputs
    void *y;         // outputs; backward: gradients of x
    void *dw;        // backward: gradient of the weights, or null
    int64_t xs[3], dys[3], ys[3];  // b, h, token strides in elements
    int H;
};
struct RotateParams {
    Rotation r;
    RotateRows q, k;
    int B, S, D;
    int splits, heads;  // waves that share a group of tokens, heads of each (set by the launch)
    float *parts;       // backward: [workgroups][2][D], a workgroup's sums for the weights
    int groups;         // its workgroups
};
// Workgroups of the forward, of 256.
int64_t rotate_groups(int B, int S, int heads, int D);
hipError_t launch_rotate(RotateParams p, int dtype, hipStream_t stream);
// Workgroups of the backward.
int rotate_backward_groups(int B, int S, int heads, int D);
hipError_t launch_rotate_backward(RotateParams p, int dtype, hipStream_t stream);

}  // namespace sa
