// Trees of drafted tokens, given by each node's parent.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sa {
namespace {

// Node `lane` of a tree of n <= 64 nodes given by their parents (an entry that is not below its own index and at least 0: none): a bit for itself
// and for each of its ancestors.  The ways up double in six steps.
__device__ __forceinline__ uint64_t tree_ancestors(const int32_t *parents, int64_t stride, int n, int lane) {
    int up = lane < n ? parents[lane * stride] : -1;
    if (up < 0 || up >= lane) up = -1;
    uint64_t bits = 1ull << lane;
#pragma unroll
    for (int step = 0; step < 6; step++) {
        const int from = up < 0 ? lane : up;
        const uint64_t more = __shfl((unsigned long long)bits, from);
        const int next = __shfl(up, from);
        bits |= more;
        up = up < 0 ? -1 : next;
    }
    return bits;
}

}  // namespace
}  // namespace sa
