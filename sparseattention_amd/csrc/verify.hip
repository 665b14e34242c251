// Verification of drafted tokens against the target's probabilities, from given random numbers, on gfx950 (MI355X).  No counterpart in the reference.
//
// From node 0 on the children of the node at hand are tried in order.  A child with token x is accepted if
//     u * rest < p(x)      (rest = 1 less the p of the siblings rejected before it; p(x) = 0 for a token rejected before), or
//     u * q(x) < p(x)      (drafts drawn from q, in a chain),
// u its random number; then its own children are.  Where no child is accepted the sequence goes on with the first token v of
//     cumsum(r)(v) > u0 * sum(r),   r = p without the rejected tokens | max(p - q, 0) | p where none was rejected.
// The tests' numbers are of one value each: all of a sequence are read at once, a node a lane, and the walk is made in registers, by every
// workgroup of the sequence for itself.  What takes time is the row of r, which several workgroups add up in parts; the last to arrive looks up
// which part the token is in and goes through that again.  Probabilities are at most 32 bits wide and all that is done with them has 64: a row of 10^5
// has sums off by 2^-37 of it, in float32 by more than most of its values.  Bound by memory: p (and q) of one row a sequence.
//
// Measured (float32): 64 trees of 32 nodes, V = 131072: 21.6 us (V = 151936 24.1), of which the row's 33.5 MB take 6.6 at the rate of a copy; the rest is the chain walk, sum, hand-over,
// search, which alone takes 12.8 us for 8 chains of 6 nodes, V = 32000.  (Parts of 512 workgroups in all 24 us, of 2048 26; eight rows of four under way 33.)
#include "fwd_common.h"
#include "tree.h"
#include "verify.h"

namespace sa {
namespace {

typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

// A probability; what is none counts as 0.
__device__ __forceinline__ double chance(float x) { return x > 0.f && x < __builtin_inff() ? (double)x : 0.0; }
template <int DT>
__device__ __forceinline__ float value_at(const void *row, int64_t at) {
    if constexpr (DT == 2) return ((const float *)row)[at];
    else if constexpr (DT == 1) return (float)((const _Float16 *)row)[at];
    else return __uint_as_float((uint32_t)((const uint16_t *)row)[at] << 16);
}
// Values v .. v + 3 of a row of V, 0 behind its end.
template <int DT>
__device__ __forceinline__ void four(const void *row, int v, int V, float (&x)[4]) {
    if constexpr (DT == 2) {
        const float *const at = (const float *)row + v;
        if (v + 4 <= V && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
            const f32x4 w = *(const f32x4 *)at;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = w[i];
            return;
        }
    } else {
        const uint16_t *const at = (const uint16_t *)row + v;
        if (v + 4 <= V && (reinterpret_cast<uintptr_t>(at) & 7) == 0) {
            const u32x2 w = *(const u32x2 *)at;
            const uint32_t lo = w.x, hi = w.y;
            if constexpr (DT == 0) {
                x[0] = __uint_as_float(lo << 16), x[1] = __uint_as_float(lo & 0xffff0000u);
                x[2] = __uint_as_float(hi << 16), x[3] = __uint_as_float(hi & 0xffff0000u);
            } else {
                const f16x2 a = __builtin_bit_cast(f16x2, lo), b = __builtin_bit_cast(f16x2, hi);
                x[0] = (float)a.x, x[1] = (float)a.y, x[2] = (float)b.x, x[3] = (float)b.y;
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = v + i < V ? value_at<DT>(row, v + i) : 0.f;
}

__device__ __forceinline__ double of_lane(double x, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double sum_upto(double x, int lane) {  // of the lanes up to this one
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const double y = __shfl_up(x, step);
        if (lane >= step) x += y;
    }
    return x;
}

struct Walk {
    int node, accepted;  // where it ends, -1: nowhere (no nodes); nodes of its path
    uint64_t rejected;   // children of that node
    int64_t token;       // this lane's
    float u0;
};
template <int DT>
__device__ __forceinline__ Walk walk(const VerifyParams &p, int b, int lane, bool write) {
    const int n = p.counts != nullptr ? min(max(p.counts[b], 0), p.n) : p.n;
    bool there = lane < n;
    int up = -1;
    int64_t x = -1;
    double u = 0.0, pt = 0.0, qt = 0.0;
    if (there) {
        up = p.parents != nullptr ? p.parents[b * p.parents_s[0] + lane * p.parents_s[1]] : lane - 1;
        if (up < 0 || up >= lane) up = -1;
        const int64_t at = b * p.tokens_s[0] + lane * p.tokens_s[1];
        x = p.tokens_64 ? ((const int64_t *)p.tokens)[at] : ((const int32_t *)p.tokens)[at];
        const float f = p.uniforms[b * p.uniforms_s[0] + lane * p.uniforms_s[1]];
        u = f > 0.f ? (double)f : 0.0;
        there = lane == 0 || (x >= 0 && x < p.V);
        if (up >= 0 && there) {
            const int64_t size = DT == 2 ? 4 : 2;
            pt = chance(value_at<DT>((const uint8_t *)p.target + size * (b * p.target_s[0] + up * p.target_s[1]), x));
            if (p.draft != nullptr) qt = chance(value_at<DT>((const uint8_t *)p.draft + size * (b * p.draft_s[0] + up * p.draft_s[1]), x));
        }
    }
    Walk w{n > 0 ? 0 : -1, n > 0 ? 1 : 0, 0ull, x, 0.f};
    w.u0 = (float)of_lane(u, 0);
    int mine = lane == 0 && n > 0 ? 0 : -1;  // of the path
    double rest = 1.0;
    for (uint64_t children = __builtin_amdgcn_ballot_w64(there && up == 0 && lane > 0); children != 0ull;) {
        const int c = __ffsll((unsigned long long)children) - 1;
        children &= children - 1;
        const int64_t xc = (int64_t)__builtin_bit_cast(uint64_t, of_lane(__builtin_bit_cast(double, x), c));
        double pc = of_lane(pt, c);
        const double uc = of_lane(u, c);
        bool yes;
        if (p.draft != nullptr) {
            yes = uc * of_lane(qt, c) < pc;
        } else {
            if (__builtin_amdgcn_ballot_w64((w.rejected >> lane & 1) != 0 && x == xc) != 0ull) pc = 0.0;
            yes = uc * rest < pc;
        }
        if (yes) {
            if (lane == w.accepted) mine = c;
            w.accepted++;
            w.node = c;
            w.rejected = 0ull;
            rest = 1.0;
            children = __builtin_amdgcn_ballot_w64(there && up == c);
        } else {
            w.rejected |= 1ull << c;
            rest -= pc;
        }
    }
    if (write) {
        if (lane < p.n) p.path[(int64_t)b * p.n + lane] = mine;
        if (lane == 0) p.accepted[b] = w.accepted;
    }
    return w;
}

template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_kernel(const VerifyParams p) {
    __shared__ uint32_t without[kVerifyMostEach / 32];  // the rejected tokens of a part, a bit each
    __shared__ f64x4 quarters;
    __shared__ double ends[kVerifyWaves];
    __shared__ uint64_t rejected_by;
    __shared__ float u0_by;
    __shared__ int node_by, last_by, first_by, end_by;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = (int)(blockIdx.x / (unsigned)p.parts), part = (int)(blockIdx.x - (unsigned)b * p.parts);
    int64_t token_of_lane = -1;  // (of the first wave)
    if (wave == 0) {
        const Walk w = walk<DT>(p, b, lane, part == 0);
        token_of_lane = w.token;
        if (lane == 0) node_by = w.node, rejected_by = w.rejected, u0_by = w.u0;
    }
    __syncthreads();
    const int node = __builtin_amdgcn_readfirstlane(node_by);
    const uint64_t rejected = rejected_by;
    if (node < 0) {
        if (part == 0 && tid == 0) {
            if (p.tokens_64) ((int64_t *)p.next)[b] = -1;
            else ((int32_t *)p.next)[b] = -1;
        }
        return;
    }
    const int64_t size = DT == 2 ? 4 : 2;
    const void *const row = (const uint8_t *)p.target + size * (b * p.target_s[0] + node * p.target_s[1]);
    const void *const drawn = p.draft != nullptr && rejected != 0ull ? (const uint8_t *)p.draft + size * (b * p.draft_s[0] + node * p.draft_s[1]) : nullptr;
    const bool some_without = p.draft == nullptr && rejected != 0ull;
    const int quarter = p.each / kVerifyWaves;

    bool plain = false;  // r = p, where nothing is left of it otherwise
    auto mark = [&](int from) {  // the rejected tokens of [from, from + each)
        if (!some_without) return;
        __syncthreads();
        for (int i = tid; i < (p.each + 31) / 32; i += kVerifyThreads) without[i] = 0u;
        __syncthreads();
        if (wave == 0 && (rejected >> lane & 1) != 0 && token_of_lane >= from && token_of_lane < (int64_t)from + p.each) {
            const int at = (int)(token_of_lane - from);
            atomicOr(&without[at >> 5], 1u << (at & 31));
        }
        __syncthreads();
    };
    // r of values v .. v + 3, v a multiple of 4 behind `from`
    auto four_of = [&](int from, int v, double (&r)[4]) __attribute__((always_inline)) {
        float x[4], y[4] = {0.f, 0.f, 0.f, 0.f};
        four<DT>(row, v, p.V, x);
        if (drawn != nullptr && !plain) four<DT>(drawn, v, p.V, y);
        uint32_t out = 0u;
        if (some_without && !plain) out = without[(v - from) >> 5] >> ((v - from) & 31);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double d = chance(x[i]) - chance(y[i]);
            r[i] = d > 0.0 && (out >> i & 1u) == 0u ? d : 0.0;
        }
    };
    auto quarter_sum = [&](int from) {  // this wave's of the part that begins there, in all its lanes
        const int v0 = from + wave * quarter, v1 = min(v0 + quarter, p.V);
        double x = 0.0;
#pragma unroll 4
        for (int v = v0 + 4 * lane; v < v1; v += 4 * 64) {
            double r[4];
            four_of(from, v, r);
            x += (r[0] + r[1]) + (r[2] + r[3]);
        }
#pragma unroll
        for (int step = 1; step < 64; step *= 2) x += __shfl_xor(x, step);
        return x;
    };

    mark(part * p.each);
    const double mine = quarter_sum(part * p.each);
    f64x4 held = {0.0, 0.0, 0.0, 0.0};  // part `lane`'s quarters
    if (p.parts > 1) {
        f64x4 *const all_sums = (f64x4 *)p.sums + (int64_t)b * p.parts;
        const HandOver io(all_sums, 32u * (uint32_t)p.parts);
        if (lane == 0) io.put(32u * (uint32_t)part + 8u * (uint32_t)wave, __builtin_bit_cast(f32x2, mine));
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (wave == 0) {
            const bool last = all_arrived(p.arrivals + (int64_t)b * p.parts, p.tag, part, p.parts);
            if (lane == 0) last_by = last;
        }
        __syncthreads();
        if (last_by == 0) return;
        if (lane < p.parts) {
            const f32x4 lo = io.get4(32u * (uint32_t)lane), hi = io.get4(32u * (uint32_t)lane + 16u);
            const f64x2 x = __builtin_bit_cast(f64x2, lo), y = __builtin_bit_cast(f64x2, hi);
            held = f64x4{x.x, x.y, y.x, y.y};
        }
    } else {
        if (lane == 0) ((double *)&quarters)[wave] = mine;
        __syncthreads();
        if (lane == 0) held = quarters;
    }
    // ---- the last workgroup: the part and the quarter of it that the token is in, then the token ----
    auto whole_of = [](const f64x4 &q) { return ((q.x + q.y) + q.z) + q.w; };
    double upto = sum_upto(whole_of(held), lane);
    if (!(of_lane(upto, 63) > 0.0) && (drawn != nullptr || some_without)) {  // (the rejected tokens were all that the target would say)
        plain = true;
        for (int i = 0; i < p.parts; i++) {
            const double x = quarter_sum(i * p.each);
            __syncthreads();
            if (lane == 0) ((double *)&quarters)[wave] = x;
            __syncthreads();
            if (lane == i) held = quarters;
        }
        upto = sum_upto(whole_of(held), lane);
    }
    const double whole = of_lane(upto, 63);
    int token = -1;
    if (whole > 0.0) {
        const double want = (double)u0_by * whole;
        // (of an empty part the running sum may be beyond what it is in front of it by a rounding)
        const bool any_there = whole_of(held) > 0.0;
        const uint64_t some = __builtin_amdgcn_ballot_w64(any_there), beyond = __builtin_amdgcn_ballot_w64(any_there && upto > want);
        const int at = beyond != 0ull ? __ffsll((unsigned long long)beyond) - 1 : 63 - __clzll((long long)some);
        double before = at > 0 ? of_lane(upto, at - 1) : 0.0;
        int k = -1;  // the quarter: the first whose end is beyond, or the last that is not empty
        {
            double c = before, start = before;
#pragma unroll
            for (int i = 0; i < kVerifyWaves; i++) {
                const double x = of_lane(held[i], at);
                if (x > 0.0 && (k < 0 || !(c > want))) {
                    k = i;
                    start = c;
                    c += x;
                }
            }
            before = start;
        }
        const int from = at * p.each;
        mark(from);
        const int q0 = from + k * quarter, q1 = min(q0 + quarter, p.V);
        // each thread a run of it
        const int run = verify_run(quarter), v0 = q0 + tid * run, v1 = min(v0 + run, q1);
        double x = 0.0;
        bool any = false;
        for (int v = v0; v < v1; v += 4) {
            double r[4];
            four_of(from, v, r);
            x += (r[0] + r[1]) + (r[2] + r[3]);
            any = any || r[0] > 0.0 || r[1] > 0.0 || r[2] > 0.0 || r[3] > 0.0;
        }
        double end = sum_upto(x, lane);
        if (lane == 63) ends[wave] = end;
        if (tid == 0) first_by = 0x7fffffff, end_by = -1;
        __syncthreads();
        double base = before;
        for (int i = 0; i < wave; i++) base += ends[i];
        end += base;
        if (any) {
            if (end > want) atomicMin(&first_by, tid);
            atomicMax(&end_by, tid);
        }
        __syncthreads();
        const int found = first_by != 0x7fffffff ? first_by : end_by;  // (beyond the last sum by a rounding: the last run that is not empty)
        if (found == tid) ends[0] = end - x;  // (where it begins)
        __syncthreads();
        if (wave == 0) {
            // the run's values, 64 a time
            double c = ends[0];
            const int r0 = q0 + found * run, r1 = min(r0 + run, q1);
            for (int v = r0; v < r1; v += 64) {
                double r = 0.0;
                if (v + lane < r1) {
                    double q[4];
                    const int v4 = v + (lane & ~3);
                    four_of(from, v4, q);
                    r = lane & 2 ? lane & 1 ? q[3] : q[2] : lane & 1 ? q[1] : q[0];
                }
                const double sum = c + sum_upto(r, lane);
                const uint64_t over = __builtin_amdgcn_ballot_w64(r > 0.0 && sum > want), there = __builtin_amdgcn_ballot_w64(r > 0.0);
                if (there != 0ull) token = v + 63 - __clzll((long long)there);  // (the last so far)
                if (over != 0ull) {
                    token = v + __ffsll((unsigned long long)over) - 1;
                    break;
                }
                c = of_lane(sum, 63);
            }
        }
    }
    if (tid == 0) {
        if (p.tokens_64) ((int64_t *)p.next)[b] = token;
        else ((int32_t *)p.next)[b] = token;
    }
}

}  // namespace

hipError_t launch_verify(const VerifyParams &p, int dtype, hipStream_t stream) {
    const dim3 grid((unsigned)(p.B * p.parts));
    if (dtype == 0) hipLaunchKernelGGL(verify_kernel<0>, grid, dim3(kVerifyThreads), 0, stream, p);
    else if (dtype == 1) hipLaunchKernelGGL(verify_kernel<1>, grid, dim3(kVerifyThreads), 0, stream, p);
    else hipLaunchKernelGGL(verify_kernel<2>, grid, dim3(kVerifyThreads), 0, stream, p);
    return hipGetLastError();
}

}  // namespace sa
