// Storing tokens in the 8-bit paged cache with their keys normed and rotated on the way, and their queries with them, on gfx950 (MI355X).  No
// counterpart in the reference.  The formula of a row is rotate.h's, a block's and its scale's paged_cache.hip's; keys go from float32 to codes in
// one rounding, queries to their own type.
//
// A workgroup has the tokens of one block of a sequence, 32 or fewer: it makes their angles once in LDS, and its waves take keys of a head, values of
// a head, or rows of queries in turn.  Bound by memory where there are many tokens, by the chain length, table, scale, block where there are few.
#include "paged_codes.h"
#include "rotate.h"
#include "tree.h"

namespace sa {
namespace {

constexpr int kRotatedThreads = 64 * kCacheWaves;
// The words of LDS: angles [32][4 ND] of 4 cosines and 4 sines, then 16 rows or a block's codes for each wave.
template <int ND>
constexpr int angle_bytes = 32 * 4 * ND * 32;
template <int ND>
constexpr int wave_bytes = ND * 1024 > 16 * row_bytes<ND> ? ND * 1024 : 16 * row_bytes<ND>;

template <int DT, int ND, bool INTER>
__global__ __launch_bounds__(kRotatedThreads, 2) void paged_rotated_kernel(const PagedRotatedParams p) {
    using X = Run4<DT>;
    constexpr int LPR = 4 * ND, T = 64 / LPR, U = 4;  // lanes of a row, rows of a step, steps under way
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    f32x4 *const angles = (f32x4 *)smem;  // of row r, four pairs l: [(r * LPR + l) * 2], cosines and sines
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane % LPR, r0 = lane / LPR;
    uint8_t *const mine = smem + angle_bytes<ND> + wave * wave_bytes<ND>;

    unsigned item = blockIdx.x;
    const int split = (int)(item % (unsigned)p.splits);
    item /= (unsigned)p.splits;
    const int nb = (int)(item % (unsigned)p.blocks), b = (int)(item / (unsigned)p.blocks);
    const int len = max(p.t.lens[b], 0);
    const int n = p.counts != nullptr ? min(max(p.counts[b], 0), p.S) : p.S;
    // row r of the block is token 32 nb + r - len % 32 of the call; rows a .. zs - 1 are the call's, a .. z - 1 new tokens, 0 .. held - 1 there already
    const int first = 32 * nb - (len & 31);
    const int held = max(-first, 0), a = held, z = min(n - first, 32), zs = min(p.S - first, 32);
    if (a >= zs) return;
    const Columns c = columns_of(l, p.c.cols, p.r.R, INTER);

    // ---- angles of rows a .. z - 1 ----
    int *const depth = (int *)(smem + angle_bytes<ND>);
    if (p.parents != nullptr) {  // (at most 64 tokens)
        if (wave == 0) depth[lane] = __popcll(tree_ancestors(p.parents + b * p.parents_stride[0], p.parents_stride[1], n, lane)) - 1;
        __syncthreads();
    }
    for (int i = threadIdx.x; i < (z - a) * (p.r.R / 2); i += kRotatedThreads) {
        const int r = a + i / (p.r.R / 2), j = i - (r - a) * (p.r.R / 2), token = first + r;
        double at;
        if (p.r.positions != nullptr) at = position_at(p.r, axis_of(p.r, j), b, token);
        else at = (double)len + (p.parents != nullptr ? depth[token] : token);
        float co, si;
        turn(at, p.r.frequencies[j], co, si);
        float *const to = (float *)(angles + (r * LPR + (j >> 2)) * 2) + (j & 3);
        to[0] = co;
        to[4] = si;
    }
    __syncthreads();
    auto turns_of = [&](int r) {
        Turns t;
        const f32x4 co = angles[(r * LPR + l) * 2], si = angles[(r * LPR + l) * 2 + 1];
#pragma unroll
        for (int i = 0; i < 4; i++) t.c[i] = co[i], t.s[i] = si[i];
        return t;
    };
    const float share = 1.f / (float)p.c.cols;
    auto row_done = [&](float (&f)[2][4], const float (&w)[2][4], bool norm, int r) __attribute__((always_inline)) {
        if (norm) norm_row<LPR>(f, w, share, p.r.eps);
        if (c.rot) rotate<INTER, false>(f, turns_of(r));
    };

    // ---- keys and values of a head each, then queries by QR rows ----
    const int blk = (len >> 5) + nb, sub = blk & ((1 << p.c.lper) - 1);
    const int page = a < z ? page_at(p.t, b, blk >> p.c.lper, p.c.pages) : -1;
    const int kv = page >= 0 ? 2 * p.c.H : 0, rows = (zs - a) * p.Hq, per = T * p.steps;
    const int items = kv + (rows + per - 1) / per;
    float wq[2][4], wk[2][4];
    weights_of(p.r.q_weight, p.r.weight_dtype, c, wq);
    weights_of(p.r.k_weight, p.r.weight_dtype, c, wk);
    for (int it = split * kCacheWaves + wave; it < items; it += p.splits * kCacheWaves) {
        if (it >= kv) {
            const int from = (it - kv) * per, to = min(from + per, rows);
            const unsigned each = (unsigned)(zs - a);
#pragma unroll 1
            for (int at = from; at < to; at += T * U) {
                typename X::T in[U][2] = {};
                int r[U], h[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int row = min(at + u * T + r0, to - 1);
                    h[u] = (int)((unsigned)row / each);
                    r[u] = a + row - h[u] * (int)each;
                    const uint16_t *const x = p.q + b * p.qs[0] + h[u] * p.qs[1] + (int64_t)(first + r[u]) * p.qs[2];
                    if (c.live && at + u * T + r0 < to && r[u] < z) {
                        in[u][0] = *(const typename X::T *)(x + c.at[0]);
                        in[u][1] = *(const typename X::T *)(x + c.at[1]);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (at + u * T >= to) break;
                    const bool live = r[u] < z;  // (rows of padding are 0)
                    float f[2][4];
                    X::floats(in[u][0], f[0]);
                    X::floats(in[u][1], f[1]);
                    row_done(f, wq, p.r.q_weight != nullptr, live ? r[u] : a);
                    if (c.live && at + u * T + r0 < to) {
                        uint16_t *const y = p.qo + b * p.qos[0] + h[u] * p.qos[1] + (int64_t)(first + r[u]) * p.qos[2];
                        const typename X::T none = {0u, 0u};
                        *(typename X::T *)(y + c.at[0]) = live ? X::rounded(f[0]) : none;
                        *(typename X::T *)(y + c.at[1]) = live ? X::rounded(f[1]) : none;
                    }
                }
            }
            continue;
        }
        const int h = it >> 1;
        if (it & 1) {
            append_block<DT, ND>(p.c, p.v + b * p.vs[0] + h * p.vs[1] + (int64_t)first * p.vs[2], p.vs[2], true, page, h, sub, held, a, z, mine);
            in_order();
            continue;
        }
        // Rows come in groups of U steps and are made twice, for the largest finite magnitude and for the codes; where there is more than one
        // group they are read again from the caches.  (A block's rows kept in float32 were 128 registers at D = 256.)
        const uint16_t *const x = p.k + b * p.ks[0] + h * p.ks[1] + (int64_t)first * p.ks[2];
        const int64_t at = block_at(p.c, page, h, sub);
        uint8_t *const out = p.c.k + at * (ND * 1024);
        float *const scale = p.c.k_scales + at;
        const int g0 = a / (T * U), g1 = (z - 1) / (T * U);
        typename X::T in[U][2];
        auto load = [&](int g) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int r = (g * U + u) * T + r0;
                const bool there = c.live && r >= a && r < z;
#pragma unroll
                for (int k = 0; k < 2; k++) in[u][k] = there ? *(const typename X::T *)(x + r * p.ks[2] + c.at[k]) : typename X::T{0u, 0u};
            }
        };
        auto row = [&](int r, int u, float (&y)[2][4]) __attribute__((always_inline)) {
            const bool live = r >= a && r < z;
            X::floats(in[u][0], y[0]);
            X::floats(in[u][1], y[1]);
            row_done(y, wk, p.r.k_weight != nullptr, live ? r : a);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (!live || !c.live) y[j >> 2][j & 3] = 0.f;
        };
        uint32_t m = 0u, all = 0u;
        load(g0);
        const int e_old = held > 0 ? exp_of_scale(*scale) : kScaleExpMin;
#pragma unroll 1
        for (int g = g0;; load(++g)) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                float y[2][4];
                row((g * U + u) * T + r0, u, y);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint32_t size = __float_as_uint(y[j >> 2][j & 3]) & 0x7fffffffu;
                    all = max(all, size);
                    m = max(m, size < 0x7f800000u ? size : 0u);
                }
            }
            if (g == g1) break;
        }
        m = wave_max(m);
        all = wave_max(all);
        const int e = max(e_old, scale_exp(__uint_as_float(m)));
        const float inv = exp2i(-e);
        const bool plain = all < 0x7f800000u && e < kScaleExpMax;
        const bool grows = held > 0 && e > e_old;
        const float f = exp2i(max(e_old - e, -126));
        if (lane == 0 && (grows || held == 0)) *scale = exp2i(e);
        // codes into LDS, four columns of a row a word, where the block has them
#pragma unroll 1
        for (int g = g1; g >= g0; g--) {
            if (g != g1) load(g);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int r = (g * U + u) * T + r0;
                float y[2][4];
                row(r, u, y);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const float(&v)[4] = y[k];
                    const int col = c.at[k];
                    *(uint32_t *)(mine + 1024 * (col >> 5) + 16 * (32 * ((col >> 4) & 1) + r) + (col & 15)) =
                        plain ? codes4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv)
                              : codes4(scaled(v[0], inv), scaled(v[1], inv), scaled(v[2], inv), scaled(v[3], inv));
                }
            }
        }
        in_order();
        const int key = lane & 31;
        const bool fresh = key >= a && key < z, old = grows && key < held;
#pragma unroll
        for (int d = 0; d < ND; d++) {
            u32x4 *const to = (u32x4 *)(out + 1024 * d + 16 * lane);
            if (fresh) {
                *to = *(const u32x4 *)(mine + 1024 * d + 16 * lane);
            } else if (old) {
                u32x4 u = *to;
#pragma unroll
                for (int i = 0; i < 4; i++) u[i] = again4(u[i], f);
                *to = u;
            }
        }
        in_order();
    }
}

template <int DT, int ND, bool INTER>
hipError_t launch(const PagedRotatedParams &p, hipStream_t stream) {
    constexpr int smem = angle_bytes<ND> + kCacheWaves * wave_bytes<ND>;
    auto kern = paged_rotated_kernel<DT, ND, INTER>;
    static unsigned long long attr_done = 0;
    if (const hipError_t e = allow_dynamic_smem(kern, smem, attr_done); e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)(p.splits * p.blocks * p.t.B)), dim3(kRotatedThreads), smem, stream, p);
    return hipGetLastError();
}
template <int DT, bool INTER>
hipError_t launch_dim(const PagedRotatedParams &p, hipStream_t stream) {
    if (p.c.D == 64) return launch<DT, 2, INTER>(p, stream);
    if (p.c.D == 128) return launch<DT, 4, INTER>(p, stream);
    if (p.c.D == 256) return launch<DT, 8, INTER>(p, stream);
    return hipErrorInvalidValue;
}

}  // namespace

// Workgroups that share a block's heads: as many as give each compute unit three workgroups, with an item for every wave.
int paged_rotated_splits(int B, int blocks, int H, int Hq, int S) {
    const int64_t tiles = (int64_t)B * blocks, want = (768 + tiles - 1) / tiles;
    const int64_t items = 2ll * H + (S == 1 ? (Hq + 3) / 4 : Hq), most = (items + kCacheWaves - 1) / kCacheWaves;
    return (int)(want < most ? want : most);
}

hipError_t launch_paged_rotated(const PagedRotatedParams &p, int dtype, hipStream_t stream) {
    if (dtype == 0) return p.r.interleaved ? launch_dim<0, true>(p, stream) : launch_dim<0, false>(p, stream);
    if (dtype == 1) return p.r.interleaved ? launch_dim<1, true>(p, stream) : launch_dim<1, false>(p, stream);
    return hipErrorInvalidValue;
}

}  // namespace sa
