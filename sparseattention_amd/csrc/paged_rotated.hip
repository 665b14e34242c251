// Storing tokens in the 8-bit paged cache with their keys normed and rotated on the way, and their queries with them, on gfx950 (MI355X).  No
// counterpart in the reference.  The formula of a row is rotate.h's, a block's and its scale's paged_cache.hip's; keys go from float32 to codes in
// one rounding, queries to their own type.
//
// One launch, whose workgroups have one of three things to do: keys of a block of a sequence, 32 tokens or fewer, 8 a wave, head by head with the angles in registers; values of
// blocks, a wave each, as paged_append_kernel stores them; or queries, a wave 64 / LPR tokens with their angles in registers, as rotate_kernel has
// them.  Bound by memory where there are many tokens, by the chain length, table, scale, block where there are few.  (With the read-back, the prompts below took 93 us by
// workgroups that had all three of a block, 75 by these, and 70 since a block's keys stay in the registers of four waves instead of 72.)
//
// Measured (32 + 8 heads, D = 128, bf16, norms, where nothing else is said): 1 token of 64 sequences 7.8 us; 4096 tokens of one 24 us, 3.8 TB/s read and written (1.2 less
// with no angles made); 16 prompts of up to 2047, 12 heads, D = 64, fp16, interleaved, no norms 45 us, 4.0 TB/s (0.8 less; a copy of 1 GiB: 5.1).
#include <algorithm>

#include "paged_codes.h"
#include "rotate.h"
#include "tree.h"

namespace sa {
namespace {

constexpr int kRotatedThreads = 64 * kCacheWaves;

template <int DT, int ND, bool INTER>
__global__ __launch_bounds__(kRotatedThreads, ND == 8 ? 2 : 4) void paged_rotated_kernel(const PagedRotatedParams p) {
    using X = Run4<DT>;
    constexpr int LPR = 4 * ND, T = 64 / LPR;  // lanes of a row, rows of a step
    __shared__ __attribute__((aligned(16))) uint8_t smem[kCacheWaves * 16 * row_bytes<ND>];  // (values: 16 rows of each wave; keys: a block)
    __shared__ u32x2 sizes[kCacheWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane % LPR, r0 = lane / LPR;
    uint8_t *const mine = smem + wave * 16 * row_bytes<ND>;
    const float share = 1.f / (float)p.c.cols;
    const auto count_of = [&](int b) { return p.counts != nullptr ? min(max(p.counts[b], 0), p.S) : p.S; };

    if (blockIdx.x >= (unsigned)p.key_groups + (unsigned)p.value_groups) {
        // ---- queries: a wave has T tokens and some of their heads ----
        const unsigned id = (blockIdx.x - p.key_groups - p.value_groups) * kCacheWaves + wave;
        const int group = (int)(id / (unsigned)p.splits), h0 = (int)(id - (unsigned)group * p.splits) * p.heads, h1 = min(h0 + p.heads, p.Hq);
        if (h0 >= h1) return;
        const Columns c = columns_of(l, p.c.cols, p.r.R, INTER);
        int b, s;
        if (p.parents != nullptr) {  // (a wave has one sequence's, whose tree it looks through)
            const int each = (p.S + T - 1) / T;
            b = group / each;
            s = (group - b * each) * T + r0;
        } else {
            const int64_t token = (int64_t)group * T + r0;
            b = (int)(min(token, (int64_t)p.t.B * p.S) / p.S);
            s = (int)(token - (int64_t)b * p.S);
        }
        if (__builtin_amdgcn_ballot_w64(b < p.t.B && s < p.S) == 0ull) return;
        const bool live = c.live && b < p.t.B && s < p.S;
        b = min(b, p.t.B - 1);
        const int n = count_of(b);
        const bool zero = s >= n;
        double at = (double)max(p.t.lens[b], 0) + s;
        if (p.parents != nullptr) {
            const int above = __popcll(tree_ancestors(p.parents + b * p.parents_stride[0], p.parents_stride[1], n, lane)) - 1;
            at += __shfl(above, s & 63) - s;
        }
        Turns t;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            t.c[i] = 1.f, t.s[i] = 0.f;
            if (live && c.rot && !zero) {
                if (p.r.positions != nullptr) at = position_at(p.r, axis_of(p.r, 4 * l + i), b, s);
                turn(at, p.r.frequencies[4 * l + i], t.c[i], t.s[i]);
            }
        }
        float w[2][4];
        weights_of(p.r.q_weight, p.r.weight_dtype, c, w);
        rotate_rows<DT, LPR, INTER, false>(p.q + b * p.qs[0] + s * p.qs[2], p.qo + b * p.qos[0] + s * p.qos[2], p.qs[1], p.qos[1], h0, h1, c, live, zero, t, p.r.q_weight, w, share,
                                           p.r.eps);
        return;
    }
    if (blockIdx.x >= (unsigned)p.key_groups) {
        // ---- values: a wave a block of a head ----
        unsigned item = (blockIdx.x - p.key_groups) * kCacheWaves + wave;
        const int h = (int)(item % (unsigned)p.c.H);
        item /= (unsigned)p.c.H;
        const int nb = (int)(item % (unsigned)p.blocks), b = (int)(item / (unsigned)p.blocks);
        if (b >= p.t.B) return;
        const int len = max(p.t.lens[b], 0), first = 32 * nb - (len & 31);  // (row r of the block is token first + r of the call)
        const int held = max(-first, 0), z = min(count_of(b) - first, 32), blk = (len >> 5) + nb;
        if (held >= z) return;
        const int page = page_at(p.t, b, blk >> p.c.lper, p.c.pages);
        append_block<DT, ND>(p.c, p.v + b * p.vs[0] + h * p.vs[1] + (int64_t)first * p.vs[2], p.vs[2], true, page, h, blk & ((1 << p.c.lper) - 1), held, held, z, mine);
        return;
    }
    // ---- keys: some heads of a block, whose rows lie in the registers of four waves, 8 each, from their loads to their codes ----
    constexpr int STEPS = 8 / T;
    unsigned item = blockIdx.x;
    const unsigned parts = ((unsigned)p.c.H + p.key_heads - 1) / p.key_heads;
    const int part = (int)(item % parts);
    item /= parts;
    const int nb = (int)(item % (unsigned)p.blocks), b = (int)(item / (unsigned)p.blocks);
    const int len = max(p.t.lens[b], 0), first = 32 * nb - (len & 31), n = count_of(b);
    const int held = max(-first, 0), a = held, z = min(n - first, 32), blk = (len >> 5) + nb, sub = blk & ((1 << p.c.lper) - 1);
    if (a >= z) return;
    const int page = page_at(p.t, b, blk >> p.c.lper, p.c.pages);
    if (page < 0) return;
    const Columns c = columns_of(l, p.c.cols, p.r.R, INTER);
    const int h0 = part * p.key_heads, h_end = min(h0 + p.key_heads, p.c.H), row0 = 8 * wave + r0;  // the lane's rows are row0 + T i
    const uint16_t *x = p.k + b * p.ks[0] + h0 * p.ks[1] + (int64_t)(first + row0) * p.ks[2];
    auto is_new = [&](int i) { return row0 + T * i >= a && row0 + T * i < z; };
    typename X::T in[STEPS][2];
    auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            in[i][0] = in[i][1] = typename X::T{0u, 0u};
            if (c.live && is_new(i)) load_runs<DT, INTER>(x + (T * i) * p.ks[2], c, in[i]);
        }
    };
    load();
    int64_t at = block_at(p.c, page, h0, sub);
    int e_old = held > 0 ? exp_of_scale(p.c.k_scales[at]) : kScaleExpMin;
    uint64_t above = 0ull;
    if (p.parents != nullptr) above = tree_ancestors(p.parents + b * p.parents_stride[0], p.parents_stride[1], n, lane);
    Turns t[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const int token = first + row0 + T * i;
        double position = (double)len + token;
        if (p.parents != nullptr) position = (double)len + __popcll(__shfl((unsigned long long)above, token & 63)) - 1;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            t[i].c[j] = 1.f, t[i].s[j] = 0.f;
            if (c.rot && is_new(i)) {
                if (p.r.positions != nullptr) position = position_at(p.r, axis_of(p.r, 4 * l + j), b, token);
                turn(position, p.r.frequencies[4 * l + j], t[i].c[j], t[i].s[j]);
            }
        }
    }
    float w[2][4];
    weights_of(p.r.k_weight, p.r.weight_dtype, c, w);
#pragma unroll 1
    for (int h = h0; h < h_end; h++) {
        float y[STEPS][2][4];
        uint32_t m = 0u, all = 0u;
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            X::floats(in[i][0], y[i][0]);
            X::floats(in[i][1], y[i][1]);
            if (p.r.k_weight != nullptr) norm_row<LPR>(y[i], w, share, p.r.eps);
            if (c.rot) rotate<INTER, false>(y[i], t[i]);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float &f = y[i][j >> 2][j & 3];
                if (!c.live || !is_new(i)) f = 0.f;
                const uint32_t size = __float_as_uint(f) & 0x7fffffffu;
                all = max(all, size);
                m = max(m, size < 0x7f800000u ? size : 0u);
            }
        }
        uint8_t *const out = p.c.k + at * (ND * 1024);
        float *const scale = p.c.k_scales + at;
        const int e_was = e_old;
        if (h + 1 < h_end) {  // (the next head's rows and scale, on their way meanwhile)
            x += p.ks[1];
            load();
            at += (int64_t)1 << p.c.lper;
            if (held > 0) e_old = exp_of_scale(p.c.k_scales[at]);
        }
        m = wave_max(m);
        all = wave_max(all);
        if (lane == 0) sizes[wave] = u32x2{m, all};
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kCacheWaves; i++) {
            const u32x2 other = sizes[i];
            m = max(m, other.x);
            all = max(all, other.y);
        }
        const int e = max(e_was, scale_exp(__uint_as_float(m)));
        const float inv = exp2i(-e);
        const bool plain = all < 0x7f800000u && e < kScaleExpMax;
        const bool grows = held > 0 && e > e_was;
        const float f = exp2i(max(e_was - e, -126));
        if (threadIdx.x == 0 && (grows || held == 0)) *scale = exp2i(e);
        // codes into LDS, four columns of a row a word, where the block has them
#pragma unroll
        for (int i = 0; i < STEPS; i++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float(&v)[4] = y[i][k];
                const int col = c.at[k];
                *(uint32_t *)(smem + 1024 * (col >> 5) + 16 * (32 * ((col >> 4) & 1) + row0 + T * i) + (col & 15)) =
                    plain ? codes4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv)
                          : codes4(scaled(v[0], inv), scaled(v[1], inv), scaled(v[2], inv), scaled(v[3], inv));
            }
        __syncthreads();
        const int key = lane & 31;
        const bool fresh = key >= a && key < z, old = grows && key < held;
#pragma unroll
        for (int d = 0; d < ND; d += kCacheWaves) {
            if (ND < kCacheWaves && wave >= ND) break;
            const int piece = 1024 * (d + wave) + 16 * lane;
            u32x4 *const to = (u32x4 *)(out + piece);
            if (fresh) {
                *to = *(const u32x4 *)(smem + piece);
            } else if (old) {
                u32x4 u = *to;
#pragma unroll
                for (int i = 0; i < 4; i++) u[i] = again4(u[i], f);
                *to = u;
            }
        }
        __syncthreads();
    }
}

template <int DT, bool INTER>
hipError_t launch_dim(const PagedRotatedParams &p, int64_t groups, hipStream_t stream) {
    const dim3 grid((unsigned)groups), block(kRotatedThreads);
    if (p.c.D == 64) hipLaunchKernelGGL((paged_rotated_kernel<DT, 2, INTER>), grid, block, 0, stream, p);
    else if (p.c.D == 128) hipLaunchKernelGGL((paged_rotated_kernel<DT, 4, INTER>), grid, block, 0, stream, p);
    else if (p.c.D == 256) hipLaunchKernelGGL((paged_rotated_kernel<DT, 8, INTER>), grid, block, 0, stream, p);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace

// Keys: the angles are made for each workgroup, which has as many heads of its block as leave about 1024 workgroups.  Queries: heads are dealt out to as many waves as fill the
// device, four at least to one.
int64_t paged_rotated_plan(PagedRotatedParams &p) {
    const int T = p.c.D == 64 ? 8 : p.c.D == 128 ? 4 : 2;
    const int64_t tiles = (int64_t)p.t.B * p.blocks;
    p.key_heads = (int)std::min<int64_t>(p.c.H, std::max<int64_t>(1, tiles * p.c.H / 1024));
    const int64_t keys = tiles * ((p.c.H + p.key_heads - 1) / p.key_heads), values = (tiles * p.c.H + kCacheWaves - 1) / kCacheWaves;
    const int64_t groups = p.parents != nullptr ? (int64_t)p.t.B * ((p.S + T - 1) / T) : ((int64_t)p.t.B * p.S + T - 1) / T;
    const int64_t want = (4096 + groups - 1) / groups, most = (p.Hq + 3) / 4;
    p.splits = (int)std::min(want, most);
    p.heads = (p.Hq + p.splits - 1) / p.splits;
    const int64_t queries = (groups * p.splits + kCacheWaves - 1) / kCacheWaves, all = keys + values + queries;
    if (all > 0x7fffffff || (int64_t)p.t.B * p.S > 0x7fffffff) return -1;
    p.key_groups = (int)keys;
    p.value_groups = (int)values;
    return all;
}

hipError_t launch_paged_rotated(const PagedRotatedParams &p, int64_t groups, int dtype, hipStream_t stream) {
    if (dtype == 0) return p.r.interleaved ? launch_dim<0, true>(p, groups, stream) : launch_dim<0, false>(p, groups, stream);
    if (dtype == 1) return p.r.interleaved ? launch_dim<1, true>(p, groups, stream) : launch_dim<1, false>(p, groups, stream);
    return hipErrorInvalidValue;
}

}  // namespace sa
