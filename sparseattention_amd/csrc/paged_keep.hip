// Keeping the accepted drafts of a tree in the 8-bit paged cache on gfx950 (MI355X): token len + path[i] of a sequence becomes token len + i.  No
// counterpart in the reference.
//
// A tree of up to 64 drafts lies in at most three blocks of a head.  A workgroup has them of one head, K or V, in LDS and writes those anew in
// which a token comes from another place.  Inside a block codes move as they are.  Where tokens come from other blocks the block's scale is
//     e' = max(e, the least exponent for these),   e only if the block held tokens in front of the drafts or keeps some of its own,
// and all that it keeps is c' = round(c * 2^(e_source - e')), which changes nothing where the exponents agree.
// Bound by the chain lengths, path, table, scales, blocks, and by memory for many sequences.
#include "paged_codes.h"

namespace sa {
namespace {

constexpr int kKeepBlocks = 3, kKeepThreads = 256;

// Where K and V have four codes of a word of a block: word w holds columns of one row (K) or rows of one column (V).
__device__ __forceinline__ int k_row(int w) { return w >> 2 & 31; }
__device__ __forceinline__ int v_row(int w) { return 16 * (w & 1) + 8 * (w >> 1 & 1) + 4 * (w >> 7 & 1); }  // and the three behind
// The byte of row r in the 16 of a column, and where they lie
__device__ __forceinline__ int v_byte(int w, int r) { return 4 * (w & ~0xff) + 512 * (r >> 2 & 1) + 16 * (w >> 2 & 31) + 8 * (r >> 3 & 1) + 4 * (r >> 4) + (r & 3); }

template <int ND>
__global__ __launch_bounds__(kKeepThreads) void paged_keep_kernel(const PagedKeepParams p) {
    constexpr int W = ND * 256;  // words of a block
    __shared__ __attribute__((aligned(16))) uint32_t codes[kKeepBlocks][W];
    __shared__ int source[32 * kKeepBlocks], goes[32 * kKeepBlocks];  // of a row: where it comes from; to which other blocks, a bit each
    __shared__ float factor[32 * kKeepBlocks];
    __shared__ unsigned largest[kKeepBlocks][kKeepBlocks];  // code of those that block [to] takes from block [from]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool values = blockIdx.x & 1u;
    const unsigned item = blockIdx.x >> 1;
    const int h = (int)(item % (unsigned)p.c.H), b = (int)(item / (unsigned)p.c.H);
    const int len = max(p.t.lens[b], 0), n = min(max(p.accepted[b], 0), p.n), off = len & 31;
    // node i's place is row off + i of the blocks
    int from = lane < n ? p.path[b * p.path_s[0] + lane * p.path_s[1]] : -1;
    if (from < 0 || from >= p.n) from = -1;
    if (__builtin_amdgcn_ballot_w64(from >= 0 && from != lane) == 0ull) return;
    const int furthest = (int)wave_max((uint32_t)(off + max(from, lane < n ? lane : 0)));
    const int blocks = (furthest >> 5) + 1;
    int64_t at[kKeepBlocks];
    int e[kKeepBlocks];
    uint8_t *const base = values ? p.c.v : p.c.k;
    float *const scales = values ? p.c.v_scales : p.c.k_scales;
#pragma unroll
    for (int k = 0; k < kKeepBlocks; k++) {
        const int blk = (len >> 5) + k, page = k < blocks ? page_at(p.t, b, blk >> p.c.lper, p.c.pages) : -1;
        at[k] = page >= 0 ? block_at(p.c, page, h, blk & ((1 << p.c.lper) - 1)) : -1;
    }
#pragma unroll
    for (int k = 0; k < kKeepBlocks; k++) {
        e[k] = at[k] >= 0 ? exp_of_scale(scales[at[k]]) : kScaleExpMin;
        if (at[k] >= 0)
            for (int i = tid; i < W / 4; i += kKeepThreads) ((u32x4 *)codes[k])[i] = ((const u32x4 *)(base + at[k] * (4 * W)))[i];
    }
    for (int r = tid; r < 32 * kKeepBlocks; r += kKeepThreads) source[r] = r, goes[r] = 0;
    if (tid < kKeepBlocks * kKeepBlocks) largest[tid / kKeepBlocks][tid % kKeepBlocks] = 0u;
    __syncthreads();
    uint32_t written = 0u, own = off > 0 ? 1u : 0u;  // blocks with a row from another place; those whose scale counts
    if (wave == 0) {
        const int s = off + from, to = off + lane;
        bool there = from >= 0;
#pragma unroll
        for (int k = 0; k < kKeepBlocks; k++)
            if (((s >> 5) == k || (to >> 5) == k) && at[k] < 0) there = false;
        if (there) {
            source[to] = s;
            if ((s >> 5) != (to >> 5)) atomicOr(&goes[s], 1 << (to >> 5));
        }
#pragma unroll
        for (int k = 0; k < kKeepBlocks; k++) {
            if (__builtin_amdgcn_ballot_w64(there && (to >> 5) == k && s != to) != 0ull) written |= 1u << k;
            // (a token that is not moved stays as it is)
            if (__builtin_amdgcn_ballot_w64(lane < n && (to >> 5) == k && (!there || (s >> 5) == k)) != 0ull) own |= 1u << k;
        }
        if (lane == 0) factor[0] = __uint_as_float(written), factor[1] = __uint_as_float(own);
    }
    __syncthreads();
    written = (uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(factor[0]));
    own = (uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(factor[1]));
    if (written == 0u) return;

    // ---- the largest code that each block takes from each other ----
#pragma unroll
    for (int k = 0; k < kKeepBlocks; k++) {
        if (k >= blocks || at[k] < 0) continue;
        uint32_t most[kKeepBlocks] = {};
        for (int w = tid; w < W; w += kKeepThreads) {
            const uint32_t word = codes[k][w];
            const int row = 32 * k + (values ? v_row(w) : k_row(w));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int to = goes[row + (values ? i : 0)];
                const uint32_t size = word >> (8 * i) & 0x7fu;
#pragma unroll
                for (int j = 0; j < kKeepBlocks; j++)
                    if (j != k && (to >> j & 1) != 0 && size != 0x7fu) most[j] = max(most[j], size);
            }
        }
#pragma unroll
        for (int j = 0; j < kKeepBlocks; j++) {
            if (j == k) continue;
            const uint32_t m = wave_max(most[j]);
            if (lane == 0 && m != 0u) atomicMax(&largest[j][k], m);
        }
    }
    __syncthreads();
    int e_new[kKeepBlocks];
#pragma unroll
    for (int j = 0; j < kKeepBlocks; j++) {
        e_new[j] = (own >> j & 1u) != 0u ? e[j] : kScaleExpMin;
#pragma unroll
        for (int k = 0; k < kKeepBlocks; k++) {
            const uint32_t m = largest[j][k];
            if (m != 0u) e_new[j] = max(e_new[j], scale_exp(__builtin_amdgcn_cvt_pk_f32_fp8((int)m, false)[0] * exp2i(e[k])));
        }
    }
    if (tid < 32 * kKeepBlocks) {
        const int to = tid >> 5, k = source[tid] >> 5;
        int diff = 0;  // (rows behind the last kept one stay as they are)
#pragma unroll
        for (int i = 0; i < kKeepBlocks; i++)
#pragma unroll
            for (int j = 0; j < kKeepBlocks; j++)
                if (i == k && j == to && tid < off + n) diff = e[i] - e_new[j];
        factor[tid] = exp2i(min(max(diff, -126), 127));
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kKeepBlocks; j++) {
        if ((written >> j & 1u) == 0u) continue;
        uint32_t *const out = (uint32_t *)(base + at[j] * (4 * W));
        for (int w = tid; w < W; w += kKeepThreads) {
            const int row = 32 * j + (values ? v_row(w) : k_row(w));
            uint32_t word = 0u;
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int to = row + (values ? i : 0), s = source[to];
                f[i] = factor[to];
                if (values) word |= (uint32_t)((const uint8_t *)codes[s >> 5])[v_byte(w, s & 31)] << (8 * i);
                else if (i == 0) word = codes[s >> 5][(w & ~0x7c) | (s & 31) << 2];
            }
            if (f[0] != 1.f || f[1] != 1.f || f[2] != 1.f || f[3] != 1.f) {
                const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true);
                word = codes4(lo.x * f[0], lo.y * f[1], hi.x * f[2], hi.y * f[3]);
            }
            out[w] = word;
        }
        if (tid == 0 && e_new[j] != e[j]) scales[at[j]] = exp2i(e_new[j]);
    }
}

}  // namespace

hipError_t launch_paged_keep(const PagedKeepParams &p, hipStream_t stream) {
    const dim3 grid(2u * (unsigned)p.c.H * (unsigned)p.t.B);
    if (p.c.D == 64) hipLaunchKernelGGL(paged_keep_kernel<2>, grid, dim3(kKeepThreads), 0, stream, p);
    else if (p.c.D == 128) hipLaunchKernelGGL(paged_keep_kernel<4>, grid, dim3(kKeepThreads), 0, stream, p);
    else if (p.c.D == 256) hipLaunchKernelGGL(paged_keep_kernel<8>, grid, dim3(kKeepThreads), 0, stream, p);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace sa
