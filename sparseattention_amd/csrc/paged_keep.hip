// Keeping the accepted drafts of a tree in the 8-bit paged cache on gfx950 (MI355X): token len + path[i] of a sequence becomes token len + i.  No
// counterpart in the reference.
//
// A tree of up to 64 drafts lies in at most three blocks of a head.  A workgroup has them of one head, K or V, in LDS and writes those anew in
// which a token comes from another place.  Inside a block codes move as they are.  Where tokens come from other blocks the block's scale is
//     e' = max(e, the least exponent for these),   e only if the block held tokens in front of the drafts or keeps some of its own,
// and all that it keeps is c' = round(c * 2^(e_source - e')), which changes nothing where the exponents agree.
// Bound by the chain lengths, path, table, scales, blocks, and by memory for many sequences.
//
// Measured (8 heads, D = 128): one sequence, 8 drafts 5.9 us; 128 sequences, 64 drafts 17.0 us, 24 MB read and written, three blocks in and out of
// a workgroup's LDS one after the other.  (Blocks written whole and largest codes always looked for: 22.)
#include "paged_codes.h"

namespace sa {
namespace {

constexpr int kKeepBlocks = 3, kKeepThreads = 256;
constexpr uint32_t kNoChange = 128;  // (changes are brought to -126 .. 127)

// Where K and V have four codes of a word of a block: word w holds columns of one row (K) or rows of one column (V).
__device__ __forceinline__ int k_row(int w) { return w >> 2 & 31; }
__device__ __forceinline__ int v_row(int w) { return 16 * (w & 1) + 8 * (w >> 1 & 1) + 4 * (w >> 7 & 1); }  // and the three behind
// The byte of row r in the 16 of a column, and where they lie
__device__ __forceinline__ int v_byte(int w, int r) { return 4 * (w & ~0xff) + 512 * (r >> 2 & 1) + 16 * (w >> 2 & 31) + 8 * (r >> 3 & 1) + 4 * (r >> 4) + (r & 3); }

template <int ND>
__global__ __launch_bounds__(kKeepThreads) void paged_keep_kernel(const PagedKeepParams p) {
    constexpr int W = ND * 256;  // words of a block
    __shared__ __attribute__((aligned(16))) uint32_t codes[kKeepBlocks][W];
    // of a row: where it comes from, and above that what its exponent changes by, + kNoChange; to which other blocks it goes, a bit each in a byte
    __shared__ __attribute__((aligned(16))) uint32_t source[32 * kKeepBlocks];
    __shared__ uint32_t goes[8 * kKeepBlocks], shared[2];
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
    if (tid < 32 * kKeepBlocks) source[tid] = (uint32_t)tid;
    if (tid < 8 * kKeepBlocks) goes[tid] = 0u;
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
            source[to] = (uint32_t)s;
            if ((s >> 5) != (to >> 5)) atomicOr(&goes[s >> 2], 1u << (8 * (s & 3) + (to >> 5)));
        }
#pragma unroll
        for (int k = 0; k < kKeepBlocks; k++) {
            if (__builtin_amdgcn_ballot_w64(there && (to >> 5) == k && s != to) != 0ull) written |= 1u << k;
            // (a token that is not moved stays as it is)
            if (__builtin_amdgcn_ballot_w64(lane < n && (to >> 5) == k && (!there || (s >> 5) == k)) != 0ull) own |= 1u << k;
        }
        // (and from which block a row goes to which other)
#pragma unroll
        for (int k = 0; k < kKeepBlocks; k++)
#pragma unroll
            for (int j = 0; j < kKeepBlocks; j++)
                if (j != k && __builtin_amdgcn_ballot_w64(there && (s >> 5) == k && (to >> 5) == j) != 0ull) own |= 0x100u << (kKeepBlocks * k + j);
        if (lane == 0) shared[0] = written, shared[1] = own;
    }
    __syncthreads();
    written = (uint32_t)__builtin_amdgcn_readfirstlane((int)shared[0]);
    own = (uint32_t)__builtin_amdgcn_readfirstlane((int)shared[1]);
    if (written == 0u) return;

    // ---- the largest code that each block takes from each other, where that block's scale is not the larger one anyway ----
#pragma unroll
    for (int k = 0; k < kKeepBlocks; k++) {
        bool looked_at = false;
#pragma unroll
        for (int j = 0; j < kKeepBlocks; j++)
            looked_at = looked_at || ((own >> (8 + kKeepBlocks * k + j) & 1u) != 0u && ((own >> j & 1u) == 0u || e[k] > e[j]));
        if (!looked_at) continue;
        uint32_t most[kKeepBlocks] = {};
        for (int w = tid; w < W; w += kKeepThreads) {
            const int row = 32 * k + (values ? v_row(w) : k_row(w));
            uint32_t four = goes[row >> 2];
            if (!values) four = (four >> (8 * (row & 3)) & 0xffu) * 0x01010101u;
            if (four == 0u) continue;
            const uint32_t word = codes[k][w];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t to = four >> (8 * i), size = word >> (8 * i) & 0x7fu;
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
        const int to = tid >> 5, k = (int)source[tid] >> 5;
        int diff = 0;  // (rows behind the last kept one stay as they are)
#pragma unroll
        for (int i = 0; i < kKeepBlocks; i++)
#pragma unroll
            for (int j = 0; j < kKeepBlocks; j++)
                if (i == k && j == to && tid < off + n) diff = e[i] - e_new[j];
        source[tid] |= (kNoChange + (uint32_t)min(max(diff, -126), 127)) << 8;
    }
    __syncthreads();
    // Words that keep their bytes are not written: those of rows in front of the drafts, as long as the scale stays.
#pragma unroll
    for (int j = 0; j < kKeepBlocks; j++) {
        if ((written >> j & 1u) == 0u) continue;
        uint32_t *const out = (uint32_t *)(base + at[j] * (4 * W));
        for (int w = tid; w < W; w += kKeepThreads) {
            const int row = 32 * j + (values ? v_row(w) : k_row(w));
            u32x4 s;
            if (values) s = *(const u32x4 *)&source[row];
            else s.x = s.y = s.z = s.w = source[row];
            bool same = true, exact = true;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                same = same && s[i] == (kNoChange << 8 | (uint32_t)(row + (values ? i : 0)));
                exact = exact && s[i] >> 8 == kNoChange;
            }
            if (same) continue;
            uint32_t word;
            if (values) {
                word = 0u;
#pragma unroll
                for (int i = 0; i < 4; i++) word |= (uint32_t)((const uint8_t *)codes[s[i] >> 5 & 7u])[v_byte(w, s[i] & 31)] << (8 * i);
            } else {
                word = codes[s.x >> 5 & 7u][(w & ~0x7c) | (s.x & 31) << 2];
            }
            if (!exact) {
                float f[4];
#pragma unroll
                for (int i = 0; i < 4; i++) f[i] = exp2i((int)(s[i] >> 8) - (int)kNoChange);
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
