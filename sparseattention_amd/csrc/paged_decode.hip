// Attention of few query rows over the 8-bit paged K/V cache on gfx950 (MI355X).
//
// The function is that of sparse_decode.hip (sparse_attention with BLOCK_Q = Sq, sparseattention/sparse_attn_kernel.py:74-146;
// the reference names decode kernels as future work, README.md:65) with K and V read from pages of e4m3 codes
// (paged.h), several query heads per K/V head, and sequences of their own lengths:
//     s = q . k / sqrt(D),  p = exp2(s - m),  o = sum p v / sum p     over the keys that a row attends to.
// The R = G * Sq rows of a K/V head go through the matrix unit together, 16 or 32 a tile; codes become bf16 or fp16 (exactly,
// V with its scale, which in fp16 rounds below its normal numbers) on their way from registers into the products, the scale of K joins the softmax's.  Bound by the
// bytes of K and V, each read once.  Per chunk of 32 keys a wave
//   * has K and V as operands straight from memory (D / 32 loads of 1 KiB each for both: paged.h has the order),
//   * computes S^T = K . Q^T (32 keys x 32 rows), masks, P = exp2(S^T - m), O^T += V^T . P^T.
// P is rounded to q's type for the second product, by up to half a step (bf16 2^-8, fp16 2^-11) of each weight, as in this library's other
// attention kernels: a split of P in two would double that product and still leave the output's own rounding.  In fp16 weights below 2^-14 (a row's
// largest is 1 or more) are rounded to steps of 2^-24: n of them are off by up to n * 2^-25 of the largest value.  Scores, reference
// values, sums and accumulators are float32.
// Measured (bf16 and one row per query head where nothing else is said): 32 sequences of up to 32768 keys, 8 x 8 heads, D = 128 286 us, 6.4 TB/s
// of K and V (a linear streaming read: 7.1); 64 ragged ones of up to 8192, 8 x 4 heads 98 us, 5.8; 16 in a window of 4096, 4 rows, 4 x 8
// heads, D = 64, fp16 17.5 us; one of 2011, 8 x 4 heads 9 us, the chain of what follows from one another.
#include "fwd_common.h"
#include "paged.h"
#include "paged_pieces.h"
#include "tree.h"

namespace sa {

namespace {

constexpr int kWaves = kPagedWaves;
constexpr int kPagedRowPad = 4;  // floats behind a row of a part: reference value and sum, and two that keep rows 16-byte aligned

template <int DT>
struct Codes;  // eight codes as an operand, times a power of two
template <>
struct Codes<0> {
    static __device__ __forceinline__ u32x4 take(uint32_t a, uint32_t b, float s) {
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, true))};
    }
};
template <>
struct Codes<1> {
    static __device__ __forceinline__ u32x4 take(uint32_t a, uint32_t b, float s) {
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, s, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, s, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, s, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, s, true))};
    }
};

// 0x80 in every byte that is a NaN code.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t nan_ones(uint32_t w) { return (nan_bytes(w) >> 7) * 0x38u; }  // the code of 1 for NaN, else 0
__device__ __forceinline__ uint32_t no_nan(uint32_t w) { return w & ~((nan_bytes(w) >> 7) * 0xffu); }

__device__ __forceinline__ float scale_of(float s) {  // (as the cache's kernels write them; anything else is brought into range)
    const int e = (int)((__float_as_uint(s) >> 23) & 0xffu);
    return __uint_as_float((uint32_t)min(max(e, 127 + kScaleExpMin), 127 + kScaleExpMax) << 23);
}

// A product of positive factors that is 0 or infinite, as the least or the largest number: 0 times the -inf of a masked key and infinity times a score
// of 0 would be NaN.
__device__ __forceinline__ float positive(float x) { return __uint_as_float(min(max(__float_as_uint(x), 1u), 0x7f7fffffu)); }

// ---- who does what (paged_pieces.h) ----
// Every workgroup takes an equal piece of the row of chunks, whatever the lengths: segments, each of one plane.  A plane that lies in several
// workgroups' pieces is added up by the last of them.  T is known on the device only, so every wave finds its workgroup's piece itself,
// by a sum over the units, or a launch in front does it for all.
struct Unit {
    int len, cnt;  // keys and query rows of its sequence
    int T0, T;     // first chunk, chunks (0: none)
    int F;         // with lists: FULL entries
};
template <bool LISTS>
__device__ __forceinline__ Unit unit_of(const PagedDecodeParams &p, int u) {
    const int b = LISTS ? u / p.c.H : u;
    const int lP = p.c.lper + 5;
    Unit r{p.t.lens[b], p.counts != nullptr ? p.counts[b] : p.Sq, 0, 0, 0};
    if constexpr (LISTS) {
        const int h = u - b * p.c.H;
        r.F = min(max(p.full_lens[b * p.fls[0] + h * p.fls[1]], 0), p.nK);
        r.T = (r.F + min(max(p.part_lens[b * p.pls[0] + h * p.pls[1]], 0), p.nK - r.F)) << p.c.lper;
    }
    r.len = min(max(r.len, 0), p.t.width << lP);
    r.cnt = min(max(r.cnt, 0), p.Sq);
    if constexpr (!LISTS) {
        r.T0 = p.window > 0 ? max(r.len - r.cnt - p.window + 1, 0) >> 5 : 0;
        r.T = ((r.len + 31) >> 5) - r.T0;
    }
    if (r.cnt == 0 || r.len == 0) r.T = 0;
    return r;
}
__device__ __forceinline__ Unit of_lane(const Unit &r, int lane) {  // (wave-uniform)
    return {__builtin_amdgcn_readlane(r.len, lane), __builtin_amdgcn_readlane(r.cnt, lane), __builtin_amdgcn_readlane(r.T0, lane),
            __builtin_amdgcn_readlane(r.T, lane), __builtin_amdgcn_readlane(r.F, lane)};
}

// Over the lanes up to this one: inside rows of 16, then from row to row.
template <class Op>
__device__ __forceinline__ int scan(int x, Op &&op) {  // op(0, x) == x for x >= 0
#define SA_SCAN_STEP(ctrl, rows) x = op(__builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false), x)
    SA_SCAN_STEP(0x111, 0xf);  // row_shr:1
    SA_SCAN_STEP(0x112, 0xf);
    SA_SCAN_STEP(0x114, 0xf);
    SA_SCAN_STEP(0x118, 0xf);
    SA_SCAN_STEP(0x142, 0xa);  // row_bcast:15 to rows 1 and 3
    SA_SCAN_STEP(0x143, 0xc);  // row_bcast:31 to rows 2 and 3
#undef SA_SCAN_STEP
    return x;
}

// all_arrived for up to kPagedMostParts workgroups, whose words a wave looks at 64 at a time.
__device__ __forceinline__ bool parts_arrived(uint64_t *words, uint64_t tag, int mine, int n) {
    if (n <= 64) return all_arrived(words, tag, mine, n);
    const int lane = threadIdx.x & 63;
    const HandOver h(words, 8u * (uint32_t)n);
    const u32x2 set = {(uint32_t)tag, (uint32_t)(tag >> 32)};
    if (lane == 0) h.put(8u * (uint32_t)mine, __builtin_bit_cast(f32x2, set));
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    bool there = true;
    for (int at = 0; at < n; at += 64) {
        const u32x2 seen = __builtin_bit_cast(u32x2, h.get2(8u * (uint32_t)min(at + lane, n - 1)));
        there = there && seen.x == set.x && seen.y == set.y;
    }
    const bool all = __builtin_amdgcn_ballot_w64(there) == ~0ull;
    for (int at = lane; all && at < n; at += 64) h.put(8u * (uint32_t)at, f32x2{0.f, 0.f});
    return all;
}

// The products of a tile of ROWS query rows, S^T = K Q^T (32 keys) and O^T += V^T P^T, on 32 x 32 or 16 x 16 matrix instructions.
// A lane has its row's share: row lane % ROWS, group lane / ROWS.
// FAR: K and V are read once by the launch, past the caches (6.3 against 5.7 TB/s at 32 sequences of up to 32768 keys); not where
// several tiles of rows read them.
template <bool FAR, class T>
__device__ __forceinline__ T load(const uint8_t *at) {
    if constexpr (FAR) return __builtin_nontemporal_load((const T *)at);
    else return *(const T *)at;
}
template <int DT, int ND, int ROWS, bool FAR>
struct Tile;
template <int DT, int ND, bool FAR>
struct Tile<DT, ND, 32, FAR> {
    using E = Elem<DT>;
    static constexpr int NS = 16, NQ = 2 * ND, NA = 16 * ND;  // scores, registers of 8 queries' elements, output elements
    static __device__ __forceinline__ int d_of_q(int i, int g) { return 32 * (i >> 1) + 16 * g + 8 * (i & 1); }
    static __device__ __forceinline__ int key(int e, int g) { return 8 * (e >> 2) + 4 * g + (e & 3); }
    static __device__ __forceinline__ int d_of(int e, int g) { return 32 * (e >> 4) + 8 * ((e & 15) >> 2) + 4 * g + (e & 3); }
    struct Operands {
        u32x4 k[ND], v[ND];
    };
    static __device__ __forceinline__ void load_k(Operands &c, const uint8_t *k, int lane) {
#pragma unroll
        for (int d = 0; d < ND; d++) c.k[d] = load<FAR, u32x4>(k + 1024 * d + 16 * lane);
    }
    static __device__ __forceinline__ void load_v(Operands &c, const uint8_t *v, int lane) {
#pragma unroll
        for (int d = 0; d < ND; d++) c.v[d] = load<FAR, u32x4>(v + 1024 * d + 16 * lane);
    }
    static __device__ __forceinline__ void scores(const Operands &c, const u32x4 (&q)[NQ], float (&s)[NS]) {
        f32x16 x;
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = 0.f;
#pragma unroll
        for (int i = 0; i < NQ; i++) x = E::mfma(Codes<DT>::take(c.k[i >> 1][2 * (i & 1)], c.k[i >> 1][2 * (i & 1) + 1], 1.0f), q[i], x);
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = x[e];
    }
    f32x16 acc[ND];
    // f(register of four codes) for every one
    template <class F>
    static __device__ __forceinline__ void each_v(Operands &c, F &&f) {
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) f(c.v[d], e);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[d][e] = 0.f;
    }
    __device__ __forceinline__ void scale(float a) {
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[d][e] *= a;
    }
    __device__ __forceinline__ void add(const Operands &c, const uint32_t (&pw)[NS / 2], float vs) {
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
            const u32x4 pk4 = u32x4{pw[4 * kc], pw[4 * kc + 1], pw[4 * kc + 2], pw[4 * kc + 3]};
#pragma unroll
            for (int d = 0; d < ND; d++) acc[d] = E::mfma(Codes<DT>::take(c.v[d][kc], c.v[d][2 + kc], vs), pk4, acc[d]);
        }
    }
    // Rows that attend to a NaN become NaN, the NaN codes 0.  att: 1 where the row attends.
    __device__ __forceinline__ void poison(Operands &c, const uint32_t (&att)[NS / 2]) {
#pragma unroll
        for (int d = 0; d < ND; d++) {
            f32x16 hits;
#pragma unroll
            for (int e = 0; e < 16; e++) hits[e] = 0.f;
#pragma unroll
            for (int kc = 0; kc < 2; kc++) {
                const u32x4 at4 = u32x4{att[4 * kc], att[4 * kc + 1], att[4 * kc + 2], att[4 * kc + 3]};
                hits = E::mfma(Codes<DT>::take(nan_ones(c.v[d][kc]), nan_ones(c.v[d][2 + kc]), 1.0f), at4, hits);
            }
#pragma unroll
            for (int e = 0; e < 16; e++) acc[d][e] = hits[e] > 0.f ? __builtin_nanf("") : acc[d][e];
#pragma unroll
            for (int e = 0; e < 4; e++) c.v[d][e] = no_nan(c.v[d][e]);
            __builtin_amdgcn_sched_barrier(0);  // (one tile's registers at a time)
        }
    }
    __device__ __forceinline__ float get(int e) const { return acc[e >> 4][e & 15]; }
    static __device__ __forceinline__ float row_max(float x) { return half_swap_max(x); }
    static __device__ __forceinline__ float row_sum(float x) { return x + __shfl_xor(x, 32); }
};
template <int DT, int ND, bool FAR>
struct Tile<DT, ND, 16, FAR> {
    using E = Elem<DT>;
    static constexpr int NS = 8, NQ = ND, NA = 8 * ND;
    static __device__ __forceinline__ int d_of_q(int i, int g) { return 64 * (i >> 1) + 16 * g + 8 * (i & 1); }
    static __device__ __forceinline__ int key(int e, int g) { return 16 * (e >> 2) + 4 * g + (e & 3); }
    static __device__ __forceinline__ int d_of(int e, int g) { return 16 * (e >> 2) + 4 * g + (e & 3); }
    struct Operands {
        u32x4 k[ND];      // [16 keys][64 d]
        u32x2 v[2 * ND];  // [16 d]
    };
    static __device__ __forceinline__ void load_k(Operands &c, const uint8_t *k, int lane) {
        const int l = lane & 15, g = lane >> 4;
        k += 1024 * (g >> 1) + 16 * (32 * (g & 1) + l);
#pragma unroll
        for (int i = 0; i < ND; i++) c.k[i] = load<FAR, u32x4>(k + 2048 * (i >> 1) + 256 * (i & 1));
    }
    static __device__ __forceinline__ void load_v(Operands &c, const uint8_t *v, int lane) {
        const int l = lane & 15, g = lane >> 4;
        v += 16 * (32 * (g & 1) + l) + 8 * (g >> 1);
#pragma unroll
        for (int i = 0; i < 2 * ND; i++) c.v[i] = load<FAR, u32x2>(v + 1024 * (i >> 1) + 256 * (i & 1));
    }
    static __device__ __forceinline__ void scores(const Operands &c, const u32x4 (&q)[NQ], float (&s)[NS]) {
        f32x4 x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < NQ; i++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const u32x4 k = c.k[2 * (i >> 1) + t];
                x[t] = E::mfma16(Codes<DT>::take(k[2 * (i & 1)], k[2 * (i & 1) + 1], 1.0f), q[i], x[t]);
            }
#pragma unroll
        for (int e = 0; e < 8; e++) s[e] = x[e >> 2][e & 3];
    }
    f32x4 acc[2 * ND];
    template <class F>
    static __device__ __forceinline__ void each_v(Operands &c, F &&f) {
#pragma unroll
        for (int d = 0; d < 2 * ND; d++)
#pragma unroll
            for (int e = 0; e < 2; e++) f(c.v[d], e);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int d = 0; d < 2 * ND; d++) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void scale(float a) {
#pragma unroll
        for (int d = 0; d < 2 * ND; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[d][e] *= a;
    }
    __device__ __forceinline__ void add(const Operands &c, const uint32_t (&pw)[NS / 2], float vs) {
        const u32x4 pk4 = u32x4{pw[0], pw[1], pw[2], pw[3]};
#pragma unroll
        for (int d = 0; d < 2 * ND; d++) acc[d] = E::mfma16(Codes<DT>::take(c.v[d].x, c.v[d].y, vs), pk4, acc[d]);
    }
    __device__ __forceinline__ void poison(Operands &c, const uint32_t (&att)[NS / 2]) {
        const u32x4 at4 = u32x4{att[0], att[1], att[2], att[3]};
#pragma unroll
        for (int d = 0; d < 2 * ND; d++) {
            const f32x4 hits = E::mfma16(Codes<DT>::take(nan_ones(c.v[d].x), nan_ones(c.v[d].y), 1.0f), at4, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int e = 0; e < 4; e++) acc[d][e] = hits[e] > 0.f ? __builtin_nanf("") : acc[d][e];
            c.v[d].x = no_nan(c.v[d].x);
            c.v[d].y = no_nan(c.v[d].y);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    __device__ __forceinline__ float get(int e) const { return acc[e >> 2][e & 3]; }
    static __device__ __forceinline__ float row_max(float x) {
        const uint32_t u = __float_as_uint(x);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        return half_swap_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
    }
    static __device__ __forceinline__ float row_sum(float x) {
        x += __shfl_xor(x, 16);
        return x + __shfl_xor(x, 32);
    }
};

// Where there are many units (kPagedFewUnits), a launch in front finds the share and where every unit begins in the row, divided by the unit's planes.
constexpr int kUnitThreads = 1024;
template <bool LISTS>
__global__ __launch_bounds__(kUnitThreads) void paged_units_kernel(const PagedDecodeParams p, const int groups) {
    __shared__ int sums[2][kUnitThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int U = LISTS ? p.t.B * p.c.H : p.t.B;
    const unsigned M = LISTS ? p.RT : (unsigned)p.c.H * p.RT;
    const int per = (U + kUnitThreads - 1) / kUnitThreads, u0 = min(tid * per, U), u1 = min(u0 + per, U);
    const auto plus = [](int a, int x) { return a + x; };
    const auto most = [](int a, int x) { return max(a, x); };
    // (of all threads, and of those in front of this one)
    auto over = [&](int x, auto &&op, int *all, int &total) {
        const int up = scan(x, op);
        if (lane == 63) all[wave] = up;
        __syncthreads();
        const int waves = scan(lane < kUnitThreads / 64 ? all[lane] : 0, op);
        total = __builtin_amdgcn_readlane(waves, 63);
        __syncthreads();
        return up - x + (wave == 0 ? 0 : __builtin_amdgcn_readlane(waves, max(wave - 1, 0)));
    };
    int sum = 0, longest = 0, total;
#pragma unroll 8
    for (int u = u0; u < u1; u++) {
        const int T = max(unit_of<LISTS>(p, u).T, 1);
        p.units->first[u] = (unsigned)T;
        sum += T;
        longest = max(longest, T);
    }
    over(sum, plus, sums[0], total);
    over(longest, most, sums[1], longest);
    const PagedShare share = paged_share((unsigned)total * M, U * M, groups, (unsigned)longest, (unsigned)p.parts, kPagedWaves / p.tiles);
    sum = 0;
    for (int u = u0; u < u1; u++) sum += (int)paged_row_length(share, p.units->first[u]);
    unsigned at = (unsigned)over(sum, plus, sums[0], total);
    for (int u = u0; u < u1; u++) {
        const unsigned n = paged_row_length(share, p.units->first[u]);
        p.units->first[u] = at;
        at += n;
    }
    if (tid == 0) {
        p.units->cuts = share.cuts;
        p.units->share = share.share;
        p.units->total = (unsigned)total * M;
    }
}

// What says which keys a row attends to: causality and window, lists, or a tree of the last tokens.
enum Who { kCausal, kLists, kTree };
// TILES: of rows that a workgroup has, kWaves / TILES waves each, which take chunks in turn.  Several read the same K and V at about the same time, from the
// caches (8 trees of 64 nodes, 8 x 4 heads, over up to 65536 keys, D = 64, fp16: 514 us with one, 369 with four, 653 TFLOP/s).  What is left then (us of these trees and of
// 25-node ones of 32 sequences up to 8192 keys, D = 128, found by leaving each out in a copy): codes to 16 bits 72 and 9, exponentials 40 and 7, parts of planes 2 and 16.
// Not kept: blocks fetched into LDS once for all tiles, four ahead (both as fast as from the caches), products of K in two sums (2 to 8 % slower).
template <int DT, int ND, int ROWS, bool FAR, int WHO, int TILES>
__global__ __launch_bounds__(kWaves * 64, paged_occupancy(ND, ROWS, TILES)) void paged_decode_kernel(const PagedDecodeParams p) {
    constexpr bool LISTS = WHO == kLists, TREE = WHO == kTree;
    using E = Elem<DT>;
    using X = Tile<DT, ND, ROWS, FAR>;
    constexpr int D = 32 * ND, PST = D + kPagedRowPad;
    constexpr int TURNS = kWaves / TILES, PLANE = ROWS * TILES;  // waves that take turns, rows of a plane
    extern __shared__ __attribute__((aligned(16))) float part[];  // [waves][ROWS][PST]
    const int tid = threadIdx.x, lane = tid & 63, lrow = lane & (ROWS - 1), lgrp = lane / ROWS;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), turn = wave / TILES, tile = wave % TILES;
    const int lP = p.c.lper + 5, sub_mask = (1 << p.c.lper) - 1;
    // What is read from the argument block where it is used: hoisted out of the loop over the segments, the strides of everything had
    // the inner loop's scalars spilled.
    typedef const __attribute__((address_space(4))) PagedDecodeParams *ArgPtr;
    auto late = [] {
        ArgPtr a = (ArgPtr)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(a));
        return a;
    };
    auto by_rows = [&](int row) { return p.Sq == 1 ? row : row / p.Sq; };  // (a division costs as much as a step of the scan)

    // ---- this workgroup's piece [x0, x1) of the row, and the unit it starts in (the host: a row is at most 2^30 chunks) ----
    const int U = LISTS ? p.t.B * p.c.H : p.t.B;                // units
    const unsigned M = LISTS ? p.RT : (unsigned)p.c.H * p.RT;  // planes of each
    PagedShare share;
    unsigned total;
    auto length = [&](int chunks) __attribute__((always_inline)) { return paged_row_length(share, (unsigned)max(chunks, 1)); };  // in the row
    // (few units: lane l has units l, 64 + l, ...; in the row: a unit, the units up to it)
    constexpr int NB = kPagedFewUnits(LISTS) / 64;
    Unit own[NB], unit;
    int mine[NB], upto[NB];
    const bool few = p.units == nullptr;
    if (few) {
        int sum = 0, longest = 0;
        const auto plus = [](int a, int x) { return a + x; };
#pragma unroll
        for (int k = 0; k < NB; k++)
            if (k == 0 || 64 * k < U) own[k] = unit_of<LISTS>(p, min(64 * k + lane, U - 1));
#pragma unroll
        for (int k = 0; k < NB; k++)
            if (k == 0 || 64 * k < U) {
                mine[k] = 64 * k + lane < U ? max(own[k].T, 1) : 0;
                upto[k] = sum + scan(mine[k], plus);
                sum = __builtin_amdgcn_readlane(upto[k], 63);
                longest = max(longest, mine[k]);
            }
        longest = __builtin_amdgcn_readlane(scan(longest, [](int a, int x) { return max(a, x); }), 63);
        share = paged_share((unsigned)sum * M, U * M, gridDim.x, (unsigned)longest, (unsigned)p.parts, TURNS);
        if (share.cuts) {
            sum = 0;
#pragma unroll
            for (int k = 0; k < NB; k++)
                if (k == 0 || 64 * k < U) {
                    mine[k] = 64 * k + lane < U ? (int)length(own[k].T) : 0;
                    upto[k] = sum + scan(mine[k], plus);
                    sum = __builtin_amdgcn_readlane(upto[k], 63);
                }
        } else {
#pragma unroll
            for (int k = 0; k < NB; k++) {
                mine[k] += 64 * k + lane < U ? (int)kPagedComing : 0;
                upto[k] += min(64 * k + lane + 1, U) * (int)kPagedComing;
            }
            sum += U * (int)kPagedComing;
        }
        total = (unsigned)sum * M;
    } else {
        share = {p.units->cuts != 0u, p.units->share};
        total = p.units->total;
    }
    const bool cuts = share.cuts;
    const int me = paged_piece(blockIdx.x, cuts ? total : gridDim.x);
    if (me < 0) return;
    const unsigned piece = cuts ? 1u : share.share, x0 = piece * me, x1 = min(x0 + piece, total);
    if (x0 >= total) return;
    int u = 0;
    unsigned base;  // of unit u
    if (few) {
        // the block of 64 units and the lane whose unit holds x0
        int k = 0;
#pragma unroll
        for (int i = 1; i < NB; i++)
            if (64 * i < U && x0 >= (unsigned)__builtin_amdgcn_readlane(upto[i - 1], 63) * M) k = i;
        unit = own[0];
        int to = upto[0], n = mine[0];
#pragma unroll
        for (int i = 1; i < NB; i++)
            if (k == i) {
                unit = own[i];
                to = upto[i];
                n = mine[i];
            }
        const int at = __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64(x0 < (unsigned)to * M)) - 1;
        u = 64 * k + at;
        base = (unsigned)__builtin_amdgcn_readlane(to - n, at) * M;
        unit = of_lane(unit, at);
    } else {
        u = paged_find_unit(U, [&](int from, int step, int left) {
            return __popcll(__builtin_amdgcn_ballot_w64(lane * step < left && p.units->first[min(from + lane * step, U - 1)] * M <= x0));
        });
        u = __builtin_amdgcn_readfirstlane(u);
        base = (unsigned)__builtin_amdgcn_readfirstlane((int)p.units->first[u]) * M;
        unit = of_lane(unit_of<LISTS>(p, u), 0);
    }

    // Of the workgroups of a compute unit the oldest goes first and is done when others have a third of their piece left; so the
    // further a workgroup is, the lower its priority.
    __builtin_amdgcn_s_setprio(3);
    unsigned x = x0, lower_at = share.share / 4;
    int quarter = 0;
    while (x < x1) {
        const unsigned done = cuts ? 0u : x - x0;
        const unsigned T = (unsigned)max(unit.T, 1), row_T = length(unit.T);
        const unsigned m = M == 1 ? 0u : (x - base) / row_T, plane_at = base + m * row_T;  // in the row
        x += paged_coming(share, x - plane_at);
        if (x >= x1) break;
        const unsigned at_row = x - plane_at;
        const PagedSegment seg = paged_segment(share, T, row_T, at_row, x1 - x);
        const int off = seg.off, n = seg.n;  // chunks off .. off + n - 1 of this plane
        const int b = LISTS ? u / p.c.H : u, hr = LISTS ? (u - b * p.c.H) * p.RT + (int)m : (int)m;
        const int h = p.RT == 1 ? hr : hr / p.RT, rt = hr - h * p.RT;
        const int plane = (b * p.c.H + h) * p.RT + rt;
        x += cuts ? 1 : n;
        if (m + 1 == M && x - plane_at == row_T) {
            base += row_T * M;
            u++;
        }
        const int len = unit.len, cnt = unit.cnt, T0 = unit.T0, F = unit.F;
        const bool keys = unit.T > 0;
        if (x < x1 && x == base) unit = of_lane(unit_of<LISTS>(p, u), 0);  // (the next segment's)
        // this lane's row: query i of query head g
        const int row = PLANE * rt + ROWS * tile + lrow, g = by_rows(row), i = row - g * p.Sq;
        const bool live = row < p.R && i < cnt;
        // without lists it sees the keys from `lo` to `hi`
        int hi = len - cnt + i, lo = p.window > 0 ? hi - p.window + 1 : 0;
        // of a tree the keys in front of its nodes from `lo` on, and those of the nodes in `above`
        uint64_t above = 0ull;
        if constexpr (TREE) {
            const int base = len - cnt;
            if (p.window > 0 || 32 * (T0 + off + n) > base) {
                const ArgPtr a = late();
                const uint64_t nodes = tree_ancestors(a->parents + b * a->parents_stride[0], a->parents_stride[1], cnt, lane);
                above = __shfl((unsigned long long)nodes, live ? i : 0);
                if (p.window > 0) {
                    const int depth = __popcll(above) - 1;
                    lo = min(base, base + depth - p.window + 1);
                    for (int far = depth + 1 - p.window; far > 0; far--) above &= above - 1;  // (ancestors' numbers are lower)
                }
            }
            hi = base - 1;
        }

        u32x4 qf[X::NQ];
        {
            const ArgPtr a = late();
            const uint16_t *qp = a->q + b * a->qs[0] + (live ? (h * a->G + g) * a->qs[1] + i * a->qs[2] : 0);
#pragma unroll
            for (int c = 0; c < X::NQ; c++) qf[c] = live && X::d_of_q(c, lgrp) < p.c.cols ? *(const u32x4 *)(qp + X::d_of_q(c, lgrp)) : u32x4{0u, 0u, 0u, 0u};
        }
        const uint32_t bits_i = (uint32_t)i << (lP - 3);

        float m_ref = 0.f, raise_above = kNegInf, l = 0.f;
        X out_rows;
        out_rows.clear();

        // This wave's chunks are off + turn + TURNS j, j < nw.  Lane j of a round of 64 of them finds where chunk j lies.
        const int nw = TILES > 1 && PLANE * rt + ROWS * tile >= p.R ? 0 : (n - turn + TURNS - 1) / TURNS;
        struct Places {
            int block, tile, slot;  // block of the pool or -1; with lists the tile, and the slot of a PARTIAL one or -1
            float ks, vs;
        };
        auto places = [&](int j0) __attribute__((always_inline)) {
            const ArgPtr a = late();
            int block = -1, at_tile = 0, slot = -1;
            float ks = 0.f, vs = 0.f;
            const int j = j0 + lane;
            const int t = T0 + off + turn + TURNS * j;
            if (j < nw && keys) {
                int tile = t >> p.c.lper;
                if constexpr (LISTS) {
                    if (tile >= F) slot = tile - F;
                    tile = tile < F ? a->full_ids[b * a->fis[0] + h * a->fis[1] + (int64_t)tile * a->fis[2]]
                                    : a->part_ids[b * a->pis[0] + h * a->pis[1] + (int64_t)(tile - F) * a->pis[2]];
                    if (tile < 0 || tile >= a->nK) tile = a->t.width;
                }
                const int sub = t & sub_mask;
                if (tile < a->t.width) {
                    at_tile = tile;
                    const int page = a->t.ids[b * a->t.s0 + tile * a->t.s1];
                    // (nothing attends to keys of a page that does not exist)
                    if ((tile << lP) + (sub << 5) < len && page >= 0 && page < a->c.pages) block = ((page * a->c.H + h) << p.c.lper) + sub;
                }
            }
            if (block >= 0) {
                ks = a->c.k_scales[block];
                vs = a->c.v_scales[block];
            }
            return Places{block, at_tile, slot, ks, vs};
        };
        // What is requested next takes the registers of what has just gone into a product: K of a later chunk is on its way during the
        // softmax and the second product, V behind it.  At D = 64 two chunks are under way, as their bytes are half as many; with
        // more registers for more there would be fewer waves, which hide as much.  Tiles that share K and V find them in the caches, and have a third
        // wave per SIMD instead (419 -> 406 us when this was tried).
        constexpr int PRE = ND == 2 && TILES == 1 ? 2 : 1;
        struct Chunk {
            int block, key0, slot;
            uint32_t bits;
        };
        auto chunk = [&](const Places &at, int j) __attribute__((always_inline)) {
            const int in = min(j, nw - 1) & 63, t = T0 + off + turn + TURNS * min(j, nw - 1);
            const int block = __builtin_amdgcn_readlane(at.block, in);
            Chunk c{j < nw ? block : -1, t << 5, -1, 0u};
            if constexpr (LISTS) {
                c.key0 = (__builtin_amdgcn_readlane(at.tile, in) << lP) + ((t & sub_mask) << 5);
                c.slot = __builtin_amdgcn_readlane(at.slot, in);
                c.bits = *(const uint32_t *)(p.packed + b * p.pks[0] + h * p.pks[1] + ((int64_t)max(c.slot, 0) * p.Sq << (lP - 3)) + ((t & sub_mask) << 2) + bits_i);
            }
            if (c.block < 0) c.key0 = len;  // (no key of it is attended to)
            return c;
        };
        // Of no block, and behind the last chunk, nothing is requested: 64 ragged sequences 102.2 -> 98.3 us, 16 in a window 18.2 -> 17.4
        // against that chunk again.  With lists the branch costs more than the pool's first block over and over, which the caches
        // hold: 31.6 | 30.8 us.  Where tiles share a workgroup it does, too: of requests that may not have been made none can be counted, so that K was waited for
        // with V behind it.
        constexpr bool ALWAYS = LISTS || TILES > 1;
        auto request_k = [&](const Chunk &c, typename X::Operands &x) {
            if (ALWAYS || c.block >= 0) X::load_k(x, p.c.k + (int64_t)max(c.block, 0) * (1024 * ND), lane);
        };
        auto request_v = [&](const Chunk &c, typename X::Operands &x) {
            if (ALWAYS || c.block >= 0) X::load_v(x, p.c.v + (int64_t)max(c.block, 0) * (1024 * ND), lane);
        };
        // (of the round of 64 chunks that is requested: their places; of the round behind it, on their way; of the round at hand: scales)
        // (There: scales that may still be on their way where the loop begins are waited for at every step, and with them all that has been requested since.  With this and the
        // requests that are always made 25-node trees of 32 sequences up to 8192, D = 128: 137 -> 124 us; 64 nodes, 8 up to 65536, D = 64: 410 -> 369.)
        auto there = [](Places &at) __attribute__((always_inline)) {
            if constexpr (TILES > 1) asm volatile("" : "+v"(at.ks), "+v"(at.vs));
        };
        Places here = places(0), next = places(64);
        there(here);
        there(next);
        float ks_at = 0.f, vs_at = 0.f;
        typename X::Operands ops[PRE] = {};  // (codes of 0 where nothing is requested)
        Chunk under_way[PRE];
        if (nw > 0)
            static_for<PRE>([&](auto i) {
                under_way[i] = chunk(here, i);
                request_k(under_way[i], ops[i]);
                request_v(under_way[i], ops[i]);
            });
        auto step = [&](int j, Chunk &c, typename X::Operands &x) __attribute__((always_inline)) {
            if (done + (unsigned)TURNS * j >= lower_at) {
                lower_at += share.share / 4;
                quarter++;
                if (quarter == 1) __builtin_amdgcn_s_setprio(2);
                else if (quarter == 2) __builtin_amdgcn_s_setprio(1);
                else if (quarter == 3) __builtin_amdgcn_s_setprio(0);
            }
            if ((j & 63) == 0) {
                ks_at = here.ks;
                vs_at = here.vs;
            }
            const float ks = positive(scale_of(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_at), j & 63))) * p.scale);
            float vs = scale_of(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs_at), j & 63)));
            const int jn = j + PRE;
            if ((jn & 63) == 0 && jn < nw) {
                here = next;
                next = places(jn + 64);  // (none behind the last chunk)
                there(next);
            }
            const Chunk nc = chunk(here, jn);
            const int key0 = c.key0;
            float s[X::NS];
            X::scores(x, qf, s);
            request_k(nc, x);

            // which keys the lane's row attends to, key k in bit k; `cut`: not all of them for every row
            // (a chunk that does not exist goes through as one that no row attends to: a way around it doubles the registers)
            const int left = len - key0;
            uint32_t see = ~0u;
            bool cut = left < 32;
            if (cut) see = (1u << left) - 1u;
            if constexpr (LISTS) {
                if (c.slot >= 0) {
                    cut = true;
                    see &= c.bits;
                }
            } else if constexpr (TREE) {
                if (key0 + 31 >= len - cnt || (p.window > 0 && key0 <= len - 1 - p.window)) {
                    cut = true;
                    const int in_front = hi + 1 - key0, from = lo - key0;  // bits from .. in_front - 1, and the nodes' behind
                    const uint32_t nodes = in_front > 0 ? in_front > 31 ? 0u : (uint32_t)above << in_front : (uint32_t)(above >> (-in_front & 63));
                    see &= nodes | (in_front >= 32 ? ~0u : in_front > 0 ? (1u << in_front) - 1u : 0u);
                    see = from > 31 ? 0u : from > 0 ? see & ~((1u << from) - 1u) : see;
                }
            } else {
                if (key0 + 31 > len - cnt || (p.window > 0 && key0 <= len - 1 - p.window)) {
                    cut = true;
                    const int last = hi - key0, from = lo - key0;  // bits from .. last
                    see = last < 0 ? 0u : see & (last >= 31 ? ~0u : (2u << last) - 1u);
                    see = from > 31 ? 0u : from > 0 ? see & ~((1u << from) - 1u) : see;
                }
            }
            if (cut) {
#pragma unroll
                for (int e = 0; e < X::NS; e++)
                    if (((see >> X::key(e, lgrp)) & 1u) == 0u) s[e] = kNegInf;
            }
            float mx = kNegInf;
#pragma unroll
            for (int e = 0; e < X::NS; e++) mx = fmaxf(mx, s[e]);
            mx = X::row_max(mx) * ks;
            const float rel = mx - m_ref;
            const bool raise = rel > raise_above;  // false for rows without an attended key so far (mx = -inf)
            if (__builtin_amdgcn_ballot_w64(raise) != 0ull) {
                const float a = raise ? (raise_above == kMaxSlack ? __builtin_amdgcn_exp2f(-rel) : 0.f) : 1.f;
                m_ref = raise ? mx : m_ref;
                raise_above = raise ? kMaxSlack : raise_above;
                l *= a;
                out_rows.scale(a);
            }
            // The reference value is a rounded score, the fma's product is not: beyond 2^24 they differ by more than 1, and the weight of a row's largest
            // score would be anything.  There the products are rounded too.
            float by = ks;
            if (__builtin_amdgcn_ballot_w64(__builtin_fabsf(m_ref) > 16777216.f) != 0ull) {
                by = 1.f;
#pragma unroll
                for (int e = 0; e < X::NS; e++) s[e] *= ks;
            }
            uint32_t pw[X::NS / 2];
#pragma unroll
            for (int e = 0; e < X::NS; e += 2) {
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], by, -m_ref)), z = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e + 1], by, -m_ref));
                l += y + z;
                pw[e >> 1] = E::pack2(y, z);
            }
            // A value that is NaN reaches the rows that attend to it and no others: 0 * NaN would be NaN in the product.  Looked
            // for where some row leaves a key out.
            if (cut) {
                uint32_t any = 0u;
                X::each_v(x, [&](auto &v, int e) { any |= nan_bytes(v[e]); });
                if (__builtin_amdgcn_ballot_w64(any != 0u) != 0ull) {
                    uint32_t att[X::NS / 2];  // 1 where the row attends to the key
#pragma unroll
                    for (int e = 0; e < X::NS; e += 2)
                        att[e >> 1] = E::pack2((see >> X::key(e, lgrp)) & 1u ? 1.f : 0.f, (see >> X::key(e + 1, lgrp)) & 1u ? 1.f : 0.f);
                    out_rows.poison(x, att);
                }
            }
            if (DT == 1 && vs > kFp16Scale) vs = within_fp16(vs, [&](auto &&f) { X::each_v(x, [&](auto &v, int e) { v[e] = f(v[e]); }); });
            out_rows.add(x, pw, vs);
            request_v(nc, x);
            c = nc;
        };
        for (int j0 = 0; j0 < nw; j0 += PRE)
            static_for<PRE>([&](auto i) {
                if (j0 + i < nw) step(j0 + i, under_way[i], ops[i]);
            });

        // ---- the waves' parts, added up in LDS ----
        l = X::row_sum(l);
        {
            float *to = part + (wave * ROWS + lrow) * PST;
#pragma unroll
            for (int e = 0; e < X::NA; e += 4) *(f32x4 *)(to + X::d_of(e, lgrp)) = f32x4{out_rows.get(e), out_rows.get(e + 1), out_rows.get(e + 2), out_rows.get(e + 3)};
            // (a row whose only scores are NaN has a sum and no reference value)
            if (lgrp == 0) *(f32x2 *)(to + D) = f32x2{raise_above == kMaxSlack ? m_ref : l == 0.f ? kNegInf : 0.f, l};
        }
        __syncthreads();
        constexpr int LPR = D / 4;  // lanes per row
        const ArgPtr a = late();
        const int rows = min(a->R - PLANE * rt, PLANE);
        struct Sum {
            float M = kNegInf, L = 0.f;
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
        };
        // parts k = 0 .. N - 1 to the sum: their rows' values, reference values and sums
        auto add_to = [](Sum &s, const auto &v, const auto &ml) __attribute__((always_inline)) {
            constexpr int N = sizeof(ml) / sizeof(ml[0]);
            float M = s.M;
#pragma unroll
            for (int k = 0; k < N; k++) M = fmaxf(M, ml[k].x);
            const float a = s.M == kNegInf ? 0.f : __builtin_amdgcn_exp2f(s.M - M);
            s.L *= a;
#pragma unroll
            for (int e = 0; e < 4; e++) s.x[e] *= a;
#pragma unroll
            for (int k = 0; k < N; k++) {
                const float w = ml[k].x == kNegInf ? 0.f : __builtin_amdgcn_exp2f(ml[k].x - M);
                s.L += w * ml[k].y;
#pragma unroll
                for (int e = 0; e < 4; e++) s.x[e] += w * v[k][e];
            }
            s.M = M;
        };
        auto finish = [&](int r, int d0, const Sum &s) __attribute__((always_inline)) {
            const int at = PLANE * rt + r, gg = by_rows(at), ii = at - gg * p.Sq, head = h * a->G + gg;
            const bool none = ii >= cnt || s.L == 0.f;  // (a row of padding may have met a NaN)
            const float inv = 1.f / s.L;
            const f32x4 y = none ? f32x4{0.f, 0.f, 0.f, 0.f} : f32x4{s.x.x * inv, s.x.y * inv, s.x.z * inv, s.x.w * inv};
            if (a->lse != nullptr && d0 == 0)
                a->lse[b * a->lses[0] + head * a->lses[1] + ii * a->lses[2]] =
                    none ? kNegInf : (s.M + __builtin_amdgcn_logf(s.L)) * 0.69314718056f;
            if (d0 < a->c.cols) *(u32x2 *)(a->o + b * a->os[0] + head * a->os[1] + ii * a->os[2] + d0) = u32x2{E::pack2(y.x, y.y), E::pack2(y.z, y.w)};
        };
        const bool whole = n == (int)T;
        const uint32_t row_bytes = PST * 4, part_bytes = (uint32_t)a->part_rows * row_bytes;
        uint8_t *const ws = reinterpret_cast<uint8_t *>(a->ws);
        // a workgroup has at most two parts: of the plane that its piece starts inside of, and of the one that goes on behind it
        const HandOver out(ws + (int64_t)(2 * me + (off == 0 ? 1 : 0)) * part_bytes, whole ? 0u : part_bytes);
        for (int it = tid; it < rows * LPR; it += kWaves * 64) {
            const int r = it / LPR, d0 = 4 * (it - r * LPR);
            f32x4 v[TURNS];
            f32x2 ml[TURNS];
#pragma unroll
            for (int w = 0; w < TURNS; w++) {
                v[w] = *(const f32x4 *)(part + (w * PLANE + r) * PST + d0);
                ml[w] = *(const f32x2 *)(part + (w * PLANE + r) * PST + D);
            }
            Sum s;
            add_to(s, v, ml);
            if (whole) {
                finish(r, d0, s);
            } else {
                out.put(r * row_bytes + 4 * d0, s.x);
                if (d0 == 0) out.put(r * row_bytes + 4 * D, f32x2{s.M, s.L});
            }
        }
        if (!whole) {
            const PagedRange range = paged_range(share, plane_at, row_T);  // the plane's workgroups
            const int g0 = range.first, parts = range.parts;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();  // every wave's rows have been handed over, and LDS has been read
            int *const told = reinterpret_cast<int *>(part + D + 2);  // (behind a row: the sum below leaves it alone)
            if (wave == 0) {
                const bool last = parts_arrived(a->arrivals + plane + g0, a->tag, (int)me - g0, parts);
                if (lane == 0) *told = last;
            }
            __syncthreads();
            const bool last = __builtin_amdgcn_readfirstlane(*told) != 0;
            if (last) {
                const HandOver in(ws + (int64_t)2 * g0 * part_bytes, (uint32_t)(2 * parts) * part_bytes);
                // Every `teams`-th part by the same threads where there are some to spare, 8 parts on their way at a time.
                const int items = rows * LPR, teams = items <= 64 ? 4 : items <= 128 ? 2 : 1;
                for (int it = tid; it < teams * items; it += kWaves * 64) {
                    const int team = it / items, it0 = it - team * items, r = it0 / LPR, d0 = 4 * (it0 - r * LPR);
                    Sum s;
                    for (int k0 = team; k0 < parts; k0 += 8 * teams) {
                        f32x4 v[8];
                        f32x2 ml[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const int at = min(k0 + k * teams, parts - 1);
                            const uint32_t from = (uint32_t)(at == 0 ? 1 : 2 * at) * part_bytes + r * row_bytes;
                            v[k] = in.get4(from + 4 * d0);
                            ml[k] = in.get2(from + 4 * D);
                        }
#pragma unroll
                        for (int k = 0; k < 8; k++)
                            if (k0 + k * teams >= parts) {  // (none there: the last one again, left out)
                                ml[k] = f32x2{kNegInf, 0.f};
                                v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
                            }
                        add_to(s, v, ml);
                    }
                    if (teams == 1) {
                        finish(r, d0, s);
                    } else {
                        float *const to = part + (team * ROWS + r) * PST;
                        *(f32x4 *)(to + d0) = s.x;
                        if (d0 == 0) *(f32x2 *)(to + D) = f32x2{s.M, s.L};
                    }
                }
                if (teams > 1) {
                    __syncthreads();
                    if (tid < items) {
                        const int r = tid / LPR, d0 = 4 * (tid - r * LPR);
                        f32x4 v[4];
                        f32x2 ml[4];
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            const float *const from = part + (min(w, teams - 1) * ROWS + r) * PST;
                            v[w] = *(const f32x4 *)(from + d0);
                            ml[w] = *(const f32x2 *)(from + D);
                            if (w >= teams) {
                                v[w] = f32x4{0.f, 0.f, 0.f, 0.f};
                                ml[w] = f32x2{kNegInf, 0.f};
                            }
                        }
                        Sum s;
                        add_to(s, v, ml);
                        finish(r, d0, s);
                    }
                }
            }
        }
        __syncthreads();  // LDS is free for the next segment
    }
}

template <int DT, int ND, int ROWS, bool FAR, int WHO, int TILES = 1>
hipError_t launch_kind(const PagedDecodeParams &p, hipStream_t stream) {
    constexpr int smem = kWaves * ROWS * (32 * ND + kPagedRowPad) * 4;
    auto kern = paged_decode_kernel<DT, ND, ROWS, FAR, WHO, TILES>;
    static unsigned long long attr_done = 0;
    if (const hipError_t e = allow_dynamic_smem(kern, smem, attr_done); e != hipSuccess) return e;
    if (p.units != nullptr) {
        hipLaunchKernelGGL(paged_units_kernel<WHO == kLists>, dim3(1), dim3(kUnitThreads), 0, stream, p, p.groups);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)p.groups), dim3(kWaves * 64), smem, stream, p);
    return hipGetLastError();
}
template <int DT, int ND, int ROWS, bool FAR>
hipError_t launch_who(const PagedDecodeParams &p, hipStream_t stream) {
    if (p.parents != nullptr) return launch_kind<DT, ND, ROWS, FAR, kTree>(p, stream);
    return p.full_ids != nullptr ? launch_kind<DT, ND, ROWS, FAR, kLists>(p, stream) : launch_kind<DT, ND, ROWS, FAR, kCausal>(p, stream);
}
template <int DT, int ND>
hipError_t launch_rows(const PagedDecodeParams &p, hipStream_t stream) {
    if (p.tiles == 2) return launch_kind<DT, ND, 32, false, kTree, 2>(p, stream);
    if (p.tiles == 4) return launch_kind<DT, ND, 32, false, kTree, 4>(p, stream);
    if (p.plane_rows == 16) return p.RT == 1 ? launch_who<DT, ND, 16, true>(p, stream) : launch_kind<DT, ND, 16, false, kTree>(p, stream);
    return p.RT == 1 ? launch_who<DT, ND, 32, true>(p, stream) : launch_who<DT, ND, 32, false>(p, stream);
}
template <int DT>
hipError_t launch_dim(const PagedDecodeParams &p, hipStream_t stream) {
    if (p.c.D == 64) return launch_rows<DT, 2>(p, stream);
    if (p.c.D == 128) return launch_rows<DT, 4>(p, stream);
    if (p.c.D == 256) return launch_rows<DT, 8>(p, stream);
    return hipErrorInvalidValue;
}

}  // namespace

size_t paged_decode_parts_bytes(int groups, int part_rows, int D) { return (size_t)groups * 2 * part_rows * (D + kPagedRowPad) * 4; }

hipError_t launch_paged_decode(const PagedDecodeParams &p, int dtype, hipStream_t stream) {
    if (dtype == 0) return launch_dim<0>(p, stream);
    if (dtype == 1) return launch_dim<1>(p, stream);
    return hipErrorInvalidValue;
}

}  // namespace sa
