// Attention of few query rows over the 8-bit paged K/V cache on gfx950 (MI355X).
//
// The function is that of sparse_decode.hip (sparse_attention with BLOCK_Q = Sq, sparseattention/sparse_attn_kernel.py:74-146;
// the reference names decode kernels as future work, README.md:65) with K and V read from pages of e4m3 codes
// (paged.h), several query heads per K/V head, and sequences of their own lengths:
//     s = q . k / sqrt(D),  p = exp2(s - m),  o = sum p v / sum p     over the keys that a row attends to.
// The R = G * Sq rows of a K/V head go through the matrix unit together, 32 a tile; codes become bf16 or fp16 (exactly,
// V with its scale) on their way from registers into the products, the scale of K joins the softmax's.  Bound by the
// bytes of K and V, each read once.  Per chunk of 32 keys a wave
//   * has K and V as operands straight from memory (D / 32 loads of 1 KiB each for both: paged.h has the order),
//   * computes S^T = K . Q^T (32 keys x 32 rows), masks, P = exp2(S^T - m), O^T += V^T . P^T.
#include "fwd_common.h"
#include "paged.h"

namespace sa {

namespace {

constexpr int kWaves = 4;

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

__device__ __forceinline__ float scale_of(float s) {  // (as the cache's kernels write them; anything else is brought into range)
    const int e = (int)((__float_as_uint(s) >> 23) & 0xffu);
    return __uint_as_float((uint32_t)min(max(e, 127 + kScaleExpMin), 127 + kScaleExpMax) << 23);
}

template <int DT, int ND, bool LISTS>
__global__ __launch_bounds__(kWaves * 64, ND == 8 ? 1 : 2) void paged_decode_kernel(const PagedDecodeParams p) {
    using E = Elem<DT>;
    constexpr int D = 32 * ND, NC = 2 * ND, PST = D + 2;
    extern __shared__ __attribute__((aligned(16))) float part[];  // [waves][32][PST]
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int plane = (int)(blockIdx.x / (unsigned)p.RT), rt = (int)(blockIdx.x - (unsigned)plane * (unsigned)p.RT);
    const int b = plane / p.c.H, h = plane - b * p.c.H;
    const int lP = p.c.lper + 5;

    const int len = min(max(p.t.lens[b], 0), p.t.width << lP);
    const int cnt = p.counts != nullptr ? min(max(p.counts[b], 0), p.Sq) : p.Sq;
    // this lane's row: query i of query head g
    const int row = 32 * rt + l32, g = row / p.Sq, i = row - g * p.Sq;
    const bool live = row < p.R && i < cnt;
    // without lists it sees the keys from `lo` to `hi`
    const int hi = len - cnt + i, lo = p.window > 0 ? hi - p.window + 1 : 0;

    u32x4 qf[NC];
    {
        const uint16_t *qp = p.q + b * p.qs[0] + (live ? (h * p.G + g) * p.qs[1] + i * p.qs[2] : 0) + 16 * hh;
#pragma unroll
        for (int c = 0; c < NC; c++) qf[c] = live ? *(const u32x4 *)(qp + 32 * (c >> 1) + 8 * (c & 1)) : u32x4{0u, 0u, 0u, 0u};
    }

    const int32_t *fid = nullptr, *pid = nullptr;
    int F = 0, T0 = 0, T1 = 0;  // chunks [T0, T1): of the sequence, or of the list
    if constexpr (LISTS) {
        fid = p.full_ids + b * p.fis[0] + h * p.fis[1];
        pid = p.part_ids + b * p.pis[0] + h * p.pis[1];
        F = min(max(p.full_lens[b * p.fls[0] + h * p.fls[1]], 0), p.nK);
        T1 = (F + min(max(p.part_lens[b * p.pls[0] + h * p.pls[1]], 0), p.nK - F)) << p.c.lper;
        if (cnt == 0) T1 = 0;
    } else if (cnt > 0) {
        T1 = (len + 31) >> 5;
        if (p.window > 0) T0 = max(len - cnt - p.window + 1, 0) >> 5;
    }
    const uint8_t *const bits = LISTS ? p.packed + b * p.pks[0] + h * p.pks[1] + ((int64_t)i << (lP - 3)) : nullptr;

    float m_ref = 0.f, raise_above = -3.0e38f, l = 0.f;
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[d][e] = 0.f;

    for (int t = T0 + wave; t < T1; t += kWaves) {
        int key0, slot = -1;  // first key of the chunk; slot of a PARTIAL tile
        if constexpr (LISTS) {
            const int e = t >> p.c.lper;
            const int tile = __builtin_amdgcn_readfirstlane(e < F ? fid[(int64_t)e * p.fis[2]] : pid[(int64_t)(e - F) * p.pis[2]]);
            if (tile < 0 || tile >= p.nK) continue;
            if (e >= F) slot = e - F;
            key0 = (tile << lP) + ((t & ((1 << p.c.lper) - 1)) << 5);
        } else {
            key0 = t << 5;
        }
        if (key0 >= len) continue;
        const int page = __builtin_amdgcn_readfirstlane(p.t.ids[b * p.t.s0 + (key0 >> lP) * p.t.s1]);
        if (page < 0 || page >= p.c.pages) continue;  // nothing attends to keys of a page that does not exist
        const int64_t at = (((int64_t)page * p.c.H + h) << p.c.lper) + ((key0 >> 5) & ((1 << p.c.lper) - 1));
        const u32x4 *const kp = (const u32x4 *)(p.c.k + at * (1024 * ND)) + lane, *const vp = (const u32x4 *)(p.c.v + at * (1024 * ND)) + lane;
        u32x4 kf[ND], vf[ND];
#pragma unroll
        for (int c = 0; c < ND; c++) kf[c] = kp[64 * c];
#pragma unroll
        for (int c = 0; c < ND; c++) vf[c] = vp[64 * c];
        const float ks = scale_of(p.c.k_scales[at]) * p.scale, vs = scale_of(p.c.v_scales[at]);

        f32x16 s;
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++) s = E::mfma(Codes<DT>::take(kf[c >> 1][2 * (c & 1)], kf[c >> 1][2 * (c & 1) + 1], 1.0f), qf[c], s);

        // which keys the lane's row attends to, key k in bit k; `cut`: not all of them for every row
        uint32_t see = ~0u;
        bool cut = key0 + 32 > len;
        if (cut) see = (1u << (len - key0)) - 1u;
        if constexpr (LISTS) {
            if (slot >= 0) {
                cut = true;
                see &= *(const uint32_t *)(bits + ((int64_t)slot * p.Sq << (lP - 3)) + (((key0 >> 5) & ((1 << p.c.lper) - 1)) << 2));
            }
        } else {
            if (key0 + 31 > len - cnt || (p.window > 0 && key0 <= len - 1 - p.window)) {
                cut = true;
                const int upto = hi - key0, from = lo - key0;  // bits from .. upto
                see = upto < 0 ? 0u : see & (upto >= 31 ? ~0u : (2u << upto) - 1u);
                see = from > 31 ? 0u : from > 0 ? see & ~((1u << from) - 1u) : see;
            }
        }
        if (cut) {
            const uint32_t w = see >> (4 * hh);
#pragma unroll
            for (int e = 0; e < 16; e++)
                if (((w >> (8 * (e >> 2) + (e & 3))) & 1u) == 0u) s[e] = kNegInf;
        }
        float mx = kNegInf;
#pragma unroll
        for (int e = 0; e < 16; e++) mx = fmaxf(mx, s[e]);
        mx = half_swap_max(mx) * ks;
        const float rel = mx - m_ref;
        const bool raise = rel > raise_above;  // false for rows without an attended key so far (mx = -inf)
        if (__builtin_amdgcn_ballot_w64(raise) != 0ull) {
            const float a = raise ? (raise_above == kMaxSlack ? __builtin_amdgcn_exp2f(-rel) : 0.f) : 1.f;
            m_ref = raise ? mx : m_ref;
            raise_above = raise ? kMaxSlack : raise_above;
            l *= a;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[d][e] *= a;
        }
        uint32_t pw[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], ks, -m_ref)), y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e + 1], ks, -m_ref));
            l += x + y;
            pw[e >> 1] = E::pack2(x, y);
        }
        // A value that is NaN reaches the rows that attend to it and no others: 0 * NaN would be NaN in the product.  Looked for
        // where some row leaves a key out.
        if (cut) {
            uint32_t any = 0u;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) any |= nan_bytes(vf[d][e]);
            if (__builtin_amdgcn_ballot_w64(any != 0u) != 0ull) {
                const uint32_t w = see >> (4 * hh);
                uint32_t att[8];  // 1 where the row attends to the key
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const int at0 = 8 * (e >> 2) + (e & 3);
                    att[e >> 1] = E::pack2((w >> at0) & 1u ? 1.f : 0.f, (w >> (at0 + 1)) & 1u ? 1.f : 0.f);
                }
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    f32x16 hits;
#pragma unroll
                    for (int e = 0; e < 16; e++) hits[e] = 0.f;
#pragma unroll
                    for (int kc = 0; kc < 2; kc++) {
                        uint32_t one[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const uint32_t n = nan_bytes(vf[d][2 * kc + e]) >> 7;  // 1 in every NaN byte
                            one[e] = n * 0x38u;                                    // (the code of 1)
                            vf[d][2 * kc + e] &= ~(n * 0xffu);
                        }
                        hits = E::mfma(Codes<DT>::take(one[0], one[1], 1.0f), u32x4{att[4 * kc], att[4 * kc + 1], att[4 * kc + 2], att[4 * kc + 3]}, hits);
                    }
#pragma unroll
                    for (int e = 0; e < 16; e++) acc[d][e] = hits[e] > 0.f ? __builtin_nanf("") : acc[d][e];
                }
            }
        }
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
            const u32x4 pk4 = u32x4{pw[4 * kc], pw[4 * kc + 1], pw[4 * kc + 2], pw[4 * kc + 3]};
#pragma unroll
            for (int d = 0; d < ND; d++) acc[d] = E::mfma(Codes<DT>::take(vf[d][2 * kc], vf[d][2 * kc + 1], vs), pk4, acc[d]);
        }
    }

    // ---- the waves' parts ----
    l += __shfl_xor(l, 32);
    {
        float *mine = part + (wave * 32 + l32) * PST;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) mine[32 * d + 8 * (e >> 2) + 4 * hh + (e & 3)] = acc[d][e];
        if (hh == 0) {
            // (a row whose only scores are NaN has a sum and no reference value)
            mine[D] = raise_above == kMaxSlack ? m_ref : l == 0.f ? kNegInf : 0.f;
            mine[D + 1] = l;
        }
    }
    __syncthreads();
    constexpr int LPR = D / 4;  // lanes per row
    for (int x = tid; x < 32 * LPR; x += kWaves * 64) {
        const int r = x / LPR, d0 = 4 * (x - r * LPR), at = 32 * rt + r;
        if (at >= p.R) break;
        float M = kNegInf, L = 0.f;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < kWaves; w++) M = fmaxf(M, part[(w * 32 + r) * PST + D]);
        if (M != kNegInf)
            for (int w = 0; w < kWaves; w++) {
                const float *pp = part + (w * 32 + r) * PST;
                const float a = pp[D] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(pp[D] - M);
                L += a * pp[D + 1];
#pragma unroll
                for (int e = 0; e < 4; e++) sum[e] += a * pp[d0 + e];
            }
        const int gg = at / p.Sq, ii = at - gg * p.Sq, head = h * p.G + gg;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        if (ii >= cnt) sum = f32x4{0.f, 0.f, 0.f, 0.f};
        if (p.lse != nullptr && d0 == 0)
            p.lse[b * p.lses[0] + head * p.lses[1] + ii * p.lses[2]] =
                ii >= cnt || L == 0.f ? kNegInf : (M + __builtin_amdgcn_logf(L)) * 0.69314718056f;
        *(u32x2 *)(p.o + b * p.os[0] + head * p.os[1] + ii * p.os[2] + d0) = u32x2{E::pack2(sum.x * inv, sum.y * inv), E::pack2(sum.z * inv, sum.w * inv)};
    }
}

template <int DT, int ND, bool LISTS>
hipError_t launch_kind(const PagedDecodeParams &p, hipStream_t stream) {
    constexpr int smem = kWaves * 32 * (32 * ND + 2) * 4;
    auto kern = paged_decode_kernel<DT, ND, LISTS>;
    static unsigned long long attr_done = 0;
    if (const hipError_t e = allow_dynamic_smem(kern, smem, attr_done); e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)p.t.B * p.c.H * p.RT), dim3(kWaves * 64), smem, stream, p);
    return hipGetLastError();
}
template <int DT, int ND>
hipError_t launch_lists(const PagedDecodeParams &p, hipStream_t stream) {
    return p.full_ids != nullptr ? launch_kind<DT, ND, true>(p, stream) : launch_kind<DT, ND, false>(p, stream);
}
template <int DT>
hipError_t launch_dim(const PagedDecodeParams &p, hipStream_t stream) {
    if (p.c.D == 64) return launch_lists<DT, 2>(p, stream);
    if (p.c.D == 128) return launch_lists<DT, 4>(p, stream);
    if (p.c.D == 256) return launch_lists<DT, 8>(p, stream);
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_paged_decode(const PagedDecodeParams &p, int dtype, hipStream_t stream) {
    if (dtype == 0) return launch_dim<0>(p, stream);
    if (dtype == 1) return launch_dim<1>(p, stream);
    return hipErrorInvalidValue;
}

}  // namespace sa
