// What the kernels that store into the paged cache share (paged_cache.hip, paged_rotated.hip, paged_keep.hip): conversions between 16-bit values,
// e4m3 codes and scales, a page's place, and the rows of a block stored by one wave.
#pragma once
#include "fwd_common.h"
#include "paged.h"

namespace sa {
namespace {

template <int DT>
struct Half16;  // what a pair of input values is, as bits
typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

template <>
struct Half16<0> {
    static constexpr uint32_t kInf = 0x7f80u;
    // the codes of two pairs, divided by a power of two, in range and finite
    static __device__ __forceinline__ uint32_t codes(uint32_t a, uint32_t b, float scale) {
        i16x2 r = {0, 0};
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, a), scale, false);
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, b), scale, true));
    }
    static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
    static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
    static __device__ __forceinline__ uint32_t cvt_lo(uint32_t w, float s) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false));
    }
    static __device__ __forceinline__ uint32_t cvt_hi(uint32_t w, float s) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true));
    }
};
template <>
struct Half16<1> {
    static constexpr uint32_t kInf = 0x7c00u;
    static __device__ __forceinline__ uint32_t codes(uint32_t a, uint32_t b, float scale) {
        i16x2 r = {0, 0};
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2, a), scale, false);
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2, b), scale, true));
    }
    static __device__ __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w).x; }
    static __device__ __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w).y; }
    static __device__ __forceinline__ uint32_t cvt_lo(uint32_t w, float s) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false));
    }
    static __device__ __forceinline__ uint32_t cvt_hi(uint32_t w, float s) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true));
    }
};

__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 <= e <= 127

// The least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), within the scales' range.
__device__ __forceinline__ int scale_exp(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, kScaleExpMin), kScaleExpMax);
}
__device__ __forceinline__ int exp_of_scale(float s) {
    return min(max((int)((__float_as_uint(s) >> 23) & 0xffu) - 127, kScaleExpMin), kScaleExpMax);
}

// Larger of m and the magnitudes of the finite values of the pair w, as bits (which order like the values).
template <int DT>
__device__ __forceinline__ uint32_t amax2(uint32_t m, uint32_t w) {
    const uint32_t a = w & 0x7fffu, b = (w >> 16) & 0x7fffu;
    m = max(m, a < Half16<DT>::kInf ? a : 0u);
    return max(m, b < Half16<DT>::kInf ? b : 0u);
}
// The larger magnitudes of two pairs, as bits, infinities and NaN among them.
__device__ __forceinline__ uint32_t larger2(uint32_t m, uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
}
// What a value becomes before it is rounded to a code: in range (beyond it only at the largest scale), infinities NaN.
__device__ __forceinline__ float scaled(float x, float inv) {
    const float y = __builtin_amdgcn_fmed3f(x * inv, -448.f, 448.f);
    return __builtin_fabsf(x) < __builtin_inff() ? y : __builtin_nanf("");
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
// Four codes times f <= 1, rounded again.
__device__ __forceinline__ uint32_t again4(uint32_t w, float f) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return codes4(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
}
// The bytes of four codes whose tokens are base .. base + 3 that lie in [a, z), as a mask.
__device__ __forceinline__ uint32_t bytes_in(int base, int a, int z) {
    const int lo = min(max(a - base, 0), 4), hi = min(max(z - base, 0), 4);
    const uint32_t upto = hi >= 4 ? ~0u : (1u << (8 * hi)) - 1u, below = lo >= 4 ? ~0u : (1u << (8 * lo)) - 1u;
    return upto & ~below;
}

// The page of block `blk` of sequence b, or -1.
__device__ __forceinline__ int page_at(const PageTable &t, int b, int slot, int pages) {
    if (slot < 0 || slot >= t.width) return -1;
    const int page = t.ids[b * t.s0 + slot * t.s1];
    return page >= 0 && page < pages ? page : -1;
}
__device__ __forceinline__ int64_t block_at(const PagedPool &c, int page, int h, int sub) {
    return (((int64_t)page * c.H + h) << c.lper) + sub;
}

// The largest of the wave's x >= 0, in all lanes.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#define SA_MAX_STEP(ctrl, rows) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false))
    SA_MAX_STEP(0x111, 0xf);  // row_shr:1
    SA_MAX_STEP(0x112, 0xf);
    SA_MAX_STEP(0x114, 0xf);
    SA_MAX_STEP(0x118, 0xf);
    SA_MAX_STEP(0x142, 0xa);  // row_bcast:15
    SA_MAX_STEP(0x143, 0xc);  // row_bcast:31
#undef SA_MAX_STEP
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

// Rows of a block in LDS, a wave's own: 16 bytes apart from the banks' period, so that the same piece of 16 rows and a row's own
// pieces both fall into different banks.  A wave's operations on LDS take effect in their order; the fence keeps the compiler, which
// sees one lane, to it.
constexpr int kCacheWaves = 4;
template <int ND>
constexpr int row_bytes = 64 * ND + 16;
__device__ __forceinline__ void in_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// One wave stores rows a .. z - 1 of one block of one head, K or V, from 16-bit tokens: row t lies at x + t * row; rows 0 .. held - 1 are there
// already.  The rows come from memory as they lie there, 1 KiB a load, and cross the lanes through LDS (`mine`, 16 rows), 16 at a time.
template <int DT, int ND>
__device__ __forceinline__ void append_block(const PagedPool &c, const uint16_t *x, int64_t row, bool values, int page, int h, int sub, int held, int a, int z,
                                             uint8_t *mine) {
    using X = Half16<DT>;
    constexpr int NG = ND / 2;                   // groups of 64 d
    constexpr int PPR = 4 * ND, RPI = 64 / PPR;  // 16-byte pieces of a row, rows of a load
    constexpr int NL = 32 / RPI;                 // loads of a block
    const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
    u32x4 in[NL];
    const int r0 = lane / PPR, piece = lane % PPR;
#pragma unroll
    for (int i = 0; i < NL; i++) {
        const int r = RPI * i + r0;
        in[i] = u32x4{0u, 0u, 0u, 0u};
        if (r >= a && r < z && 8 * piece < c.cols) in[i] = __builtin_nontemporal_load((const u32x4 *)(x + r * row + 8 * piece));
    }
    if (page < 0) return;
    const int64_t at = block_at(c, page, h, sub);
    uint8_t *const out = (values ? c.v : c.k) + at * (ND * 1024);
    float *const scale = (values ? c.v_scales : c.k_scales) + at;
    const int e_old = held > 0 ? exp_of_scale(*scale) : kScaleExpMin;
    // V of a block that is not all new: what there is, d = 64 g + 2 l32 and the next one
    u32x4 was[2 * NG];
    const bool mixed = values && z - a < 32;
    auto v_at = [&](int g) { return (u32x4 *)(out + 1024 * (2 * g + (l32 >> 4)) + 16 * (32 * hh + 2 * (l32 & 15))); };
    if (mixed) {
#pragma unroll
        for (int g = 0; g < NG; g++) {
            was[2 * g] = v_at(g)[0];
            was[2 * g + 1] = v_at(g)[1];
        }
    }

    // (finite values, as nearly always, go the short way)
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < NL; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) m = larger2(m, in[i][j]);
    m = wave_max(max(m & 0xffffu, m >> 16));
    const bool finite = m < X::kInf;
    if (!finite) {
        m = 0u;
#pragma unroll
        for (int i = 0; i < NL; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) m = amax2<DT>(m, in[i][j]);
        m = wave_max(m);
    }
    const int e = max(e_old, scale_exp(DT == 0 ? __uint_as_float(m << 16) : X::lo(m)));
    const float up = exp2i(e), inv = exp2i(-e);
    const bool plain = finite && e < kScaleExpMax;
    // codes of four values in two pairs
    auto code = [&](uint32_t a, uint32_t b) {
        return plain ? X::codes(a, b, up) : codes4(scaled(X::lo(a), inv), scaled(X::hi(a), inv), scaled(X::lo(b), inv), scaled(X::hi(b), inv));
    };
    const bool grows = held > 0 && e > e_old;
    const float f = exp2i(max(e_old - e, -126));
    if (lane == 0 && (grows || held == 0)) *scale = up;

    u32x4 made[2 * NG];  // codes: of 16 d of a token per piece (K), of 16 tokens of two d (V)
#pragma unroll
    for (int half = 0; half < 2; half++) {  // rows 16 half ..
        if (a >= 16 * half + 16 || z <= 16 * half) continue;
#pragma unroll
        for (int i = 0; i < NL / 2; i++) *(u32x4 *)(mine + (RPI * i + r0) * row_bytes<ND> + 16 * piece) = in[NL / 2 * half + i];
        in_order();
        if (!values) {
            if ((l32 >> 4) == half) {
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    const u32x4 *const from = (const u32x4 *)(mine + (l32 & 15) * row_bytes<ND> + 64 * d + 32 * hh);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        made[d][i] = code(from[i >> 1][2 * (i & 1)], from[i >> 1][2 * (i & 1) + 1]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int i = half; i < 4; i += 2) {
                    uint32_t q[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) q[j] = *(const uint32_t *)(mine + (8 * (i >> 1) + 4 * hh + j) * row_bytes<ND> + 128 * g + 4 * l32);
                    // two tokens of a d in a pair
                    constexpr uint32_t lows = 0x05040100u, highs = 0x07060302u;
                    made[2 * g][i] = code(__builtin_amdgcn_perm(q[1], q[0], lows), __builtin_amdgcn_perm(q[3], q[2], lows));
                    made[2 * g + 1][i] = code(__builtin_amdgcn_perm(q[1], q[0], highs), __builtin_amdgcn_perm(q[3], q[2], highs));
                }
        }
        in_order();
    }

    if (!values) {
        const bool fresh = l32 >= a && l32 < z, old = grows && l32 < held;
#pragma unroll
        for (int d = 0; d < ND; d++) {
            u32x4 *const to = (u32x4 *)(out + 1024 * d + 16 * lane);
            if (fresh) {
                *to = made[d];
            } else if (old) {
                u32x4 u = *to;
#pragma unroll
                for (int i = 0; i < 4; i++) u[i] = again4(u[i], f);
                *to = u;
            }
        }
    } else {
        uint32_t isnew[4], isold[4], any = 0u;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int base = 16 * (i & 1) + 8 * (i >> 1) + 4 * hh;
            isnew[i] = bytes_in(base, a, z);
            isold[i] = grows ? bytes_in(base, 0, held) : 0u;
            any |= isnew[i] | isold[i];
        }
        if (any == 0u) return;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                u32x4 u = made[2 * g + k];
                if (mixed) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t w = was[2 * g + k][i];
                        if (grows) w = (w & ~isold[i]) | (again4(w, f) & isold[i]);
                        u[i] = isnew[i] == 0u ? w : (w & ~isnew[i]) | (u[i] & isnew[i]);
                    }
                }
                v_at(g)[k] = u;
            }
    }
}

}  // namespace
}  // namespace sa
