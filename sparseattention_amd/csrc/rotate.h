// Norm and position rotation of the rows of heads: what rotate.hip and paged_rotated.hip share.
//
// A row x of D values:  y = x * r * w,  r = 1 / sqrt(mean(x^2) + eps)  (or y = x), then of its first R columns the pairs (a, b) at columns
// (j, j + R/2) or, interleaved, (2j, 2j + 1) become  (a cos t - b sin t, a sin t + b cos t),  t = position * frequency of j.
//
// A row is held by LPR lanes, 8 columns each in two runs of 4: columns 4l .. and R/2 + 4l .. where pairs lie R/2 apart, so that a lane has both
// of its four pairs and nothing crosses the lanes but the norm's sum; else 8l .. and 8l + 4 ...  Rows of other tokens are in the wave's other lanes.
#pragma once
#include "fwd_common.h"
#include "rotation.h"

namespace sa {
namespace {

// cos and sin of position * frequency.  Positions reach 2^31 and angles 2^31 radians, of which float32 would keep nothing: the product and its
// remainder of quarter turns are 64 bits wide (off by 2^-24 of a turn at most up to 2^31), what is left of it, an eighth of a turn x at most, 32.
// There the series of sine and cosine end with x^9 and x^10: what follows is less than 2^-28.
__device__ __forceinline__ void turn(double position, double frequency, float &c, float &s) {
#pragma clang fp contract(off)
    const double t = position * frequency * 0.15915494309189533577;  // in turns
    const double quarters = __builtin_rint(4.0 * t);
    const float x = (float)(t - 0.25 * quarters) * 6.283185307f, z = x * x;
    auto fma = [](float a, float b, float c) { return __builtin_fmaf(a, b, c); };
    const float sine = fma(x * z, fma(z, fma(z, fma(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
    const float cosine = fma(z, fma(z, fma(z, fma(z, fma(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
    const int turned = (int)(quarters - 4.0 * __builtin_floor(0.25 * quarters));  // 0 .. 3
    const float a = turned & 1 ? sine : cosine, b = turned & 1 ? cosine : sine;
    c = turned == 1 || turned == 2 ? -a : a;
    s = turned & 2 ? -b : b;
}

template <int DT>
struct Run4 {  // four values in memory
    typedef u32x2 T;
    static __device__ __forceinline__ void floats(T w, float (&x)[4]) {
        if constexpr (DT == 0) {
            x[0] = __uint_as_float(w.x << 16), x[1] = __uint_as_float(w.x & 0xffff0000u);
            x[2] = __uint_as_float(w.y << 16), x[3] = __uint_as_float(w.y & 0xffff0000u);
        } else {
            const uint32_t lo = w.x, hi = w.y;  // (of an element of a vector the bit cast would take the first one)
            const f16x2 a = __builtin_bit_cast(f16x2, lo), b = __builtin_bit_cast(f16x2, hi);
            x[0] = (float)a.x, x[1] = (float)a.y, x[2] = (float)b.x, x[3] = (float)b.y;
        }
    }
    static __device__ __forceinline__ T rounded(const float (&x)[4]) { return T{Elem<DT>::pack2(x[0], x[1]), Elem<DT>::pack2(x[2], x[3])}; }
};
template <>
struct Run4<2> {
    typedef f32x4 T;
    static __device__ __forceinline__ void floats(T w, float (&x)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = w[i];
    }
    static __device__ __forceinline__ T rounded(const float (&x)[4]) { return T{x[0], x[1], x[2], x[3]}; }
};
template <int DT>
using RowElem = std::conditional_t<DT == 2, float, uint16_t>;

// The columns of a lane, l of LPR of its row.
struct Columns {
    bool live, rot;  // whether it has any; whether they are rotated
    int at[2];       // where its two runs of 4 begin
};
__device__ __forceinline__ Columns columns_of(int l, int D, int R, bool interleaved) {
    Columns c;
    c.live = 8 * l < D;
    c.rot = 8 * l < R;
    const bool apart = c.rot && !interleaved;
    c.at[0] = apart ? 4 * l : 8 * l;
    c.at[1] = apart ? R / 2 + 4 * l : 8 * l + 4;
    return c;
}

// A lane's two runs from and to memory: where they lie behind one another, 16 bits wide, in one piece.
template <int DT, bool INTER>
__device__ __forceinline__ void load_runs(const RowElem<DT> *x, const Columns &c, typename Run4<DT>::T (&in)[2]) {
    if constexpr (INTER && DT != 2) {
        const u32x4 w = *(const u32x4 *)(x + c.at[0]);
        in[0] = u32x2{w.x, w.y};
        in[1] = u32x2{w.z, w.w};
    } else {
        in[0] = *(const typename Run4<DT>::T *)(x + c.at[0]);
        in[1] = *(const typename Run4<DT>::T *)(x + c.at[1]);
    }
}
// FAR: past the caches (a number of the kernel: of a choice at run time the compiler makes one store through them).
template <int DT, bool INTER, bool FAR>
__device__ __forceinline__ void store_runs(RowElem<DT> *y, const Columns &c, const typename Run4<DT>::T &a, const typename Run4<DT>::T &b) {
    typedef typename Run4<DT>::T T;
    if constexpr (INTER && DT != 2) {
        const u32x4 w = {a.x, a.y, b.x, b.y};
        if constexpr (FAR) __builtin_nontemporal_store(w, (u32x4 *)(y + c.at[0]));
        else *(u32x4 *)(y + c.at[0]) = w;
    } else if constexpr (FAR) {
        __builtin_nontemporal_store(a, (T *)(y + c.at[0]));
        __builtin_nontemporal_store(b, (T *)(y + c.at[1]));
    } else {
        *(T *)(y + c.at[0]) = a;
        *(T *)(y + c.at[1]) = b;
    }
}

// The sum over the LPR lanes of a row, in all of them.
template <int LPR>
__device__ __forceinline__ float row_total(float x) {
#define SA_ROW_STEP(ctrl) x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), ctrl, 0xf, 0xf, true))
    SA_ROW_STEP(0xb1);   // with the neighbour
    SA_ROW_STEP(0x4e);   // in fours
    SA_ROW_STEP(0x141);  // in eights (mirrored)
    if constexpr (LPR >= 16) SA_ROW_STEP(0x140);
#undef SA_ROW_STEP
    if constexpr (LPR == 32) {
        const uint32_t u = __float_as_uint(x);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return x;
}

// The weights of a lane's columns in float32.
__device__ __forceinline__ void weights_of(const void *w, int dtype, const Columns &c, float (&out)[2][4]) {
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = c.at[k] + i;
            float x = 0.f;
            if (w != nullptr && c.live) {
                if (dtype == 2) x = ((const float *)w)[at];
                else if (dtype == 1) x = (float)((const _Float16 *)w)[at];
                else x = __uint_as_float((uint32_t)((const uint16_t *)w)[at] << 16);
            }
            out[k][i] = x;
        }
}

// A row over its root mean square times its weights.  Here and below the fused products are written out, so that kernels that share these functions give
// the same to the bit.
template <int LPR>
__device__ __forceinline__ float row_factor(const float (&x)[2][4], float share, float eps) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) sum = __builtin_fmaf(x[i >> 2][i & 3], x[i >> 2][i & 3], sum);
    return __builtin_amdgcn_rsqf(__builtin_fmaf(row_total<LPR>(sum), share, eps));
}
template <int LPR>
__device__ __forceinline__ void norm_row(float (&x)[2][4], const float (&w)[2][4], float share, float eps) {
    const float n = row_factor<LPR>(x, share, eps);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i >> 2][i & 3] = x[i >> 2][i & 3] * n * w[i >> 2][i & 3];
}

// cos and sin of the four pairs of a lane.
struct Turns {
    float c[4], s[4];
};
// y in a lane's two runs turned by t; back: by -t.
// (INTER as a number of the kernel: chosen at run time, the runs went through scratch memory)
template <bool INTER, bool BACK>
__device__ __forceinline__ void rotate(float (&y)[2][4], const Turns &t) {
    auto pair = [&](float &a, float &b, float c, float s) __attribute__((always_inline)) {
        const float a0 = a, b0 = b;
        if constexpr (BACK) s = -s;
        a = __builtin_fmaf(a0, c, -(b0 * s));
        b = __builtin_fmaf(a0, s, b0 * c);
    };
    if constexpr (!INTER) {
#pragma unroll
        for (int i = 0; i < 4; i++) pair(y[0][i], y[1][i], t.c[i], t.s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) pair(y[i >> 1][2 * (i & 1)], y[i >> 1][2 * (i & 1) + 1], t.c[i], t.s[i]);
    }
}

__device__ __forceinline__ double position_at(const Rotation &r, int axis, int64_t b, int64_t s) {
    const int64_t at = axis * r.position_strides[0] + b * r.position_strides[1] + s * r.position_strides[2];
    return r.positions_64 ? (double)((const int64_t *)r.positions)[at] : (double)((const int32_t *)r.positions)[at];
}
__device__ __forceinline__ int axis_of(const Rotation &r, int j) { return r.axes != nullptr ? min(max(r.axes[j], 0), r.num_axes - 1) : 0; }

// Heads a .. z - 1 of the tokens at x (and y, where they go): of each `heads` elements apart the lane's columns, normed if there is a weight, and turned.  live: the lane
// has columns of a token; its rows are read, or are 0 where `zero`.
template <int DT, int LPR, bool INTER, bool FAR>
__device__ __forceinline__ void rotate_rows(const RowElem<DT> *x, RowElem<DT> *y, int64_t x_head, int64_t y_head, int a, int z, const Columns &c, bool live, bool zero,
                                            const Turns &t, const void *weight, const float (&w)[2][4], float share, float eps) {
    using X = Run4<DT>;
    constexpr int U = 4;  // heads under way
    for (int h = a; h < z; h += U) {
        typename X::T in[U][2] = {};
#pragma unroll
        for (int u = 0; u < U; u++)
            if (h + u < z && live && !zero) load_runs<DT, INTER>(x + (h + u) * x_head, c, in[u]);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (h + u >= z) break;
            float f[2][4];
            X::floats(in[u][0], f[0]);
            X::floats(in[u][1], f[1]);
            if (weight != nullptr) norm_row<LPR>(f, w, share, eps);
            if (c.rot) rotate<INTER, false>(f, t);
            if (live) {
                const typename X::T none = {};
                store_runs<DT, INTER, FAR>(y + (h + u) * y_head, c, zero ? none : X::rounded(f[0]), zero ? none : X::rounded(f[1]));
            }
        }
    }
}

}  // namespace
}  // namespace sa
