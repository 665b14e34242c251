// Norms of queries and keys for each head with the position rotation in the same pass, and its gradients, on gfx950 (MI355X).  No counterpart in
// the reference, whose attention takes q and k as they are (sparseattention/sparse_attn_kernel.py:149); the formula and the lanes are in rotate.h.
//
// Backward, with g = the upstream gradient turned back, per row:
//     dx = r w g - x r^3 mean(x w g),   dw = sum over rows of g x r       (without a norm dx = g, and x is not read)
// Everything between the loads and the one rounding at the end is float32.  Bound by memory: every row is read and written once, q and k
// in one launch.  A wave has 64 / LPR tokens and some of their heads, so that the angles, which take as long as four rows, are made once for these.
//
// Measured: 4 x 4096 tokens, 32 + 8 heads, D = 128, bf16, norms: forward 63 us, 5.3 TB/s read and written, backward 86, 5.9, and 5 for the sums of the weights
// (a copy of 1 GiB: 5.1); 2 x 1031 tokens of three axes, 16 + 16 heads, D = 80, fp16: 8.6 us a call, a launch and 21 MB (as
// long with no angles made); 2 x 4096 tokens, float32, norms: forward 55 us, 6.1 TB/s, with the backward 145, 5.8.
// Not kept: rows requested before the angles (no gain); reads past the caches, too (8.6 -> 9.8 us).
#include <algorithm>

#include "rotate.h"

namespace sa {
namespace {

constexpr int kRotateWaves = 4;
constexpr int kFullWaves = 4096;        // waves that fill the device
constexpr int kBackwardGroups = 1024;   // workgroups of a backward at most, which leave a row of sums each

// A wave has 64 / LPR tokens, a row of LPR lanes each, and goes through heads with their angles in registers.
template <int DT, int LPR>
struct WaveRows {
    static constexpr int T = 64 / LPR;
    Columns c;
    bool live;  // whether the lane has a token and columns
    int64_t b, s;
    Turns t;
    __device__ __forceinline__ WaveRows(const RotateParams &p, int group) {
        const int lane = threadIdx.x & 63, l = lane % LPR;
        const int64_t token = (int64_t)group * T + lane / LPR;
        c = columns_of(l, p.D, p.r.R, p.r.interleaved);
        live = c.live && token < (int64_t)p.B * p.S;
        b = live ? (int)token / p.S : 0;
        s = live ? (int)token - (int)b * p.S : 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            t.c[i] = 1.f, t.s[i] = 0.f;
            if (live && c.rot) turn(position_at(p.r, axis_of(p.r, 4 * l + i), b, s), p.r.frequencies[4 * l + i], t.c[i], t.s[i]);
        }
    }
};

template <int DT, int LPR, bool INTER, bool FAR>
__global__ __launch_bounds__(64 * kRotateWaves) void rotate_kernel(const RotateParams p) {
    using E = RowElem<DT>;
    const int id = blockIdx.x * kRotateWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = id / p.splits, h0 = (id - group * p.splits) * p.heads, h1 = min(h0 + p.heads, p.q.H + p.k.H);
    if (h0 >= h1 || (int64_t)group * WaveRows<DT, LPR>::T >= (int64_t)p.B * p.S) return;
    const WaveRows<DT, LPR> w(p, group);
    float wq[2][4], wk[2][4];
    weights_of(p.r.q_weight, p.r.weight_dtype, w.c, wq);
    weights_of(p.r.k_weight, p.r.weight_dtype, w.c, wk);
    const float share = 1.f / (float)p.D;
    auto rows = [&](const RotateRows &r, const void *weight, const float (&ww)[2][4], int a, int z) __attribute__((always_inline)) {
        rotate_rows<DT, LPR, INTER, FAR>((const E *)r.x + w.b * r.xs[0] + w.s * r.xs[2], (E *)r.y + w.b * r.ys[0] + w.s * r.ys[2], r.xs[1], r.ys[1], a, z, w.c, w.live, false, w.t, weight,
                                    ww, share, p.r.eps);
    };
    if (h0 < p.q.H) rows(p.q, p.r.q_weight, wq, h0, min(h1, p.q.H));
    if (h1 > p.q.H) rows(p.k, p.r.k_weight, wk, max(h0 - p.q.H, 0), h1 - p.q.H);
}

template <int DT, int LPR, bool INTER, bool FAR>
__global__ __launch_bounds__(64 * kRotateWaves) void rotate_backward_kernel(const RotateParams p) {
    using E = RowElem<DT>;
    using X = Run4<DT>;
    __shared__ float sums[kRotateWaves][2][8 * LPR];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l = lane % LPR;
    const Columns c = columns_of(l, p.D, p.r.R, p.r.interleaved);
    float wq[2][4], wk[2][4], dwq[2][4] = {}, dwk[2][4] = {};
    weights_of(p.r.q_weight, p.r.weight_dtype, c, wq);
    weights_of(p.r.k_weight, p.r.weight_dtype, c, wk);
    const float share = 1.f / (float)p.D;
    constexpr int T = WaveRows<DT, LPR>::T;
    const int token_groups = (int)(((int64_t)p.B * p.S + T - 1) / T);
    const int64_t items = (int64_t)token_groups * p.splits;
    for (int64_t id = (int64_t)blockIdx.x * kRotateWaves + wave; id < items; id += (int64_t)p.groups * kRotateWaves) {
        const int group = (int)(id / p.splits), h0 = (int)(id - (int64_t)group * p.splits) * p.heads, h1 = min(h0 + p.heads, p.q.H + p.k.H);
        if (h0 >= h1) continue;
        const WaveRows<DT, LPR> w(p, group);
        auto rows = [&](const RotateRows &r, const void *weight, const float (&ww)[2][4], float (&dw)[2][4], int a, int z) __attribute__((always_inline)) {
            const E *const x = (const E *)r.x + w.b * r.xs[0] + w.s * r.xs[2];
            const E *const dy = (const E *)r.dy + w.b * r.dys[0] + w.s * r.dys[2];
            E *const dx = (E *)r.y + w.b * r.ys[0] + w.s * r.ys[2];
            constexpr int U = 2;
            for (int h = a; h < z; h += U) {
                typename X::T in[U][2] = {}, up[U][2] = {};
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (h + u < z && w.live) {
                        load_runs<DT, INTER>(dy + (h + u) * r.dys[1], c, up[u]);
                        if (weight != nullptr) load_runs<DT, INTER>(x + (h + u) * r.xs[1], c, in[u]);
                    }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (h + u >= z) break;
                    float g[2][4];
                    X::floats(up[u][0], g[0]);
                    X::floats(up[u][1], g[1]);
                    if (c.rot) rotate<INTER, true>(g, w.t);
                    if (weight != nullptr) {
                        float f[2][4];
                        X::floats(in[u][0], f[0]);
                        X::floats(in[u][1], f[1]);
                        float along = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; i++) along += f[i >> 2][i & 3] * (ww[i >> 2][i & 3] * g[i >> 2][i & 3]);
                        const float n = row_factor<LPR>(f, share, p.r.eps);
                        const float m = row_total<LPR>(along) * share * n * n;
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float xi = f[i >> 2][i & 3], gi = g[i >> 2][i & 3];
                            if (w.live) dw[i >> 2][i & 3] += gi * (xi * n);  // (n may be infinite where there is no row)
                            g[i >> 2][i & 3] = n * (ww[i >> 2][i & 3] * gi - xi * m);
                        }
                    }
                    if (w.live) store_runs<DT, INTER, FAR>(dx + (h + u) * r.ys[1], c, X::rounded(g[0]), X::rounded(g[1]));
                }
            }
        };
        if (h0 < p.q.H) rows(p.q, p.r.q_weight, wq, dwq, h0, min(h1, p.q.H));
        if (h1 > p.q.H) rows(p.k, p.r.k_weight, wk, dwk, max(h0 - p.q.H, 0), h1 - p.q.H);
    }
    if (p.parts == nullptr) return;
    // over the wave's tokens, then over the waves
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float a = dwq[i >> 2][i & 3], b = dwk[i >> 2][i & 3];
#pragma unroll
        for (int step = LPR; step < 64; step *= 2) {
            a += __shfl_xor(a, step);
            b += __shfl_xor(b, step);
        }
        if (lane < LPR && c.live) {
            sums[wave][0][c.at[i >> 2] + (i & 3)] = a;
            sums[wave][1][c.at[i >> 2] + (i & 3)] = b;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.D; i += 64 * kRotateWaves) {
        const int which = i >= p.D, col = i - which * p.D;
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < kRotateWaves; w++) x += sums[w][which][col];
        p.parts[((int64_t)blockIdx.x * 2 + which) * p.D + col] = x;
    }
}

// The workgroups' sums added up, in their order: 32 columns of one of the weights a workgroup.
constexpr int kWeightThreads = 1024;
__global__ __launch_bounds__(kWeightThreads) void rotate_weights_kernel(const RotateParams p) {
    __shared__ double sums[kWeightThreads / 32][33];
    const int which = blockIdx.y, col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    void *const out = which ? p.k.dw : p.q.dw;
    if (out == nullptr) return;
    double x = 0.0;
    if (col < p.D) {
#pragma unroll 8
        for (int i = part; i < p.groups; i += kWeightThreads / 32) x += p.parts[((int64_t)i * 2 + which) * p.D + col];
    }
    sums[part][threadIdx.x & 31] = x;
    __syncthreads();
    if (part != 0 || col >= p.D) return;
    x = 0.0;
#pragma unroll
    for (int i = 0; i < kWeightThreads / 32; i++) x += sums[i][threadIdx.x];
    if (p.r.weight_dtype == 2) ((float *)out)[col] = (float)x;
    else if (p.r.weight_dtype == 1) ((_Float16 *)out)[col] = (_Float16)(float)x;
    else ((__bf16 *)out)[col] = (__bf16)(float)x;
}

// Outputs of that many bytes go past the caches, for training's sake: what a forward writes there drives out what the backward reads.  us through the caches | past them, 32 + 8 heads,
// D = 128, bf16, norms, inputs that change from call to call, by MiB of outputs (float32 at D = 64 likewise):
//   forward and backward   80 95 | -;        128 159 | 144;   160 188 | 165;   320 350 | 330
//   backward               64 47.5 | 47.5;   96 66 | 63;      128 93 | 81;     192 136 | 133;   256 176 | 172;   512 336 | 331
//   forward                64 29 | 31;       96 39 | 45;      128 51 | 58;     192 86 | 84;     256 114 | 112;   512 216 | 210
//   and its outputs read   64 52 | 59;       96 71 | 80;      128 97 | 108;    192 151 | 160;   256 202 | 212;   512 398 | 401
// (A forward alone would do better with a border of its own, at about 192 MiB, or none where its outputs are read next.)
constexpr int64_t kRotateFar = 128ll << 20;

// Heads are dealt out to as many waves as fill the device, four at least to one, as the angles of its tokens are made once for all of them.
void share_heads(RotateParams &p) {
    const int T = p.D <= 64 ? 8 : p.D <= 128 ? 4 : 2, heads = p.q.H + p.k.H;
    const int64_t groups = ((int64_t)p.B * p.S + T - 1) / T;
    const int64_t want = (kFullWaves + groups - 1) / groups, most = (heads + 3) / 4;
    p.splits = (int)std::min(want, most);
    p.heads = (heads + p.splits - 1) / p.splits;
}

template <class F>
hipError_t with_rows(const RotateParams &p, int dtype, F &&f) {
    const int D = p.D;
    const bool far = (int64_t)p.B * p.S * (p.q.H + p.k.H) * D * (dtype == 2 ? 4 : 2) >= kRotateFar;
    auto stores = [&](auto dt, auto lpr, auto inter) { return far ? f(dt, lpr, inter, std::true_type{}) : f(dt, lpr, inter, std::false_type{}); };
    auto pairs = [&](auto dt, auto lpr) { return p.r.interleaved ? stores(dt, lpr, std::true_type{}) : stores(dt, lpr, std::false_type{}); };
    auto lanes = [&](auto dt) {
        if (D <= 64) return pairs(dt, std::integral_constant<int, 8>{});
        if (D <= 128) return pairs(dt, std::integral_constant<int, 16>{});
        return pairs(dt, std::integral_constant<int, 32>{});
    };
    if (dtype == 0) return lanes(std::integral_constant<int, 0>{});
    if (dtype == 1) return lanes(std::integral_constant<int, 1>{});
    return lanes(std::integral_constant<int, 2>{});
}

}  // namespace

int64_t rotate_groups(int B, int S, int heads, int D) {
    RotateParams p{};
    p.B = B, p.S = S, p.D = D, p.q.H = heads;
    share_heads(p);
    const int T = D <= 64 ? 8 : D <= 128 ? 4 : 2;
    return (((int64_t)B * S + T - 1) / T * p.splits + kRotateWaves - 1) / kRotateWaves;
}

hipError_t launch_rotate(RotateParams p, int dtype, hipStream_t stream) {
    share_heads(p);
    return with_rows(p, dtype, [&](auto dt, auto lpr, auto inter, auto past) {
        hipLaunchKernelGGL((rotate_kernel<decltype(dt)::value, decltype(lpr)::value, decltype(inter)::value, decltype(past)::value>), dim3((unsigned)rotate_groups(p.B, p.S, p.q.H + p.k.H, p.D)), dim3(64 * kRotateWaves), 0, stream, p);
        return hipGetLastError();
    });
}

int rotate_backward_groups(int B, int S, int heads, int D) { return (int)std::min<int64_t>(rotate_groups(B, S, heads, D), kBackwardGroups); }

hipError_t launch_rotate_backward(RotateParams p, int dtype, hipStream_t stream) {
    share_heads(p);
    p.groups = rotate_backward_groups(p.B, p.S, p.q.H + p.k.H, p.D);
    const hipError_t e = with_rows(p, dtype, [&](auto dt, auto lpr, auto inter, auto past) {
        hipLaunchKernelGGL((rotate_backward_kernel<decltype(dt)::value, decltype(lpr)::value, decltype(inter)::value, decltype(past)::value>), dim3((unsigned)p.groups), dim3(64 * kRotateWaves), 0, stream, p);
        return hipGetLastError();
    });
    if (e != hipSuccess || p.parts == nullptr) return e;
    hipLaunchKernelGGL(rotate_weights_kernel, dim3((p.D + 31) / 32, 2), dim3(kWeightThreads), 0, stream, p);
    return hipGetLastError();
}

}  // namespace sa
