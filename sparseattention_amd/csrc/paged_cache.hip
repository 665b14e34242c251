// The 8-bit paged K/V cache on gfx950 (MI355X): storing tokens, reading them back, copying, forking, compacting and
// listing pages.  No counterpart in the reference, which keeps no cache; the attention over it is paged_decode.hip, the
// layout of a block paged.h.
//
// A block of 32 tokens of one head holds codes c and a scale 2^e:  x = c * 2^e, c of e4m3, e the least integer with
// max|x| <= 448 * 2^e over the finite values.  Tokens that come to a block that holds some take
//     e' = max(e, e of the new ones),   c = round(x / 2^e'),   and the old ones   c' = round(c * 2^(e - e')),
// which changes nothing but codes that fall below 2^-6.  NaN and infinities are held as NaN.
// All of it moves memory: per element 2 bytes read and 1 written (append) or the reverse (gather).  A copy of 2 GiB runs at 4.86 TB/s
// of bytes read and written, 7 where little is read.
#include <algorithm>

#include "paged_codes.h"

namespace sa {

namespace {

// One wave stores the new tokens of one block of one head, K or V.  The rows come from memory as they lie there, 1 KiB a load, and
// cross the lanes through LDS, 16 at a time.
// Bound by memory: 32 prompts of 32768 tokens, 8 heads, D = 128 1.17 ms, 4.7 TB/s; by latency: one token of 64 sequences 5.8 us (length,
// table, scale, block).  Loads of a lane's own pieces instead of rows, without LDS: ragged prompts with their read-back 62 us, now 45.
template <int DT, int ND>
__global__ __launch_bounds__(64 * kCacheWaves, ND == 8 ? 2 : 4) void paged_append_kernel(const PagedAppendParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t smem[kCacheWaves * 16 * row_bytes<ND>];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned item = blockIdx.x * kCacheWaves + wave;
    const bool values = item & 1u;
    item >>= 1;
    const int h = (int)(item % (unsigned)p.c.H);
    item /= (unsigned)p.c.H;
    const int nb = (int)(item % (unsigned)p.blocks), b = (int)(item / (unsigned)p.blocks);
    if (b >= p.t.B) return;
    const int room = p.t.width << (p.c.lper + 5);  // tokens that the table has place for
    const int len = max(p.t.lens[b], 0);
    if (len >= room) return;
    const int n = p.counts != nullptr ? min(max(p.counts[b], 0), p.S) : p.S;
    const int blk = (len >> 5) + nb;
    // tokens [a, z) of the block are new, [0, held) are there
    const int first = 32 * blk;
    if (first >= room) return;
    const int held = max(len - first, 0), a = held, z = min(len + n - first, 32);
    if (a >= z) return;
    const int page = page_at(p.t, b, blk >> p.c.lper, p.c.pages);
    // row t of the block is token first + t of the sequence, first + t - len of the new ones
    const int64_t *const xs = values ? p.vs : p.ks;
    const int64_t row = xs[2];
    const uint16_t *const x = (values ? p.v : p.k) + b * xs[0] + h * xs[1] + (int64_t)(first - len) * row;
    append_block<DT, ND>(p.c, x, row, values, page, h, blk & ((1 << p.c.lper) - 1), held, a, z, smem + wave * 16 * row_bytes<ND>);
}

// One wave reads one block of one head, K or V, into rows; rows that hold nothing become zero.  The rows cross the lanes in LDS and leave
// 1 KiB a store, 16 rows at a time, so that all the waves that a compute unit holds have their place there.  FAR: the stores pass the
// caches by, for outputs larger than those.
// 192 MiB of zeros and tokens of 16 ragged sequences, D = 64 36 us, 7.3 TB/s; 768 MiB, D = 128 204 us, 5.3 TB/s.  One or two waves a
// workgroup are no faster, streaming loads slower (37 -> 51 us).
template <int DT, int ND, bool FAR>
__global__ __launch_bounds__(64 * kCacheWaves) void paged_gather_kernel(const PagedGatherParams p) {
    using X = Half16<DT>;
    constexpr int NG = ND / 2, PPR = 4 * ND, RPI = 64 / PPR, NL = 16 / RPI;
    __shared__ __attribute__((aligned(16))) uint8_t smem[kCacheWaves * 16 * row_bytes<ND>];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint8_t *const mine = smem + wave * 16 * row_bytes<ND>;
    const int l32 = lane & 31, hh = lane >> 5;
    const unsigned blocks = ((unsigned)p.length + 31) / 32;
    unsigned item = blockIdx.x * kCacheWaves + wave;
    const bool values = item & 1u;
    item >>= 1;
    const int blk = (int)(item % blocks);
    item /= blocks;
    const int h = (int)(item % (unsigned)p.c.H), b = (int)(item / (unsigned)p.c.H);
    if (b >= p.t.B) return;
    const int first = 32 * blk, rows = min(p.length - first, 32);
    const int page = page_at(p.t, b, blk >> p.c.lper, p.c.pages);
    const int n = page < 0 ? 0 : min(max(max(p.t.lens[b], 0) - first, 0), rows);  // rows that hold something
    const int64_t at = block_at(p.c, max(page, 0), h, blk & ((1 << p.c.lper) - 1));
    const uint8_t *const in = (values ? p.c.v : p.c.k) + at * (ND * 1024);
    u32x4 u[ND];
    float scale = 0.f;
    if (n > 0) {
#pragma unroll
        for (int c = 0; c < ND; c++)
            u[c] = *(const u32x4 *)(in + (values ? 1024 * (2 * (c >> 1) + (l32 >> 4)) + 16 * (32 * hh + 2 * (l32 & 15) + (c & 1)) : 1024 * c + 16 * lane));
        scale = exp2i(exp_of_scale((values ? p.c.v_scales : p.c.k_scales)[at]));
        if (DT == 1 && scale > kFp16Scale)
            scale = within_fp16(scale, [&](auto &&f) {
#pragma unroll
                for (int c = 0; c < ND; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) u[c][i] = f(u[c][i]);
            });
    }
    const int64_t *const xs = values ? p.vs : p.ks;
    uint16_t *const x = (values ? p.v : p.k) + b * xs[0] + h * xs[1] + (int64_t)first * xs[2];
    const int r0 = lane / PPR, piece = lane % PPR;
#pragma unroll
    for (int half = 0; half < 2; half++) {  // rows 16 half ..
        if (n > 16 * half) {
            if (!values) {
                if ((l32 >> 4) == half) {
#pragma unroll
                    for (int c = 0; c < ND; c++) {
                        u32x4 *const to = (u32x4 *)(mine + (l32 & 15) * row_bytes<ND> + 64 * c + 32 * hh);
                        to[0] = u32x4{X::cvt_lo(u[c].x, scale), X::cvt_hi(u[c].x, scale), X::cvt_lo(u[c].y, scale), X::cvt_hi(u[c].y, scale)};
                        to[1] = u32x4{X::cvt_lo(u[c].z, scale), X::cvt_hi(u[c].z, scale), X::cvt_lo(u[c].w, scale), X::cvt_hi(u[c].w, scale)};
                    }
                }
            } else {
#pragma unroll
                for (int g = 0; g < NG; g++)  // d = 64 g + 2 l32 and the next one
#pragma unroll
                    for (int i = half; i < 4; i += 2) {
                        uint32_t *const to = (uint32_t *)(mine + (8 * (i >> 1) + 4 * hh) * row_bytes<ND> + 128 * g + 4 * l32);
                        const uint32_t a0 = X::cvt_lo(u[2 * g][i], scale), a1 = X::cvt_hi(u[2 * g][i], scale);
                        const uint32_t b0 = X::cvt_lo(u[2 * g + 1][i], scale), b1 = X::cvt_hi(u[2 * g + 1][i], scale);
                        to[0] = (a0 & 0xffffu) | (b0 << 16);
                        to[row_bytes<ND> / 4] = (a0 >> 16) | (b0 & 0xffff0000u);
                        to[2 * row_bytes<ND> / 4] = (a1 & 0xffffu) | (b1 << 16);
                        to[3 * row_bytes<ND> / 4] = (a1 >> 16) | (b1 & 0xffff0000u);
                    }
            }
            in_order();
        }
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int r = RPI * i + r0, t = 16 * half + r;
            u32x4 y = u32x4{0u, 0u, 0u, 0u};
            if (t < n) y = *(const u32x4 *)(mine + r * row_bytes<ND> + 16 * piece);
            if (t < rows && 8 * piece < p.c.cols) {
                u32x4 *const to = (u32x4 *)(x + t * xs[2] + 8 * piece);
                if constexpr (FAR) __builtin_nontemporal_store(y, to);
                else *to = y;
            }
        }
        in_order();
    }
}

// The first `blocks` blocks of head h of page `src` to page `dst`, by a workgroup of 256.  Half of a pool of 3000 pages of 64 tokens, 8 heads,
// D = 128 in a compaction: 366 MB read and written in 68 us, 5.3 TB/s.
__device__ __forceinline__ void copy_head(const PagedPool &c, int src, int dst, int h, int blocks) {
    const int64_t from = block_at(c, src, h, 0), to = block_at(c, dst, h, 0);
    const int pieces = blocks * c.D * 2;  // of 16 bytes
    const u32x4 *const k0 = (const u32x4 *)(c.k + from * (32 * c.D)), *const v0 = (const u32x4 *)(c.v + from * (32 * c.D));
    u32x4 *const k1 = (u32x4 *)(c.k + to * (32 * c.D)), *const v1 = (u32x4 *)(c.v + to * (32 * c.D));
    for (int i = threadIdx.x; i < pieces; i += 256) {
        const u32x4 a = k0[i], b = v0[i];
        k1[i] = a;
        v1[i] = b;
    }
    if ((int)threadIdx.x < blocks) {
        c.k_scales[to + threadIdx.x] = c.k_scales[from + threadIdx.x];
        c.v_scales[to + threadIdx.x] = c.v_scales[from + threadIdx.x];
    }
}
// Whether one of n copies behind copy i, of those that take place, has the same destination (the last one's page stays).
template <class F>
__device__ __forceinline__ bool named_again(const int32_t *dst, int i, int n, F &&takes_place) {
    const int mine = dst[i];
    int found = 0;
    for (int j = i + 1 + (int)threadIdx.x; j < n; j += 256)
        if (dst[j] == mine) found |= takes_place(j) ? 1 : 0;
    return __syncthreads_or(found) != 0;
}

// A workgroup of copy and fork has a pair, and of its page as many heads as keep what it reads of the pairs behind its own, 2 n bytes in the
// mean, to a quarter of what it copies.  us, a head each | so: 32768 pages of 8 heads, 32 tokens, D = 64 1962 | 715, 2048 28 | 21.
int heads_each(int n, const PagedPool &c) {
    const int64_t head = (int64_t)(64 << c.lper) * c.D;  // bytes of K and V
    return (int)std::min<int64_t>((8 * (int64_t)n + head - 1) / head, c.H);
}

__global__ __launch_bounds__(256) void paged_copy_kernel(const PagedCopyParams p) {
    const unsigned shares = ((unsigned)p.c.H + p.heads - 1) / p.heads;
    const int i = (int)(blockIdx.x / shares), h0 = (int)(blockIdx.x - (unsigned)i * shares) * p.heads;
    const int dst = p.dst[i];
    if (dst < 0 || dst >= p.c.pages) return;
    auto takes_place = [&](int j) { return p.src[j] >= 0 && p.src[j] < p.c.pages && p.src[j] != dst; };
    if (!takes_place(i) || named_again(p.dst, i, p.n, takes_place)) return;
    for (int h = h0; h < min(h0 + p.heads, p.c.H); h++) copy_head(p.c, p.src[i], dst, h, 1 << p.c.lper);
}

__global__ __launch_bounds__(256) void paged_fork_kernel(const PagedForkParams p) {
    const unsigned shares = ((unsigned)p.c.H + p.heads - 1) / p.heads;
    const int i = (int)(blockIdx.x / shares), h0 = (int)(blockIdx.x - (unsigned)i * shares) * p.heads;
    const int lP = p.c.lper + 5, fresh = p.new_pages[i];
    struct Child {
        int b, len, full, tail, src;  // src: the page that is copied, or -1
    };
    auto child = [&](int j) {
        Child x{p.parents[j], 0, 0, 0, -1};
        if (x.b >= 0 && x.b < p.t.B) x.len = min(max(p.t.lens[x.b], 0), p.t.width << lP);
        x.full = x.len >> lP;
        x.tail = x.len & ((1 << lP) - 1);
        if (x.tail != 0 && fresh >= 0 && fresh < p.c.pages) x.src = page_at(p.t, x.b, x.full, p.c.pages);
        if (x.src == fresh) x.src = -1;
        return x;
    };
    const Child x = child(i);
    if (h0 == 0) {
        const int used = x.full + (x.tail != 0 ? 1 : 0);
        for (int j = threadIdx.x; j < p.t.width; j += 256)
            p.new_ids[(int64_t)i * p.t.width + j] = j >= used ? -1 : x.src >= 0 && j == x.full ? fresh : p.t.ids[x.b * p.t.s0 + j * p.t.s1];
        if (threadIdx.x == 0) p.new_lens[i] = x.len;
    }
    if (x.src < 0 || named_again(p.new_pages, i, p.n, [&](int j) { return child(j).src >= 0; })) return;
    for (int h = h0; h < min(h0 + p.heads, p.c.H); h++) copy_head(p.c, x.src, fresh, h, (x.tail + 31) >> 5);
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanPages = 8192;  // whose lists a workgroup writes (16384: 29 -> 30 us, 11 -> 13 at 32768 used of 40000)
// Sum over the lanes up to this one, and over the threads in front of this one (and of all).
__device__ __forceinline__ int lanes_up_to(int x) {
#define SA_SUM_STEP(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false)
    SA_SUM_STEP(0x111, 0xf);
    SA_SUM_STEP(0x112, 0xf);
    SA_SUM_STEP(0x114, 0xf);
    SA_SUM_STEP(0x118, 0xf);
    SA_SUM_STEP(0x142, 0xa);
    SA_SUM_STEP(0x143, 0xc);
#undef SA_SUM_STEP
    return x;
}
__device__ __forceinline__ int before_me(int x, int *waves, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sum = lanes_up_to(x);
    __syncthreads();
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
    const int up = lanes_up_to(lane < kPlanThreads / 64 ? waves[lane] : 0);
    total = __builtin_amdgcn_readlane(up, 63);
    return sum - x + (wave == 0 ? 0 : __shfl(up, wave - 1));
}

// A bit per page that a sequence uses, then the pairs of a compaction or the free list.  Every workgroup reads the whole table and has all bits in
// LDS (2^20 pages: 128 KiB), in one launch: what the small tables of most programs cost is that.  Each writes the lists of its own part of the pages, 64 pages
// a step of a wave.  Free list, us, by one workgroup whose threads write the pages of their own words | so: 64 sequences in 2048 columns, 70000
// pages 61 | 29; in 8192 columns, 2^20 pages 709 | 117; 24 in 128 columns, 6147 pages 5.8 | 6.3.  Most of it is a table entry's VALU work, 20 instructions.
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(const PagedPlanParams p) {
    extern __shared__ __attribute__((aligned(8))) uint32_t bits[];
    __shared__ int waves[kPlanThreads / 64], before[kPlanThreads];  // before: pages in use in front of a thread's words
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pairs = (p.pages + 63) >> 6, words = 2 * pairs;
    for (int i = tid; i < words; i += kPlanThreads) bits[i] = 0u;
    __syncthreads();
    // a thread's entries, kPlanThreads apart: slot `at` of sequence b, `off` in the table
    constexpr int kEntries = 8;  // and their lengths, on their way at a time
    const int width = p.t.width, step_b = kPlanThreads / width, step_at = kPlanThreads - step_b * width;
    const int64_t step = step_b * p.t.s0 + step_at * p.t.s1, wrap = p.t.s0 - width * p.t.s1;
    unsigned b = (unsigned)(tid / width);
    int at = tid - (int)b * width;
    int64_t off = b * p.t.s0 + at * p.t.s1;
    while (b < (unsigned)p.t.B) {
        int page[kEntries], len[kEntries], first[kEntries];
#pragma unroll
        for (int k = 0; k < kEntries; k++) {
            page[k] = -1;
            len[k] = 0;
            if (b < (unsigned)p.t.B) {
                len[k] = p.t.lens[b];
                page[k] = p.t.ids[off];
            }
            first[k] = at << p.lP;  // (a table has at most 2^30 tokens a sequence)
            b += step_b;
            at += step_at;
            off += step;
            if (at >= width) {
                at -= width;
                b++;
                off += wrap;
            }
        }
#pragma unroll
        for (int k = 0; k < kEntries; k++)
            if (first[k] < len[k] && (unsigned)page[k] < (unsigned)p.pages) atomicOr(&bits[page[k] >> 5], 1u << (page[k] & 31));
    }
    __syncthreads();
    const int per = (words + kPlanThreads - 1) / kPlanThreads, w0 = min(tid * per, words), w1 = min(w0 + per, words);  // (per: at most 32)
    int used = 0, total;
    for (int w = w0; w < w1; w++) used += __popc(bits[w]);
    before[tid] = before_me(used, waves, total);
    __syncthreads();
    // pages in use below page x, by a whole wave
    auto used_below = [&](int x) {
        if (x >= p.pages) return total;
        const int w = x >> 5, t = w / per, in = w - t * per;  // (word `in` of thread t's)
        const uint32_t mine = lane <= in ? bits[t * per + lane] : 0u;
        return before[t] + __builtin_amdgcn_readlane(lanes_up_to(__popc(lane < in ? mine : mine & ((1u << (x & 31)) - 1u))), 63);
    };
    // this wave's pairs of words
    const int all_waves = (int)gridDim.x * (kPlanThreads / 64), per_wave = (pairs + all_waves - 1) / all_waves;
    const int q0 = min(((int)blockIdx.x * (kPlanThreads / 64) + wave) * per_wave, pairs), q1 = min(q0 + per_wave, pairs);
    auto in_use = [&](int q) { return *(const uint64_t *)(bits + 2 * q); };
    auto below = [&](int q, int x) { return x >= 64 * q + 64 ? ~0ull : x <= 64 * q ? 0ull : (1ull << (x - 64 * q)) - 1ull; };
    // put(place, page) for the pages that of(pair) gives, their places from `place` on
    auto each = [&](auto &&of, int place, auto &&put) {
        for (int q = q0; q < q1; q += 64) {
            const uint64_t m = q + lane < q1 ? of(q + lane) : 0ull;
            const int n = __popcll(m), up = lanes_up_to(n);
            for (int j = 0; j < min(64, q1 - q); j++) {
                const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)m, j), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(m >> 32), j);
                const int first = place + __builtin_amdgcn_readlane(up - n, j);
                if (((lane < 32 ? lo : hi) >> (lane & 31)) & 1u) put(first + (int)__builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0u)), 64 * (q + j) + lane);
            }
            place += __builtin_amdgcn_readlane(up, 63);
        }
    };
    const int start = min(64 * q0, p.pages), used_before = used_below(start);
    const bool first_thread = blockIdx.x == 0 && tid == 0;
    if (p.free_list != nullptr) {
        const int free_total = p.pages - total;
        each([&](int q) { return ~in_use(q) & below(q, p.pages); }, start - used_before, [&](int i, int page) { p.free_list[i] = page; });
        for (int i = free_total + (int)blockIdx.x * kPlanThreads + tid; i < p.pages; i += (int)gridDim.x * kPlanThreads) p.free_list[i] = -1;
        if (first_thread) *p.count = free_total;
        return;
    }
    const int L = total, stay = used_below(L);  // pages in use below L: those that are where they are to be
    each([&](int q) { return ~in_use(q) & below(q, L); }, min(start, L) - min(used_before, stay), [&](int i, int page) { p.holes[i] = page; });
    each([&](int q) { return in_use(q) & ~below(q, L); }, max(used_before - stay, 0), [&](int i, int page) {
        p.movers[i] = page;
        p.rank[page] = i;
    });
    if (first_thread) {
        *p.count = L;
        *p.moves = L - stay;
    }
}

// Moves the pages of the plan and writes the table that goes with them.
__global__ __launch_bounds__(256) void paged_compact_kernel(const PagedCompactParams p) {
    const int64_t entries = (int64_t)p.t.B * p.t.width;
    const int L = *p.count, lP = p.c.lper + 5;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)gridDim.x * 256) {
        const int b = (int)(i / p.t.width), j = (int)(i - (int64_t)b * p.t.width);
        int page = -1;
        if (((int64_t)j << lP) < p.t.lens[b]) page = page_at(p.t, b, j, p.c.pages);
        p.new_ids[i] = page >= L ? p.holes[p.rank[page]] : page;
    }
    const int64_t items = (int64_t)*p.moves * p.c.H;
    for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
        const int m = (int)(i / p.c.H);
        copy_head(p.c, p.movers[m], p.holes[m], (int)(i - (int64_t)m * p.c.H), 1 << p.c.lper);
    }
}

template <class F>
hipError_t with_sizes(int dtype, int D, F &&f) {
    auto by_dim = [&](auto dt) {
        if (D == 64) return f(dt, std::integral_constant<int, 2>{});
        if (D == 128) return f(dt, std::integral_constant<int, 4>{});
        if (D == 256) return f(dt, std::integral_constant<int, 8>{});
        return hipErrorInvalidValue;
    };
    if (dtype == 0) return by_dim(std::integral_constant<int, 0>{});
    if (dtype == 1) return by_dim(std::integral_constant<int, 1>{});
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendParams &p, int dtype, hipStream_t stream) {
    return with_sizes(dtype, p.c.D, [&](auto dt, auto nd) {
        hipLaunchKernelGGL((paged_append_kernel<decltype(dt)::value, decltype(nd)::value>), dim3((2u * p.c.H * p.blocks * p.t.B + kCacheWaves - 1) / kCacheWaves), dim3(64 * kCacheWaves), 0, stream, p);
        return hipGetLastError();
    });
}
// Outputs of that many bytes go past the caches (L2 and the memory-side cache hold 288 MiB, what reads the output brings its own).
// us, through them | past them: 64 MiB 24.4 | 27.1 (with the fork in front), 192 MiB 58.4 | 55.3, 768 MiB (with the compaction) 296 | 278.
constexpr int64_t kGatherFar = 128ll << 20;

hipError_t launch_paged_gather(const PagedGatherParams &p, int dtype, hipStream_t stream) {
    const unsigned blocks = ((unsigned)p.length + 31) / 32;
    const bool far = (int64_t)p.t.B * p.c.H * p.length * p.c.cols * 4 >= kGatherFar;
    return with_sizes(dtype, p.c.D, [&](auto dt, auto nd) {
        constexpr int DT = decltype(dt)::value, ND = decltype(nd)::value;
        hipLaunchKernelGGL((far ? paged_gather_kernel<DT, ND, true> : paged_gather_kernel<DT, ND, false>), dim3((2u * p.c.H * blocks * p.t.B + kCacheWaves - 1) / kCacheWaves), dim3(64 * kCacheWaves), 0, stream, p);
        return hipGetLastError();
    });
}
hipError_t launch_paged_copy(PagedCopyParams p, hipStream_t stream) {
    p.heads = heads_each(p.n, p.c);
    hipLaunchKernelGGL(paged_copy_kernel, dim3((unsigned)p.n * ((p.c.H + p.heads - 1) / p.heads)), dim3(256), 0, stream, p);
    return hipGetLastError();
}
hipError_t launch_paged_fork(PagedForkParams p, hipStream_t stream) {
    p.heads = heads_each(p.n, p.c);
    hipLaunchKernelGGL(paged_fork_kernel, dim3((unsigned)p.n * ((p.c.H + p.heads - 1) / p.heads)), dim3(256), 0, stream, p);
    return hipGetLastError();
}
hipError_t launch_paged_plan(const PagedPlanParams &p, hipStream_t stream) {
    const int smem = ((p.pages + 63) / 64) * 8;
    static unsigned long long attr_done = 0;
    if (const hipError_t e = allow_dynamic_smem(paged_plan_kernel, kPagedMostPages / 8, attr_done); e != hipSuccess) return e;
    const int groups = (p.pages + kPlanPages - 1) / kPlanPages;
    hipLaunchKernelGGL(paged_plan_kernel, dim3(groups), dim3(kPlanThreads), smem, stream, p);
    return hipGetLastError();
}
hipError_t launch_paged_compact(const PagedCompactParams &p, hipStream_t stream) {
    hipLaunchKernelGGL(paged_compact_kernel, dim3(2048), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace sa
