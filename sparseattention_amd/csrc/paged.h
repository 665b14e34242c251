// The 8-bit paged K/V cache: its layout and the parameters of its kernels (paged_cache.hip, paged_decode.hip).
//
// A page holds page_size tokens of every head, as blocks of 32 consecutive tokens of one head; a block is 32 * D bytes,
// e4m3 codes, and has one scale 2^e.  The power of two costs no accuracy, as the codes are floating-point numbers, and makes
// scaling exact: what a block holds does not change when its scale grows, but for codes that become subnormal.
// Inside a block the codes lie in the order in which the attention's matrix instructions take them, so that a wave reads a
// block with D / 32 loads of 1 KiB each, straight into their operands:
//   K  16 bytes of lane (key = lane % 32, hh = lane / 32) of piece c: d = 32 c + 16 hh ..+15 of that key
//   V  16 bytes of lane (d % 32 = lane % 32, hh) of piece d / 32: keys 16 (j / 4 % 2) + 8 (j / 8) + 4 hh + j % 4, j = 0..15
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sa {

constexpr int kScaleExpMin = -96, kScaleExpMax = 119;  // 448 * 2^120 would be beyond bf16 and float32
constexpr int kPagedMostPages = 1 << 20;               // (compaction keeps a bit per page in LDS)

// In fp16 a code times 2^e, e > 7, may be beyond the type: fp16 tokens up to 65504 make blocks of the scale 2^8, where 65504 itself is held as 65536,
// bf16 tokens blocks of any scale, and codes that no token has, or that a row leaves out, stand for up to 114688 and more; times a weight of 0 these must
// be 0.  What lies beyond 65504 counts as 61440, the largest value within the type that four bits hold; NaN stays NaN.
// within_fp16 gives the scale that the block has from there on; each(f) is to replace every register w of four codes by f(w).
// Up to e = 21 61440 is a code of the block's own, at which larger ones stop.  From 22 on it is none, and codes from 8 on are beyond: the
// block is taken to 2^8, where 61440 is code 0x77 and the multiples of 2^13 below 2^16 that codes 1 .. 7 may be have codes too.
constexpr float kFp16Scale = 128.f;  // (448 * 2^7 is within)
template <class Each>
__device__ __forceinline__ float within_fp16(float scale, Each &&each) {
    const int e = (int)(__float_as_uint(scale) >> 23) - 127;
    if (e <= 21) {
        const uint32_t most = (uint32_t)(0x77 - 8 * (e - 8)) * 0x01010101u;
        each([=](uint32_t w) {
            const uint32_t size = w & 0x7f7f7f7fu, nan = (size + 0x01010101u) & 0x80808080u;
            const uint32_t over = (((size + (0x7f7f7f7fu - most)) & 0x80808080u & ~nan) >> 7) * 0x7fu;
            return (w & ~over) | (most & over);
        });
        return scale;
    }
    // what codes 0 .. 3 and 4 .. 7 become: n * 2^(e - 9) over 2^8
    const uint32_t low = e == 22 ? 0x6c686000u : e == 23 ? 0x74706800u : e == 24 ? 0x77777000u : 0x77777700u, high = e == 22 ? 0x76747270u : 0x77777777u;
    each([=](uint32_t w) {
        const uint32_t size = w & 0x7f7f7f7fu, nan = ((size + 0x01010101u) & 0x80808080u) >> 7, over = ((size + 0x78787878u) & 0x80808080u) >> 7;
        const uint32_t within = __builtin_amdgcn_perm(high, low, size & 0x07070707u) & ~(over * 0x7fu);
        return (w & 0x80808080u) | within | over * 0x77u | nan * 0x7fu;
    });
    return 256.f;
}

struct PagedPool {
    uint8_t *k, *v;            // [pages, H, per, 32 * D]
    float *k_scales, *v_scales;  // [pages, H, per]
    int pages, H, lper, D;     // per = page_size / 32 = 2^lper
    int cols;                  // of the caller's tensors: a multiple of 8, at most D; the pool's others are zero
};
struct PageTable {
    const int32_t *ids;
    int64_t s0, s1;  // strides in elements
    const int32_t *lens;
    int B, width;
};

struct PagedAppendParams {
    PagedPool c;
    PageTable t;
    const uint16_t *k, *v;
    int64_t ks[3], vs[3];   // b, h, token strides in elements (d stride 1)
    const int32_t *counts;  // or null: S of every sequence
    int S, blocks;          // blocks: the most that S tokens touch
};
hipError_t launch_paged_append(const PagedAppendParams &p, int dtype, hipStream_t stream);

struct PagedGatherParams {
    PagedPool c;
    PageTable t;
    uint16_t *k, *v;
    int64_t ks[3], vs[3];
    int length;
};
hipError_t launch_paged_gather(const PagedGatherParams &p, int dtype, hipStream_t stream);

struct PagedCopyParams {
    PagedPool c;
    const int32_t *src, *dst;
    int n;
    int heads;  // of a workgroup (set by the launch)
};
hipError_t launch_paged_copy(PagedCopyParams p, hipStream_t stream);

struct PagedForkParams {
    PagedPool c;
    PageTable t;
    const int32_t *parents, *new_pages;
    int n;
    int32_t *new_ids, *new_lens;  // [n, width], [n]
    int heads;
};
hipError_t launch_paged_fork(PagedForkParams p, hipStream_t stream);

// Which pages are in use, by a bit per page in LDS, and what follows from it.
struct PagedPlanParams {
    PageTable t;
    int pages, lP;
    int32_t *count;  // pages in use (compaction) or free (free list)
    // compaction: the j-th lowest free page below `count` and the j-th lowest page in use from `count` on, how many such pairs
    // there are, and the j of a page in use from `count` on
    int32_t *holes, *movers, *moves, *rank;
    int32_t *free_list;  // or the free pages in rising order, -1 behind the last
};
hipError_t launch_paged_plan(const PagedPlanParams &p, hipStream_t stream);

struct PagedCompactParams {
    PagedPool c;
    PageTable t;
    const int32_t *count, *holes, *movers, *moves, *rank;
    int32_t *new_ids;  // [B, width]
};
hipError_t launch_paged_compact(const PagedCompactParams &p, hipStream_t stream);

// Where the units of a launch's row begin (paged_decode.hip), found by a launch in front.
struct PagedUnits {
    unsigned cuts, share, total, pad;
    unsigned first[1];  // [units]
};
struct PagedDecodeParams {
    PagedPool c;
    PageTable t;
    const uint16_t *q;
    uint16_t *o;
    float *lse;  // or null
    int64_t qs[3], os[3], lses[3];  // b, h, row strides in elements
    const int32_t *counts;  // valid query rows of each sequence, or null: Sq
    int G, Sq, R, RT;       // query heads of a K/V head; rows of one: R = G * Sq in RT tiles of 16 (all of them) or 32
    int window;             // or 0
    // tile lists, tile = page, all null: every key that causality and window leave
    const int32_t *full_ids, *full_lens, *part_ids, *part_lens;
    int64_t fis[3], fls[2], pis[3], pls[2];  // b, h (and entry) strides
    const uint8_t *packed;  // PARTIAL tiles, Sq rows of page_size bits (PackParams layout)
    int64_t pks[2];
    int nK;
    float scale;  // softmax scale / ln 2
    // The launch's workgroups, the most parts a plane has, and what planes that several workgroups share are added up by:
    // (paged_pieces.h)
    //   ws        [groups][2][part_rows][D + 4] floats: unnormalised rows, reference value and sum of each
    //   arrivals  [planes + groups] words (all_arrived), the number of the launch
    int groups, parts, part_rows;
    float *ws;
    uint64_t *arrivals;
    uint64_t tag;
    PagedUnits *units;  // or null: every workgroup finds them itself
};
// Bytes of ws.
size_t paged_decode_parts_bytes(int groups, int part_rows, int D);
hipError_t launch_paged_decode(const PagedDecodeParams &p, int dtype, hipStream_t stream);

}  // namespace sa
