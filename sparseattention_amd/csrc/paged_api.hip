// C ABI of the 8-bit paged K/V cache: argument validation and dispatch.  The declarations and their contracts live in
// include/sparseattn.h.
#include <hip/hip_runtime.h>

#include "api_common.h"
#include "paged.h"
#include "paged_pieces.h"
#include "rotation_api.h"
#include "sparseattn.h"

namespace {

using sa::fail;

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int pool_of(const char *who, const sa_paged_cache *c, sa::PagedPool &out) {
    if (!c || !c->k || !c->v || !c->k_scales || !c->v_scales) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null cache", who);
    if (c->num_pages <= 0 || c->num_pages > sa::kPagedMostPages || c->H <= 0)
        return fail(SA_ERR_INVALID_ARGUMENT, "%s: num_pages must be 1 .. %d and H positive (got %d, %d)", who, sa::kPagedMostPages, c->num_pages, c->H);
    if (c->page_size != 32 && c->page_size != 64 && c->page_size != 128 && c->page_size != 256)
        return fail(SA_ERR_UNSUPPORTED, "%s: page_size must be 32, 64, 128 or 256 (got %d)", who, c->page_size);
    if (c->D != 64 && c->D != 128 && c->D != 256) return fail(SA_ERR_UNSUPPORTED, "%s: head dim %d not supported (64, 128 and 256 are)", who, c->D);
    if (c->head_dim <= 0 || c->head_dim > c->D || c->head_dim % 8)
        return fail(SA_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8 up to %d (got %d)", who, c->D, c->head_dim);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scales, 4) || !aligned(c->v_scales, 4))
        return fail(SA_ERR_UNSUPPORTED, "%s: the cache's codes must be 16-byte aligned", who);
    const int per = c->page_size / 32;
    if ((int64_t)c->num_pages * c->H * per > 0x7fffffff) return fail(SA_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 blocks in the cache", who);
    int lper = 0;
    while ((1 << lper) < per) lper++;
    out = {c->k, c->v, c->k_scales, c->v_scales, c->num_pages, c->H, lper, c->D, c->head_dim};
    return SA_OK;
}

int table_of(const char *who, const int32_t *ids, const int64_t strides[2], const int32_t *lens, int B, int width, int page_size, sa::PageTable &out) {
    if (!ids || !strides || !lens) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null page table or lengths", who);
    if (B <= 0 || width <= 0) return fail(SA_ERR_INVALID_ARGUMENT, "%s: B and the table's width must be positive (got %d, %d)", who, B, width);
    if ((int64_t)width * page_size > (1 << 30)) return fail(SA_ERR_UNSUPPORTED, "%s: a table of more than 2^30 tokens per sequence", who);
    out = {ids, strides[0], strides[1], lens, B, width};
    return SA_OK;
}

// Rows of 16-byte pieces: unit last stride, the others multiples of 8 elements.
int rows_of(const char *who, const char *name, const void *p, const int64_t s[4]) {
    if (!p || !s) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null %s", who, name);
    if (s[3] != 1 || s[0] % 8 || s[1] % 8 || s[2] % 8 || !aligned(p, 16))
        return fail(SA_ERR_UNSUPPORTED, "%s: %s needs a contiguous last dimension, strides of multiples of 8 elements and 16-byte alignment", who, name);
    return SA_OK;
}

int half_dtype(const char *who, int dtype) {
    if (dtype != SA_DTYPE_BF16 && dtype != SA_DTYPE_FP16) return fail(SA_ERR_UNSUPPORTED, "%s: dtype %d not supported (bf16 and fp16 are)", who, dtype);
    return SA_OK;
}

int launched(const char *who, hipError_t e) {
    return e == hipSuccess ? SA_OK : fail(SA_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
}
int grid_fits(const char *who, int64_t workgroups) {
    return workgroups <= 0x7fffffff ? SA_OK : fail(SA_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 workgroups", who);
}

constexpr int kMostRows = 1 << 20;
constexpr int kTreeNodes = 64;

// Compute units of the current device.
int compute_units() {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) {
        (void)hipGetLastError();
        return 256;
    }
    return n;
}

#define SA_TRY(x)                              \
    do {                                       \
        if (const int rc_ = (x)) return rc_;   \
    } while (0)

}  // namespace

extern "C" {

int sa_paged_cache_append(const sa_paged_cache *cache, const void *k, const int64_t k_strides[4], const void *v, const int64_t v_strides[4],
                          const int32_t *page_table, const int64_t page_table_strides[2], const int32_t *lens, const int32_t *counts, int B, int S,
                          int pages_per_sequence, int dtype, void *stream) {
    const char *who = "sa_paged_cache_append";
    sa::PagedAppendParams p{};
    SA_TRY(pool_of(who, cache, p.c));
    SA_TRY(table_of(who, page_table, page_table_strides, lens, B, pages_per_sequence, cache->page_size, p.t));
    SA_TRY(rows_of(who, "k", k, k_strides));
    SA_TRY(rows_of(who, "v", v, v_strides));
    SA_TRY(half_dtype(who, dtype));
    if (S <= 0 || S > (1 << 30)) return fail(SA_ERR_INVALID_ARGUMENT, "%s: S must be 1 .. 2^30 (got %d)", who, S);
    p.k = static_cast<const uint16_t *>(k);
    p.v = static_cast<const uint16_t *>(v);
    for (int i = 0; i < 3; i++) p.ks[i] = k_strides[i], p.vs[i] = v_strides[i];
    p.counts = counts;
    p.S = S;
    p.blocks = (S + 62) / 32;  // the first one may have room for one token only
    SA_TRY(grid_fits(who, (int64_t)2 * p.c.H * p.blocks * B));
    return launched(who, sa::launch_paged_append(p, dtype, static_cast<hipStream_t>(stream)));
}

int sa_paged_cache_append_rotated(const sa_paged_cache *cache, const void *q, const int64_t q_strides[4], void *q_out, const int64_t q_out_strides[4],
                                  const void *k, const int64_t k_strides[4], const void *v, const int64_t v_strides[4], const int32_t *page_table,
                                  const int64_t page_table_strides[2], const int32_t *lens, const int32_t *counts, const int32_t *parents,
                                  const int64_t parents_strides[2], const sa_rotation *rotation, int B, int Hq, int S, int pages_per_sequence, int dtype,
                                  void *stream) {
    const char *who = "sa_paged_cache_append_rotated";
    sa::PagedRotatedParams p{};
    SA_TRY(pool_of(who, cache, p.c));
    SA_TRY(table_of(who, page_table, page_table_strides, lens, B, pages_per_sequence, cache->page_size, p.t));
    SA_TRY(rows_of(who, "q", q, q_strides));
    SA_TRY(rows_of(who, "q_out", q_out, q_out_strides));
    SA_TRY(rows_of(who, "k", k, k_strides));
    SA_TRY(rows_of(who, "v", v, v_strides));
    SA_TRY(half_dtype(who, dtype));
    SA_TRY(sa::rotation_of(who, rotation, p.c.cols, dtype, true, p.r));
    if (S <= 0 || S > (1 << 30)) return fail(SA_ERR_INVALID_ARGUMENT, "%s: S must be 1 .. 2^30 (got %d)", who, S);
    if (Hq <= 0 || Hq > kMostRows) return fail(SA_ERR_INVALID_ARGUMENT, "%s: Hq must be 1 .. %d (got %d)", who, kMostRows, Hq);
    if (p.r.axes && !p.r.positions) return fail(SA_ERR_INVALID_ARGUMENT, "%s: axes need positions", who);
    if (parents) {
        if (!parents_strides) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null strides of the parents", who);
        if (p.r.positions) return fail(SA_ERR_INVALID_ARGUMENT, "%s: positions come from the parents or are given, not both", who);
        if (S > kTreeNodes) return fail(SA_ERR_UNSUPPORTED, "%s: trees of at most %d nodes (got %d)", who, kTreeNodes, S);
        p.parents = parents;
        for (int i = 0; i < 2; i++) p.parents_stride[i] = parents_strides[i];
    }
    p.q = static_cast<const uint16_t *>(q);
    p.k = static_cast<const uint16_t *>(k);
    p.v = static_cast<const uint16_t *>(v);
    p.qo = static_cast<uint16_t *>(q_out);
    for (int i = 0; i < 3; i++) p.qs[i] = q_strides[i], p.ks[i] = k_strides[i], p.vs[i] = v_strides[i], p.qos[i] = q_out_strides[i];
    p.counts = counts;
    p.Hq = Hq;
    p.S = S;
    p.blocks = (S + 62) / 32;
    const int64_t groups = sa::paged_rotated_plan(p);
    if (groups < 0 || groups > sa::kMostGroups256) return fail(SA_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens or 2^24 - 1 workgroups", who);
    return launched(who, sa::launch_paged_rotated(p, groups, dtype, static_cast<hipStream_t>(stream)));
}

int sa_paged_cache_gather(const sa_paged_cache *cache, void *k, const int64_t k_strides[4], void *v, const int64_t v_strides[4],
                          const int32_t *page_table, const int64_t page_table_strides[2], const int32_t *lens, int B, int length,
                          int pages_per_sequence, int dtype, void *stream) {
    const char *who = "sa_paged_cache_gather";
    sa::PagedGatherParams p{};
    SA_TRY(pool_of(who, cache, p.c));
    SA_TRY(table_of(who, page_table, page_table_strides, lens, B, pages_per_sequence, cache->page_size, p.t));
    SA_TRY(rows_of(who, "k", k, k_strides));
    SA_TRY(rows_of(who, "v", v, v_strides));
    SA_TRY(half_dtype(who, dtype));
    if (length <= 0 || length > (1 << 30)) return fail(SA_ERR_INVALID_ARGUMENT, "%s: length must be 1 .. 2^30 (got %d)", who, length);
    p.k = static_cast<uint16_t *>(k);
    p.v = static_cast<uint16_t *>(v);
    for (int i = 0; i < 3; i++) p.ks[i] = k_strides[i], p.vs[i] = v_strides[i];
    p.length = length;
    SA_TRY(grid_fits(who, (int64_t)2 * p.c.H * ((length + 31) / 32) * B));
    return launched(who, sa::launch_paged_gather(p, dtype, static_cast<hipStream_t>(stream)));
}

int sa_paged_cache_copy(const sa_paged_cache *cache, const int32_t *src, const int32_t *dst, int n, void *stream) {
    const char *who = "sa_paged_cache_copy";
    sa::PagedCopyParams p{};
    SA_TRY(pool_of(who, cache, p.c));
    if (!src || !dst || n <= 0) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null list or n not positive", who);
    p.src = src;
    p.dst = dst;
    p.n = n;
    SA_TRY(grid_fits(who, (int64_t)n * p.c.H));
    return launched(who, sa::launch_paged_copy(p, static_cast<hipStream_t>(stream)));
}

int sa_paged_cache_keep(const sa_paged_cache *cache, const int32_t *page_table, const int64_t page_table_strides[2], const int32_t *lens, const int32_t *path,
                        const int64_t path_strides[2], const int32_t *accepted, int B, int n, int pages_per_sequence, void *stream) {
    const char *who = "sa_paged_cache_keep";
    sa::PagedKeepParams p{};
    SA_TRY(pool_of(who, cache, p.c));
    SA_TRY(table_of(who, page_table, page_table_strides, lens, B, pages_per_sequence, cache->page_size, p.t));
    if (!path || !path_strides || !accepted) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null path", who);
    if (n <= 0 || n > kTreeNodes) return fail(SA_ERR_UNSUPPORTED, "%s: trees of 1 .. %d nodes (got %d)", who, kTreeNodes, n);
    p.path = path;
    for (int i = 0; i < 2; i++) p.path_s[i] = path_strides[i];
    p.accepted = accepted;
    p.n = n;
    if ((int64_t)2 * p.c.H * B > sa::kMostGroups256) return fail(SA_ERR_UNSUPPORTED, "%s: more than 2^23 sequences' heads", who);
    return launched(who, sa::launch_paged_keep(p, static_cast<hipStream_t>(stream)));
}

int sa_paged_cache_fork(const sa_paged_cache *cache, const int32_t *page_table, const int64_t page_table_strides[2], const int32_t *lens, int B,
                        int pages_per_sequence, const int32_t *parents, const int32_t *new_pages, int n, int32_t *new_table, int32_t *new_lens,
                        void *stream) {
    const char *who = "sa_paged_cache_fork";
    sa::PagedForkParams p{};
    SA_TRY(pool_of(who, cache, p.c));
    SA_TRY(table_of(who, page_table, page_table_strides, lens, B, pages_per_sequence, cache->page_size, p.t));
    if (!parents || !new_pages || !new_table || !new_lens || n <= 0) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null list or n not positive", who);
    p.parents = parents;
    p.new_pages = new_pages;
    p.n = n;
    p.new_ids = new_table;
    p.new_lens = new_lens;
    SA_TRY(grid_fits(who, (int64_t)n * p.c.H));
    return launched(who, sa::launch_paged_fork(p, static_cast<hipStream_t>(stream)));
}

size_t sa_paged_cache_compact_workspace_bytes(int num_pages) {
    if (num_pages <= 0 || num_pages > sa::kPagedMostPages) return 0;
    return (3 * (size_t)num_pages + 4) * sizeof(int32_t);
}

int sa_paged_cache_compact(const sa_paged_cache *cache, const int32_t *page_table, const int64_t page_table_strides[2], const int32_t *lens, int B,
                           int pages_per_sequence, int32_t *new_table, int32_t *used, void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "sa_paged_cache_compact";
    sa::PagedCompactParams p{};
    SA_TRY(pool_of(who, cache, p.c));
    SA_TRY(table_of(who, page_table, page_table_strides, lens, B, pages_per_sequence, cache->page_size, p.t));
    if (!new_table || !used) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null output", who);
    const size_t need = sa_paged_cache_compact_workspace_bytes(p.c.pages);
    if (!workspace || workspace_bytes < need || !aligned(workspace, 4))
        return fail(SA_ERR_WORKSPACE, "%s: workspace of %zu bytes required (got %zu)", who, need, workspace ? workspace_bytes : (size_t)0);
    int32_t *const ws = static_cast<int32_t *>(workspace);
    sa::PagedPlanParams plan{};
    plan.t = p.t;
    plan.pages = p.c.pages;
    plan.lP = p.c.lper + 5;
    plan.count = used;
    plan.moves = ws;
    plan.holes = ws + 4;
    plan.movers = plan.holes + p.c.pages;
    plan.rank = plan.movers + p.c.pages;
    SA_TRY(launched(who, sa::launch_paged_plan(plan, static_cast<hipStream_t>(stream))));
    p.count = used;
    p.moves = plan.moves;
    p.holes = plan.holes;
    p.movers = plan.movers;
    p.rank = plan.rank;
    p.new_ids = new_table;
    return launched(who, sa::launch_paged_compact(p, static_cast<hipStream_t>(stream)));
}

int sa_paged_cache_free_pages(const int32_t *page_table, const int64_t page_table_strides[2], const int32_t *lens, int B, int pages_per_sequence,
                              int num_pages, int page_size, int32_t *free_pages, int32_t *free_count, void *stream) {
    const char *who = "sa_paged_cache_free_pages";
    sa::PagedPlanParams p{};
    if (page_size != 32 && page_size != 64 && page_size != 128 && page_size != 256)
        return fail(SA_ERR_UNSUPPORTED, "%s: page_size must be 32, 64, 128 or 256 (got %d)", who, page_size);
    if (num_pages <= 0 || num_pages > sa::kPagedMostPages)
        return fail(SA_ERR_INVALID_ARGUMENT, "%s: num_pages must be 1 .. %d (got %d)", who, sa::kPagedMostPages, num_pages);
    SA_TRY(table_of(who, page_table, page_table_strides, lens, B, pages_per_sequence, page_size, p.t));
    if (!free_pages || !free_count) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null output", who);
    p.pages = num_pages;
    while ((1 << p.lP) < page_size) p.lP++;
    p.count = free_count;
    p.free_list = free_pages;
    return launched(who, sa::launch_paged_plan(p, static_cast<hipStream_t>(stream)));
}

static size_t units_bytes(int64_t units) { return (sizeof(sa::PagedUnits) + (size_t)units * 4 + 15) / 16 * 16; }

// Rows of a plane.  Trees have many: where there is little work planes are small, as one workgroup adds a plane's parts up, row by row; where there is much
// several tiles of rows read K and V together.  us with planes of 16 | 32 | 64 | 128 rows, D = 128, bf16, of R rows of H K/V heads, C chunks in all:
//   R  32, H   8: C  504  12.4 | 18.9; 8000  26.8 | 37.1;    H 512: C 32256  76 | 59
//   R 128, H   8: C  504  18.6 | 21.6 | 26.7 | 42.9;         H 64: C 4032  30 | 34 | 33 | 45
//          H 256: C 16128  116 | 67 | 63 | 71; 32000  240 | 127 | 99 | 114; 65536  488 | 249 | 204 | 199; 160000  1338 | 674 | 455 | 434
//          H  16: C 32768  271 | 97 | 108 | 160 (few planes, of many parts)
//   R  64, H 256: C 32000  140 | 64 | 66; 65536  290 | 133 | 126; 262144  1224 | 532 | 400
// At the other head dims the same numbers are used, not always to their best:
//   D  64, R  32, H   8: C  504  10 | 13;   R 128, H 64: C 4032  24 | 23 | 26 | 46;    H 256: C 16128   80 |  41 |  48 |  53; 32000  157 |  68 |  75 |  74; 64000   301 | 125 | 124 | 125
//   D 256, R  32, H   8: C  504  19 | 30;   R 128, H 64: C 4032  61 | 39 | 65 | 84;    H 256: C 16128  308 | 176 | 125 | 124; 32000  713 | 377 | 253 | 218; 64000  1382 | 707 | 462 | 413
// C goes by the tables' width: 64 heads, R 128, C 4032, D 128 take 31 us with tables of 63 chunks, 46 with such of 4096.
static int decode_plane_rows(bool tree, int64_t heads, int R, int64_t chunks) {
    if (R <= 16) return 16;
    if (!tree) return 32;
    const int64_t work = heads * chunks;  // (of the tables: the sequences may be shorter)
    if (work * ((R + 15) / 16) <= 24 << 10) return 16;
    if (R <= 32 || heads < 64 || work * ((R + 63) / 64) <= 40 << 10) return 32;
    return R <= 64 || work < 64 << 10 ? 64 : 128;
}

static size_t decode_workspace_bytes(int most_rows, int B, int Hq, int H, int Sq, int D, int pages_per_sequence, int page_size) {
    if (B <= 0 || H <= 0 || Hq <= 0 || Hq % H || Sq <= 0 || Sq > most_rows || (D != 64 && D != 128 && D != 256) || pages_per_sequence <= 0 || page_size < 32 ||
        (int64_t)Hq / H * Sq > kMostRows)
        return 0;
    const int R = Hq / H * Sq;
    const int64_t heads = (int64_t)B * H, chunks = (int64_t)pages_per_sequence * (page_size / 32);
    const int plane_rows = decode_plane_rows(most_rows == kTreeNodes, heads, R, chunks);
    const int64_t planes = heads * ((R + plane_rows - 1) / plane_rows);
    const sa::PagedDecodePlan plan = sa::paged_decode_plan(planes, R, D, chunks, compute_units(), plane_rows);
    return sa::paged_decode_parts_bytes(plan.groups, plan.part_rows, D) + (size_t)(planes + plan.groups) * 8 + units_bytes((int64_t)B * H);
}

size_t sa_decode_paged_workspace_bytes(int B, int Hq, int H, int Sq, int D, int pages_per_sequence, int page_size) {
    return decode_workspace_bytes(32, B, Hq, H, Sq, D, pages_per_sequence, page_size);
}
size_t sa_decode_tree_workspace_bytes(int B, int Hq, int H, int n, int D, int pages_per_sequence, int page_size) {
    return decode_workspace_bytes(kTreeNodes, B, Hq, H, n, D, pages_per_sequence, page_size);
}

// What the two attentions have in common: p has the cache, the table and who attends.
static int decode(const char *who, sa::PagedDecodeParams &p, int most_rows, const void *q, const int64_t q_strides[4], void *o, const int64_t o_strides[4],
                  const int32_t *counts, int B, int Hq, int Sq, int window, int dtype, float sm_scale_log2, void *workspace, size_t workspace_bytes, float *lse,
                  const int64_t lse_strides[3], void *stream) {
    SA_TRY(rows_of(who, "q", q, q_strides));
    SA_TRY(rows_of(who, "o", o, o_strides));
    SA_TRY(half_dtype(who, dtype));
    if (Sq <= 0 || Sq > most_rows) return fail(SA_ERR_UNSUPPORTED, "%s: 1 .. %d query rows (got %d)", who, most_rows, Sq);
    if (Hq <= 0 || Hq % p.c.H) return fail(SA_ERR_INVALID_ARGUMENT, "%s: Hq (%d) must be a multiple of the cache's H (%d)", who, Hq, p.c.H);
    if (!(sm_scale_log2 > 0.f) || sm_scale_log2 > 3e38f) return fail(SA_ERR_INVALID_ARGUMENT, "%s: softmax scale must be positive and finite", who);
    if (window < 0) return fail(SA_ERR_INVALID_ARGUMENT, "%s: window must not be negative (got %d)", who, window);
    if (lse && !lse_strides) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null lse strides", who);
    p.q = static_cast<const uint16_t *>(q);
    p.o = static_cast<uint16_t *>(o);
    p.lse = lse;
    for (int i = 0; i < 3; i++) {
        p.qs[i] = q_strides[i];
        p.os[i] = o_strides[i];
        p.lses[i] = lse ? lse_strides[i] : 0;
    }
    p.counts = counts;
    p.G = Hq / p.c.H;
    p.Sq = Sq;
    if ((int64_t)p.G * Sq > kMostRows) return fail(SA_ERR_UNSUPPORTED, "%s: more than %d rows per K/V head", who, kMostRows);
    p.R = p.G * Sq;
    const int64_t heads = (int64_t)B * p.c.H, chunks = (int64_t)p.t.width << p.c.lper;
    p.plane_rows = decode_plane_rows(p.parents != nullptr, heads, p.R, chunks);
    p.tiles = p.plane_rows < 64 ? 1 : p.plane_rows / 32;
    p.RT = (p.R + p.plane_rows - 1) / p.plane_rows;
    p.window = window < (1 << 30) ? window : 0;  // (no table is that long)
    p.scale = sm_scale_log2;
    const int64_t planes = heads * p.RT;
    if (planes > (1 << 24) || planes * chunks > (1 << 30))
        return fail(SA_ERR_UNSUPPORTED, "%s: %lld planes of %d rows and %lld chunks of 32 keys each; a launch has at most 2^24 planes and 2^30 chunks of all of them", who, (long long)planes,
                    p.plane_rows, (long long)chunks);
    const sa::PagedDecodePlan plan = sa::paged_decode_plan(planes, p.R, p.c.D, chunks, compute_units(), p.plane_rows);
    const size_t parts_bytes = sa::paged_decode_parts_bytes(plan.groups, plan.part_rows, p.c.D), units_at = parts_bytes + (size_t)(planes + plan.groups) * 8,
                 need = units_at + units_bytes((int64_t)B * p.c.H);
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
        return fail(SA_ERR_WORKSPACE, "%s: workspace of %zu bytes required, 16-byte aligned (got %zu)", who, need, workspace ? workspace_bytes : (size_t)0);
    p.groups = plan.groups;
    p.parts = plan.parts;
    p.part_rows = plan.part_rows;
    p.ws = static_cast<float *>(workspace);
    p.arrivals = reinterpret_cast<uint64_t *>(static_cast<uint8_t *>(workspace) + parts_bytes);
    p.tag = sa::next_launch_tag() | 1;
    if ((p.full_ids != nullptr ? (int64_t)B * p.c.H : B) > sa::kPagedFewUnits(p.full_ids != nullptr)) p.units = reinterpret_cast<sa::PagedUnits *>(static_cast<uint8_t *>(workspace) + units_at);
    return launched(who, sa::launch_paged_decode(p, dtype, static_cast<hipStream_t>(stream)));
}

int sa_sparse_attention_decode_paged(const void *q, const int64_t q_strides[4], const sa_paged_cache *cache, const int32_t *page_table,
                                     const int64_t page_table_strides[2], const int32_t *lens, const int32_t *counts, int pages_per_sequence, void *o,
                                     const int64_t o_strides[4], const int32_t *full_ids, const int64_t full_ids_strides[4], const int32_t *full_lens,
                                     const int64_t full_lens_strides[3], const int32_t *part_ids, const int64_t part_ids_strides[4],
                                     const int32_t *part_lens, const int64_t part_lens_strides[3], const uint8_t *packed,
                                     const int64_t packed_strides[2], int tiles, int B, int Hq, int Sq, int window, int dtype, float sm_scale_log2,
                                     void *workspace, size_t workspace_bytes, float *lse, const int64_t lse_strides[3], void *stream) {
    const char *who = "sa_sparse_attention_decode_paged";
    sa::PagedDecodeParams p{};
    SA_TRY(pool_of(who, cache, p.c));
    SA_TRY(table_of(who, page_table, page_table_strides, lens, B, pages_per_sequence, cache->page_size, p.t));
    if (full_ids || full_lens || part_ids || part_lens || packed) {
        if (!full_ids || !full_lens || !part_ids || !part_lens || !packed || !full_ids_strides || !full_lens_strides || !part_ids_strides ||
            !part_lens_strides || !packed_strides)
            return fail(SA_ERR_INVALID_ARGUMENT, "%s: the four lists and the packed tiles come together", who);
        if (window) return fail(SA_ERR_INVALID_ARGUMENT, "%s: a window goes with no lists", who);
        if (tiles <= 0 || tiles > pages_per_sequence)
            return fail(SA_ERR_INVALID_ARGUMENT, "%s: lists of %d tiles, the table has %d pages per sequence", who, tiles, pages_per_sequence);
        if (!aligned(packed, 4) || packed_strides[0] % 4 || packed_strides[1] % 4)
            return fail(SA_ERR_UNSUPPORTED, "%s: packed tiles need 4-byte alignment", who);
        p.full_ids = full_ids;
        p.full_lens = full_lens;
        p.part_ids = part_ids;
        p.part_lens = part_lens;
        p.packed = packed;
        for (int i = 0; i < 2; i++) {
            p.fis[i] = full_ids_strides[i];
            p.pis[i] = part_ids_strides[i];
            p.fls[i] = full_lens_strides[i];
            p.pls[i] = part_lens_strides[i];
            p.pks[i] = packed_strides[i];
        }
        p.fis[2] = full_ids_strides[3];
        p.pis[2] = part_ids_strides[3];
        p.nK = tiles;
    }
    return decode(who, p, 32, q, q_strides, o, o_strides, counts, B, Hq, Sq, window, dtype, sm_scale_log2, workspace, workspace_bytes, lse, lse_strides, stream);
}

int sa_sparse_attention_decode_tree(const void *q, const int64_t q_strides[4], const sa_paged_cache *cache, const int32_t *page_table,
                                    const int64_t page_table_strides[2], const int32_t *lens, const int32_t *parents, const int64_t parents_strides[2],
                                    const int32_t *counts, int pages_per_sequence, void *o, const int64_t o_strides[4], int B, int Hq, int n, int window,
                                    int dtype, float sm_scale_log2, void *workspace, size_t workspace_bytes, float *lse, const int64_t lse_strides[3],
                                    void *stream) {
    const char *who = "sa_sparse_attention_decode_tree";
    sa::PagedDecodeParams p{};
    SA_TRY(pool_of(who, cache, p.c));
    SA_TRY(table_of(who, page_table, page_table_strides, lens, B, pages_per_sequence, cache->page_size, p.t));
    if (!parents || !parents_strides) return fail(SA_ERR_INVALID_ARGUMENT, "%s: null parents", who);
    p.parents = parents;
    for (int i = 0; i < 2; i++) p.parents_stride[i] = parents_strides[i];
    return decode(who, p, kTreeNodes, q, q_strides, o, o_strides, counts, B, Hq, n, window, dtype, sm_scale_log2, workspace, workspace_bytes, lse, lse_strides, stream);
}

}  // extern "C"
