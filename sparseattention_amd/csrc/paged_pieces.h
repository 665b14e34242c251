// Which chunks of a batch a workgroup of the paged attention takes (paged_decode.hip).  Plain C++, so that the map can be looked at on the host.
//
// The work is a row of chunks of 32 keys: units (a sequence, with lists a sequence and K/V head) one behind the other, of every unit its planes
// (head, tile of query rows), of every plane its T chunks, at least one, so that planes without keys are written too.
#pragma once

#include <math.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#define SA_PIECES_FN __host__ __device__ __forceinline__
#else
#define SA_PIECES_FN inline
#endif

namespace sa {

constexpr int kPagedWaves = 4;       // of a workgroup, which take chunks in turn
constexpr int kPagedMostParts = 128;  // of a plane (131072 keys of one K/V head, 8 rows: 32.7 us with 64, 30.3 with 128; of two heads 30.6, 27.9)
// Where pieces begin and end anywhere, what it costs a workgroup to come to a plane (queries, places and the first chunk to wait for, rows to
// hand over) stands in the row in front of the plane, as so many chunks: 64 ragged sequences of up to 8192 keys 103.7 us with none, 103.4 with
// 2, 102.9 with 4, 102.0 with 8, 103.6 with 16; 16 sequences at D = 256 75.8 -> 73.6 with 8.
constexpr unsigned kPagedComing = 8;

// Up to that many units (sequences, with lists their K/V heads) every wave finds its piece itself, of more a launch in front finds where they
// begin.  us, by every wave | by a launch: lists of 256 sequences x 8 heads 61 | 41, of 1024 x 8 191 | 89; 256 sequences without lists 31.6 | 34,
// 16384 164 | 122.
constexpr int kPagedFewUnits(bool lists) { return lists ? 64 : 256; }
// Workgroups that a compute unit holds (a wave of each per SIMD), by D / 32 and the rows of a tile.
constexpr int paged_occupancy(int nd, int rows, int tiles = 1) { return nd == 2 ? (rows == 16 || tiles > 1 ? 3 : 2) : nd == 4 ? (rows == 16 ? 3 : 2) : 1; }

// A launch: its workgroups (a multiple of 8), the most parts a plane is meant to have, rows of a part.
// As many workgroups as the device holds at once: with more, the pieces of a workgroup that starts late do not make up for its start
// (32 sequences of up to 32768 keys: 294 us; twice as many workgroups 304, four times 324).
// One workgroup adds a plane's parts up, 8 to 32 at a time.  So there are no more of them than let every compute unit read at full speed (a
// chunk of 8 KiB a wave, one workgroup each, or two of 4 KiB), but at least 16: 16 planes of 1000 chunks with 16 | 32 | 62 parts 32.3 |
// 37.9 | 41.6 us.
struct PagedDecodePlan {
    int groups, parts, part_rows;
};
// plane_rows: 16, or tiles of 32 that a workgroup has, kPagedWaves / tiles waves each (0: one tile).
inline PagedDecodePlan paged_decode_plan(int64_t planes, int R, int D, int64_t chunks, int cus, int plane_rows = 0) {
    PagedDecodePlan r;
    if (plane_rows == 0) plane_rows = R <= 16 ? 16 : 32;
    const int tiles = plane_rows < 64 ? 1 : plane_rows / 32, waves = kPagedWaves / tiles;
    const int64_t even = (int64_t)cus * (D == 64 ? 2 : 1) / planes;
    r.parts = (int)(even < 16 ? 16 : even < kPagedMostParts - 2 ? even : kPagedMostParts - 2);
    const int64_t resident = (int64_t)cus * paged_occupancy(D / 32, plane_rows == 16 ? 16 : 32, tiles);
    const int64_t fine = (chunks + waves - 1) / waves;  // parts of a plane of a chunk a wave
    const int64_t most = planes * ((fine < r.parts ? fine : r.parts) + 1);
    r.groups = ((int)(most < resident ? most : resident) + 7) / 8 * 8;
    r.part_rows = R < plane_rows ? R : plane_rows;
    return r;
}

// Either pieces of `share` chunks of the row, wherever they begin and end; or (cuts) every plane in even parts of up to `share` chunks, a workgroup
// each, so that none has two planes' latencies; the row is then one of parts.  The second where a plane is many parts, whose ends are
// then even, or where a part is short, so that latencies are all there is: at 8 parts a plane (64 planes of 129 chunks) 21.5 -> 18.3 us, 8
// planes of 63 chunks 12.1 -> 9.1, 104 planes of one chunk 14 -> 11; at 3 parts (256 planes of 700 ... 1024) it would be 290 -> 319.
// A plane has no more parts than `parts`, and no more than balance the chunks that a wave has one after the other (1.15 us each) with the
// sum over the parts: sqrt(2 T) of T chunks, but 16 at least.
// total: chunks of all planes (less than 2^31); longest: of a plane; waves: of a workgroup that take chunks in turn.  No division more than it takes: each costs as much as a step of the scan.
struct PagedShare {
    bool cuts;
    unsigned share;
};
SA_PIECES_FN PagedShare paged_share(unsigned total, unsigned planes, unsigned groups, unsigned longest, unsigned parts, unsigned waves = kPagedWaves) {
#ifdef __HIP_DEVICE_COMPILE__
    const unsigned balanced = (unsigned)__builtin_amdgcn_sqrtf(2.f * (float)longest);
#else
    const unsigned balanced = (unsigned)sqrtf(2.f * (float)longest);
#endif
    const unsigned most = balanced < 16u ? 16u : balanced;
    parts = parts < most ? parts : most;
    PagedShare r;
    r.cuts = planes < groups && (8 * planes <= groups || total <= 2 * waves * (groups - planes));
    const unsigned among = r.cuts ? groups - planes : groups;  // (a part of each plane may be short)
    if (!r.cuts) total += planes * kPagedComing;  // (the host: at most 2^24 planes)
    r.share = (total + among - 1) / among;
    if (r.cuts && r.share < waves) r.share = waves;
    if ((uint64_t)longest > (uint64_t)r.share * parts) r.share = (longest + parts - 1) / parts;
    return r;
}

// The last of U units that begins at a place of the row or in front of it, as a wave finds it, which looks at 64 at a time: count(u, step, left) is how
// many of the units u, u + step, ... (64 at most, below u + left) do, and the first of them does.
template <class Count>
SA_PIECES_FN int paged_find_unit(int U, Count &&count) {
    int u = 0;
    for (int left = U; left > 1;) {
        const int step = (left + 63) >> 6, skip = (count(u, step, left) - 1) * step;
        u += skip;
        left = step < left - skip ? step : left - skip;
    }
    return u;
}

// A plane of T chunks in the row.
SA_PIECES_FN unsigned paged_row_length(PagedShare s, unsigned T) { return s.cuts ? (T + s.share - 1) / s.share : T + kPagedComing; }
// What of a plane's place in the row, from at_row on, is not its chunks.
SA_PIECES_FN unsigned paged_coming(PagedShare s, unsigned at_row) { return s.cuts || at_row >= kPagedComing ? 0u : kPagedComing - at_row; }

// The piece of workgroup `block`, of `pieces` in all, or -1.  Consecutive workgroups go to the 8 XCDs in turn, consecutive pieces of the row
// to one, so that row tiles of a head read K and V from one L2: 224 rows over a window of 4955 111 -> 76 us, one row or few 0 ... 3 % less.
SA_PIECES_FN int paged_piece(unsigned block, unsigned pieces) {
    const unsigned per_xcd = (pieces + 7) >> 3, at = (block & 7) * per_xcd + (block >> 3);
    return (block >> 3) < per_xcd && at < pieces ? (int)at : -1;
}

// Of a plane that is row_T long in the row, from position at_row on, at most `left` of the row: chunks off .. off + n - 1.
struct PagedSegment {
    int off, n;
};
SA_PIECES_FN PagedSegment paged_segment(PagedShare s, unsigned T, unsigned row_T, unsigned at_row, unsigned left) {
    // (even parts: at most `share`, and no fewer than row_T of them hold the plane)
    const unsigned step = s.cuts ? (T + row_T - 1) / row_T : left, off = s.cuts ? at_row * step : at_row - kPagedComing;
    return {(int)off, (int)(T - off < step ? T - off : step)};
}

// The pieces that a plane at position plane_at of the row lies in: the first, and how many.
struct PagedRange {
    int first, parts;
};
SA_PIECES_FN PagedRange paged_range(PagedShare s, unsigned plane_at, unsigned row_T) {
    if (s.cuts) return {(int)plane_at, (int)row_T};
    const unsigned first = (plane_at + kPagedComing) / s.share;
    return {(int)first, (int)((plane_at + row_T - 1) / s.share - first + 1)};
}

}  // namespace sa
