// How the one-token attention over a paged cache is cut into work (paged.hip; plain C++ as well, for the CPU test).
//
// A row's seen positions, from the 16-aligned one at or before the first, are units of 128. The units of all rows and of all `pairs` (kv head, block of
// 16 query heads) of a row form one line: rows in order, within a row pair after pair, within a pair unit after unit. Each worker (a workgroup) takes a
// stretch of the line, all stretches of the same length but for one unit, so rows of any lengths load the card evenly. A stretch is cut into segments
// where a pair ends; a segment that is all of its pair writes the result, any other one leaves a partial sum: a worker has at most two, its
// first and its last segment. The partial sums of a pair are joined in the workers' order, which depends on the lengths alone.
// All numbers fit 31 bits (the entry point refuses larger calls), so that the divisions are 32-bit ones.
#pragma once
#ifdef __HIPCC__
#define MERV_HD __host__ __device__ __forceinline__
#else
#define MERV_HD inline
#endif

namespace merv {

constexpr int PAGED_UNIT = 128;        // positions: one tile of 32 for each of a workgroup's four waves
constexpr int PAGED_HEAD_BLOCK = 16;   // query heads of one workgroup: the columns of its matrix instructions
constexpr int PAGED_MAX_WORKERS = 512; // two workgroups on each of 256 CUs

struct PagedSpan {
    int base, lo, len, units;  // units count from `base`; positions lo <= j < len are seen
};
// a length that is not positive, or over the capacity, has no units (such rows are written apart); window 0: none
MERV_HD PagedSpan paged_span(int len, int window, int capacity) {
    PagedSpan s{0, 0, len, 0};
    if (len <= 0 || len > capacity) return s;
    s.lo = window > 0 && len > window ? len - window : 0;
    s.base = s.lo & ~15;
    s.units = (len - s.base + PAGED_UNIT - 1) / PAGED_UNIT;
    return s;
}

// `total` units on the line for `most` workers: the first `more` have each + 1 of them, the others each, and where there are fewer units than workers
// the last have none
struct PagedShare {
    int workers, each, more;
};
MERV_HD PagedShare paged_share(int total, int most) {
    const int workers = total < most ? total : most;
    if (workers <= 0) return PagedShare{0, 0, 0};
    return PagedShare{workers, total / workers, total % workers};
}
MERV_HD int paged_start(const PagedShare& s, int w) { return w * s.each + (w < s.more ? w : s.more); }
MERV_HD int paged_owner(const PagedShare& s, int unit) {
    const int long_ones = s.more * (s.each + 1);
    return unit < long_ones ? unit / (s.each + 1) : s.more + (unit - long_ones) / s.each;
}
// Whether each pair of each row is left whole, a workgroup for each of the `all` pairs and nothing to join. A pair alone on its CU takes about a quarter of the
// time for a unit that the fully loaded card needs for one more unit for each of its workers, and splitting costs four to five such quarters (workers
// change rows, sums are joined): so no pair may be longer than that buys. Fewer than 512 pairs leave part of the card's bandwidth unused, which
// counts once there are more than three units for each worker. Measured, 8-bit, 128 dims: 64 x 8 pairs of up to 9 units 23.0 us whole, 27.2 split; 33 x 4 of up
// to 9: 16.0 and 20.9; 64 dims, 16 bits: 24 x 12 of 8 units: 20.9 and 19.1.
constexpr int PAGED_MOST_WHOLE = 4096;
MERV_HD bool paged_whole(int total, int most, int all, int grid) {
    if (all > grid || all < 128 || most > 24 || (most - 4) * 128 > total) return false;
    return all >= PAGED_MAX_WORKERS || total <= 3 * PAGED_MAX_WORKERS;
}
// A worker's partial sums: slot 2w is its first segment's, 2w + 1 its last one's where that is another. All workers of a pair but the one it begins in leave
// its sum in 2w.
MERV_HD int paged_slot(int w, bool first_segment) { return 2 * w + (first_segment ? 0 : 1); }

// What a call launches, from sizes alone (the rows' lengths are on the device). Where a row cannot be long, one workgroup for each pair takes it whole and
// there is no join: up to 9 units, or 16 where there are pairs enough (the longest possible row then costs 18 us). Of eight waves where every pair has
// a CU to itself and more than one round of four waves to do.
// Measured, 128 dims, this and the split one in us (16 bits; 8 bits where they differ by more):
//   9 units   1 x 8 pairs 10.5,  9.8; 1 x 32 11.6, 12.5 (11.1, 11.1); 8 x 8 11.8, 14.0; 33 x 4 12.8, 17.6
//   10 units  1 x 8 11.5,  9.8; 1 x 32 12.6, 13.1 (12.1, 11.1); 8 x 8 12.6, 13.2 (12.1, 11.5); a row of 1049 in a table of 1280, 1 x 32: 11.1, 12.0 (11.0, 11.1)
//   12 units  1 x 8 12.7,  9.9; 1 x 32 14.0, 13.4 (13.6, 11.2); 8 x 8 13.9, 14.7 (13.8, 12.1)
//   14 units  1 x 8 14.2, 10.5; 1 x 32 15.2, 14.3 (15.2, 12.1); 8 x 8 15.4, 16.0 (15.5, 13.3)
//   16 units  1 x 8 15.4, 10.5; 1 x 32 16.5, 14.6 (16.6, 12.7); 8 x 8 16.4, 16.8 (16.8, 13.7); 33 x 4 19.8, 24.0
// Between 9 and 16 units neither form is the better one for all pairs and both types; the most that the rule gives away there is 2.5 us (2 x 32 pairs, 16 bits,
// 10 units: 12.8, 15.3). Eight and four waves: 4 units, 1 x 8 pairs 7.6 and 7.2 us; 9 units 9.9 and 11.5; 64 x 8 pairs of 9 units 36.7 and 35.9.
inline bool paged_direct(long units, long pairs) { return units <= 9 || (units <= 16 && pairs >= 128); }
inline int paged_direct_waves(long units, long pairs) { return units > 4 && pairs <= 256 ? 8 : 4; }

struct PagedPlan {
    int head_blocks, workers, grid, waves;
    bool direct;
};
inline PagedPlan paged_plan(int rows, int H, int kv_heads, long capacity) {
    PagedPlan pl;
    pl.head_blocks = (H / kv_heads + PAGED_HEAD_BLOCK - 1) / PAGED_HEAD_BLOCK;
    const long units = (capacity + PAGED_UNIT - 1) / PAGED_UNIT;
    const long pairs = (long)rows * kv_heads * pl.head_blocks, most = units * pairs;
    pl.workers = (int)(most < PAGED_MAX_WORKERS ? most : PAGED_MAX_WORKERS);
    pl.direct = paged_direct(units, pairs);
    pl.waves = pl.direct ? paged_direct_waves(units, pairs) : 4;
    pl.grid = (int)(pl.direct || (pairs > pl.workers && pairs <= PAGED_MOST_WHOLE) ? pairs : pl.workers);
    return pl;
}

}  // namespace merv
