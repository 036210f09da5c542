// How the one-token attention over a paged cache is cut into work (paged.hip; plain C++ as well, for the CPU test).
//
// A row's seen positions, from the 16-aligned one at or before the first, are units of 128. The units of all rows and of all `pairs` (kv head, block of
// 16 query heads) of a row form one line: rows in order, within a row pair after pair, within a pair unit after unit. Each worker (a workgroup) takes a
// stretch of the line, all stretches of the same length but for one unit, so rows of any lengths load the card evenly. A stretch is cut into segments
// where a pair ends; a segment that is all of its pair writes the result, any other one leaves a partial sum: a worker has at most two, its
// first and its last segment. The partial sums of a pair are joined in the workers' order, which depends on the lengths alone.
#pragma once
#ifdef __HIPCC__
#define MERV_HD __host__ __device__ inline
#else
#define MERV_HD inline
#endif

namespace merv {

constexpr int PAGED_UNIT = 128;        // positions: one tile of 32 for each of a workgroup's four waves
constexpr int PAGED_HEAD_BLOCK = 16;   // query heads of one workgroup: the columns of its matrix instructions
constexpr int PAGED_MAX_WORKERS = 512; // two workgroups on each of 256 CUs

struct PagedSpan {
    long base, lo, len;  // units count from `base`; positions lo <= j < len are seen
    int units;
};
// a length that is not positive, or over the capacity, has no units (the join writes such rows)
MERV_HD PagedSpan paged_span(long len, long window, long capacity) {
    PagedSpan s{0, 0, len, 0};
    if (len <= 0 || len > capacity) return s;
    s.lo = window > 0 && len > window ? len - window : 0;
    s.base = s.lo & ~15L;
    s.units = (int)((len - s.base + PAGED_UNIT - 1) / PAGED_UNIT);
    return s;
}

// `total` units on the line, `workers` workers at most: each has one unit or more
MERV_HD int paged_workers(long total, int workers) { return total < workers ? (int)total : workers; }
MERV_HD long paged_start(int w, long total, int workers) { return total * w / workers; }
MERV_HD int paged_owner(long unit, long total, int workers) { return (int)(((unit + 1) * workers - 1) / total); }
// the partial sum that worker w leaves of the pair whose units begin at `first`: slot 2w if the pair is in its first segment, 2w + 1 if in its last
MERV_HD int paged_slot(int w, long first, long total, int workers) { return 2 * w + (paged_start(w, total, workers) < first ? 1 : 0); }

}  // namespace merv
