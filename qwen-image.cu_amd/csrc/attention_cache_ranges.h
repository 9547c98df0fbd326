// attention_cache_ranges.h — into what lengths attention_cache.hip cuts the keys of its
// row tiles. The tile kernels and the join kernel each work a length out from the same
// sums, and the join reads the parts that this length says were written, so every kernel
// has to come to the same number: fp32 products and sums in a fixed order, none contracted
// into a fused one, as the compiler may do in one kernel and not in another.
#pragma once

#include <cmath>

namespace qimg {

namespace {

// Workgroups of tiles of 16 (NR = 1), 32 (2) and MR rows that run at once, by registers (512
// of 16 rows: one token of 64 long int8 caches 180 to 175 us, but 64 tokens of 24/24 heads
// behind 4096 int8 keys 44 to 50)
__host__ __device__ constexpr int few_grid(int rows) { return rows == 16 ? 768 : 512; }
constexpr int kManyGrid = 512;

// Sums over the sequences of a launch, in steps: with causal halves, with all that a mask
// hides, the row tiles; a step's least length for the ranges that there is room for, and
// the longest tile's steps.
struct RangeSums {
    float work, all, tiles;
    int least, longest;
};

// steps of `tiles` row tiles of n steps, the first of which has `fewer` steps less than the last
__host__ __device__ inline float seen_steps(float tiles, int n, int fewer) {
#pragma clang fp contract(off)
    return tiles * (static_cast<float>(n) - 0.5f * static_cast<float>(fewer));
}
// the sums of one head, for `heads`
__host__ __device__ inline void times_heads(RangeSums& s, int heads) {
#pragma clang fp contract(off)
    const float h = static_cast<float>(heads);
    s.work *= h;
    s.all *= h;
    s.tiles *= h;
}

// Shares of `share` steps against `whole` of the tiles themselves: in steps, what a workgroup
// has to do, starts and joins (6) and the float results (6 for each workgroup, and tile).
__host__ __device__ inline bool shares_pay(float share, float tiles, float whole) {
#pragma clang fp contract(off)
    return 1.05f * share + 6.0f + (kManyGrid + tiles) * (6.0f / kManyGrid) < whole;
}

// Steps of a share of tiles of MR rows, for the workgroups that run at once, where these take
// less time than whole tiles; 0: tiles are whole.
__host__ __device__ inline int share_length(const RangeSums& s, bool causal) {
#pragma clang fp contract(off)
    if (s.all >= 0x1p30f) return 0;
    const float each = s.work / kManyGrid, longest = static_cast<float>(s.longest), share = s.all / kManyGrid;
    // whole tiles: rounds of the longest, or what evens out while the last ones run
    const float rounds = ceilf(s.tiles / kManyGrid) * longest, mixed = each + (causal ? 0.25f : 1.0f) * longest;
    const float whole = fmaxf(fminf(rounds, mixed), fmaxf(each, longest));
    if (!shares_pay(share, s.tiles, whole)) return 0;
    const int steps = static_cast<int>(share) + 1, most = steps > 4 ? steps : 4;
    return most > s.least ? most : s.least;
}

// Steps of a range of tiles of few rows, about: as many as make the launch one item a
// workgroup, at least two a wave.
__host__ __device__ inline int few_length(const RangeSums& s, int rows) {
#pragma clang fp contract(off)
    // (offsets that overlap may sum to any number)
    const int per = static_cast<int>(fminf(s.work / fmaxf(static_cast<float>(few_grid(rows)), 1.25f * s.tiles), 0x1p25f)) + 1;
    const int most = per > 2 * 4 ? per : 2 * 4;
    return most > s.least ? most : s.least;
}

}  // namespace

}  // namespace qimg
