// attention_cache.hip — attention over the pages of a quantized cache:
//   s_ij = sm_scale * q_i . k_j             (j visible to i)
//   o_i  = sum_j e^(s_ij - m_i) v_j / sum_j e^(s_ij - m_i)
// for sequences whose queries lie packed one behind the other and whose keys lie in
// pages named by a table, grouped heads, q in bf16 or fp16, codes int8 or e4m3 with a
// power of two a row (cache_codes.h). Key j of a sequence with lq queries and lk keys
// is visible to query i when j < lk and, if causal, j <= i + lk - lq. In front of them
// all queries see the keys of one prefix, whose pages are read once for the whole
// batch: its row tiles run over the queries of all sequences. A query that sees no key
// gives zeros.
//
// Codes become q's type on their way into the matrix unit, exactly (a power of two
// times 8 bits), so the products are those of an unquantized cache that holds the
// same values: fp32 accumulation, base-2 online softmax with the running maximum and
// sum in fp32, P rounded to q's type, the row sum over the rounded values. With u half
// a step of the type (2^-8 in bf16, 2^-11 in fp16) that leaves an error of at most
// sum_j u p_j |v_j - o| beside the result's own rounding. The maximum moves only when a
// tile exceeds it by kSlack (log2 units). P carries a factor 2^kPBias: in fp16 weights
// keep their digits down to 2^-21 of the maximum; in bf16 sums of P V stay below 2^128
// for any V (weights below 2^-88 of the maximum vanish).
//
// Rows: a tile's rows are (token, head of the group) pairs of one sequence and one kv
// head, so the heads of a group share the codes they read.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_cache_ranges.h"
#include "attention_tiles.h"
#include "cache_codes.h"

namespace qimg {

namespace {

template <class T>
__device__ __forceinline__ typename T::frag as_frag(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(typename T::frag, (u32x4){a, b, c, d});
}

// max over the four lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float quarter_max(float v) {
    unsigned u = __float_as_uint(v);
    auto sw = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    u = __float_as_uint(v);
    sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}

// Loads of a lane's `off` bytes (and a uniform `at`) behind a uniform address, through a descriptor that ends
// `bytes` behind it: the address costs a lane one register (through pointers of 64 bits
// the kernels below spill).
struct Buffer {
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ Buffer(const uint8_t* p, int bytes)
        : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, kRsrcWord3)) {}
    template <typename V>
    __device__ __forceinline__ V load(uint32_t off, int at = 0) const {
        V v{};
#if defined(__HIP_DEVICE_COMPILE__)  // (the host pass rejects the builtins)
        if constexpr (sizeof(V) == 16) v = __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, off, at, 0));
        else if constexpr (sizeof(V) == 8) v = __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(r, off, at, 0));
        else if constexpr (sizeof(V) == 4) v = __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b32(r, off, at, 0));
        else v = __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b8(r, off, at, 0));
#endif
        return v;
    }
};

// One sequence's tile of rows and range of keys. Sequence `batch` is the prefix: its
// queries are those of all sequences.
struct RowTile {
    int b, q0, lq, lk;   // sequence, its first query, numbers of queries and keys
    int row0;            // first (token, head) row of the tile in the sequence
    int split, splits;   // key range of it, and into how many the sequence's keys are cut
    bool found;
};
struct Sequence {
    int q0, lq, lk;
};
// Offsets outside [0, total] or falling ones and lengths past the table are clamped, so
// no tile reaches past the tensors.
__device__ __forceinline__ Sequence load_sequence(const AttnCacheArgs& a, int b, int end) {
    Sequence s = {0, 0, 0};
    if (b < end) {
        const bool own = b < a.batch;
        const int from = own ? a.cu_q[b] : a.cu_q[0], to = own ? a.cu_q[b + 1] : a.cu_q[a.batch];
        const int len = own ? a.k_lens[b] : a.prefix_len[0];
        const int64_t most = static_cast<int64_t>(own ? a.max_blocks : a.prefix_blocks) << a.c.page_shift;
        s.q0 = min(max(from, 0), a.total_q);
        s.lq = min(max(to, s.q0), a.total_q) - s.q0;
        s.lk = static_cast<int>(len < 0 ? 0 : len < most ? len : most);
    }
    return s;
}
__device__ __forceinline__ int row_tiles(const AttnCacheArgs& a, int lq, int rows) {
    return static_cast<int>((static_cast<int64_t>(lq) * a.group + rows - 1) / rows);
}
// What a launch works on: the sequences [lo, hi) and `heads` kv heads from h0 on, in tiles
// of `rows` rows, whose keys are taken in steps of `SK` or, in tiles of MR rows, `MK` keys.
struct Part {
    int lo, hi, rows, h0, heads;
};
constexpr int SK = 32;
__device__ __forceinline__ int steps_of(const Part& part, int lk) {
    return part.rows == MR ? (lk + MK - 1) / MK : (lk + SK - 1) / SK;
}
__device__ __forceinline__ int most_ranges(const AttnCacheArgs& a, int b) {
    return max(b == a.batch ? a.prefix_splits : a.own_splits, 1);
}
// key ranges of about `per` steps, equally long, that n steps are cut into (per = 0: one)
__device__ __forceinline__ int key_ranges(int n, int per, int most) {
    return per == 0 ? 1 : min(max((2 * n + per) / (2 * per), 1), most);
}
// steps of a range where n steps are cut into `parts`
__device__ __forceinline__ int range_steps(int n, int parts) { return max((n + parts - 1) / parts, 1); }

// Where a workgroup's walk over rising items is: the 64 sequences from b0 on, of which some
// may lie behind the last, and the items in front of them.
struct Walk {
    int b0, before;
    Sequence s;
};
// Item `idx` of the launch: the sequences in order, each with its row tiles times its key
// ranges. A lane takes one sequence, a wave scans 64 at a time. Tiles of MR rows are whole,
// inside a causal sequence the last, longest one first.
__device__ __forceinline__ RowTile find_tile(const AttnCacheArgs& a, Walk& w, const Part& part, int idx, int per) {
    const int lane = threadIdx.x & 63;
    RowTile t;
    t.found = false;
    t.b = t.q0 = t.lq = t.lk = t.row0 = t.split = 0;
    t.splits = 1;
    for (;;) {
        const int n = w.b0 + lane < part.hi ? row_tiles(a, w.s.lq, part.rows) : 0;
        const int parts = part.rows == MR ? 1 : key_ranges(steps_of(part, w.s.lk), per, most_ranges(a, w.b0 + lane));
        const int incl = wave_scan(n * parts);
        const int total = __builtin_amdgcn_readlane(incl, 63);
        const uint64_t hit = __ballot(w.before + incl > idx);
        if (idx < w.before + total && hit != 0) {
            const int src = __builtin_ctzll(hit);
            t.b = w.b0 + src;
            t.q0 = __builtin_amdgcn_readlane(w.s.q0, src);
            t.lq = __builtin_amdgcn_readlane(w.s.lq, src);
            t.lk = __builtin_amdgcn_readlane(w.s.lk, src);
            t.splits = __builtin_amdgcn_readlane(parts, src);
            const int cnt = __builtin_amdgcn_readlane(n, src);
            const int i = idx - (w.before + __builtin_amdgcn_readlane(incl, src) - cnt * t.splits);
            if (i < 0 || i >= cnt * t.splits) return t;  // (sums past 2^31: offsets that overlap many times)
            const int tile = i / t.splits;
            t.split = i - tile * t.splits;
            t.row0 = (part.rows == MR && a.causal && t.b != a.batch ? cnt - 1 - tile : tile) * part.rows;
            t.found = true;
            return t;
        }
        if (w.b0 + 64 >= part.hi) return t;
        w.before += total;
        w.b0 += 64;
        w.s = load_sequence(a, w.b0 + lane, part.hi);
    }
}
// Tiles of MR rows in shares: the steps of all tiles one behind the other, sequence by
// sequence, head by head, tile by tile (a causal tile with all of its sequence's), of
// which each workgroup takes the same number, whatever tiles they belong to.
__device__ __forceinline__ int tile_steps(const AttnCacheArgs& a, const Part& part, const Sequence& s, int b, int hi) {
    return b < hi ? row_tiles(a, s.lq, part.rows) * steps_of(part, s.lk) * part.heads : 0;
}
// steps of the sequences [lo, hi)
__device__ __forceinline__ int count_steps(const AttnCacheArgs& a, const Sequence& first, const Part& part, int hi) {
    const int lane = threadIdx.x & 63;
    int total = 0;
    for (int b0 = part.lo; b0 < hi; b0 += 64)
        total += wave_sum_dpp(tile_steps(a, part, b0 == part.lo ? first : load_sequence(a, b0 + lane, hi), b0 + lane, hi));
    return __builtin_amdgcn_readfirstlane(total);
}
// row tiles of all sequences
__device__ __forceinline__ int count_tiles(const AttnCacheArgs& a, const Sequence& first, const Part& part) {
    const int lane = threadIdx.x & 63;
    int total = 0;
    for (int b0 = part.lo; b0 < part.hi; b0 += 64) {
        const Sequence s = b0 == part.lo ? first : load_sequence(a, b0 + lane, part.hi);
        total += wave_sum_dpp(b0 + lane < part.hi ? row_tiles(a, s.lq, part.rows) : 0);
    }
    return __builtin_amdgcn_readfirstlane(total);
}
// Shares of a tile of n steps that begins at step `start`: the first one and their number.
struct Shares {
    int first, count;
};
__device__ __forceinline__ Shares tile_shares(int start, int n, int share) {
    const int first = start / share;
    return {first, n > 0 ? (start + n - 1) / share - first + 1 : 0};
}
// The tile of step x, its head and the step's number in it; t.split, t.splits: which of the
// tile's shares `of` is.
__device__ __forceinline__ RowTile find_step(const AttnCacheArgs& a, const Sequence& first, const Part& part, int x, int share,
                                             int of, int& hk, int& step) {
    const int lane = threadIdx.x & 63;
    RowTile t;
    t.found = false;
    int before = 0;
    for (int b0 = part.lo; b0 < part.hi; b0 += 64) {
        const Sequence s = b0 == part.lo ? first : load_sequence(a, b0 + lane, part.hi);
        const int v = tile_steps(a, part, s, b0 + lane, part.hi), incl = wave_scan(v);
        const int total = __builtin_amdgcn_readlane(incl, 63);
        const uint64_t hit = __ballot(before + incl > x);
        if (x < before + total && hit != 0) {
            const int src = __builtin_ctzll(hit);
            t.b = b0 + src;
            t.q0 = __builtin_amdgcn_readlane(s.q0, src);
            t.lq = __builtin_amdgcn_readlane(s.lq, src);
            t.lk = __builtin_amdgcn_readlane(s.lk, src);
            const int n = steps_of(part, t.lk), tiles = row_tiles(a, t.lq, part.rows);
            const int i = x - (before + __builtin_amdgcn_readlane(incl, src) - __builtin_amdgcn_readlane(v, src));
            const int tile = i / n;
            step = i - tile * n;
            hk = tile / tiles;
            t.row0 = (tile - hk * tiles) * part.rows;
            const Shares shares = tile_shares(x - step, n, share);
            t.split = of - shares.first;
            t.splits = shares.count;
            t.found = hk < part.heads;
            hk += part.h0;
            return t;
        }
        before += total;
    }
    return t;
}

// Steps of a range, about, or of a share; 0: tiles are whole. Lengths are known on the
// device alone, so this and the ranges follow them in a captured graph.
__device__ __forceinline__ int find_range_length(const AttnCacheArgs& a, const Sequence& first, const Part& part) {
    if (a.own_splits <= 1 && a.prefix_splits <= 1) return 0;
    const int lane = threadIdx.x & 63;
    RangeSums sums = {0.0f, 0.0f, 0.0f, 1, 0};  // no last digit is needed, but the same one everywhere
    for (int b0 = part.lo; b0 < part.hi; b0 += 64) {
        const Sequence s = b0 == part.lo ? first : load_sequence(a, b0 + lane, part.hi);
        const int n = steps_of(part, s.lk);
        const float t = b0 + lane < part.hi ? static_cast<float>(row_tiles(a, s.lq, part.rows)) : 0.0f;
        // (a causal sequence's first tile sees lq keys fewer than its last)
        const int fewer = part.rows == MR && a.causal && b0 + lane != a.batch ? steps_of(part, min(s.lq, s.lk)) : 0;
        sums.work += wave_sum_dpp(seen_steps(t, n, fewer));
        sums.all += wave_sum_dpp(seen_steps(t, n, 0));
        sums.tiles += wave_sum_dpp(t);
        const int most = max(most_ranges(a, b0 + lane) - (part.rows == MR ? 1 : 0), 1);
        sums.least = max(sums.least, wave_reduce_dpp((n + most - 1) / most, [](int x, int y) { return max(x, y); }));
        sums.longest = max(sums.longest, wave_reduce_dpp(n, [](int x, int y) { return max(x, y); }));
    }
    times_heads(sums, part.heads);
    if (part.rows == MR) return most_ranges(a, part.lo) == 1 ? 0 : share_length(sums, a.causal != 0);
    return few_length(sums, part.rows);
}
// Uniform for the compiler too, as are the totals above: a tile that it takes for divergent
// has each of its DMA instructions in a loop over descriptors (8 a step, 15 to 25% of it).
__device__ __forceinline__ int range_length(const AttnCacheArgs& a, const Sequence& first, const Part& part) {
    return __builtin_amdgcn_readfirstlane(find_range_length(a, first, part));
}

// number of keys that the query of `token` sees
__device__ __forceinline__ int visible(const AttnCacheArgs& a, const RowTile& t, int token) {
    if (!a.causal || t.b == a.batch) return t.lk;
    return min(max(token + 1 + t.lk - t.lq, 0), t.lk);
}

// E channels of an output row: acc / tot, zeros where the row sees no key
template <class T, int E>
__device__ __forceinline__ void store_row(uint16_t* op, const float (&acc)[E], float tot, bool none) {
    const float inv = 1.0f / tot;
    uint32_t st[E / 2];
#pragma unroll
    for (int c = 0; c < E / 2; ++c) st[c] = none ? 0u : T::pack(acc[2 * c] * inv, acc[2 * c + 1] * inv);
    if constexpr (E == 8)
        *reinterpret_cast<u32x4*>(op) = (u32x4){st[0], st[1], st[2], st[3]};
    else
        *reinterpret_cast<uint2*>(op) = make_uint2(st[0], st[1]);
}

// ---- few rows: 16 NR of them, the keys over the waves ------------------------
// Four waves share a tile of rows and take its 32-key tiles in turn, codes straight
// from memory to registers, the next tile's under way while one is worked on: nothing
// is shared between waves until their (O, m, sum) are joined through LDS.
//
// Products by v_mfma_f32_16x16x32, transposed: S^T = K Q^T leaves a lane (g, c) = (lane
// / 16, lane % 16) the scores of query row c and keys 4 g .. 4 g + 3 of a 16-key group,
// which are P as the second product's operand when its k index (g, j) stands for key
// 4 g + j of the first group (j < 4) or 4 g + j - 4 of the second. V^T is then four
// neighbouring keys a lane, of the D / 16 channels c D / 16 ..: a lane loads those of
// its eight keys, decodes them (a pair is two channels of one key, with that key's
// scale) and takes channel and key of pairs crosswise with v_perm_b32. The k index of
// the first product is a channel, in any order that K and Q share: a lane's 16 codes.
//
// Bound by memory where every row tile has keys of its own: one token of 64 sequences of
// 28/4 heads over 12541 to 16384 int8 keys 172 us, 5.5 TB/s (a large read reaches 6.1). By
// the vector unit where row tiles share keys, behind a prefix: 385 vector and 190 scalar
// instructions a wave and tile of 16 rows, mostly the decoding, V's crosswise pairs and
// the exponentials; 32 rows decode once for both. Small calls by latency: 16 tokens over
// up to 8192 keys 14.8 us (two or three tiles a wave), of which their 47 MB take 8. Loading
// K a whole tile earlier changed none of these. A third and fourth 16 rows did not fit the
// registers (and gave wrong rows where they spilled most).
constexpr int SW = 4;

// A wave's 32-key tile as it lies in the cache, each half loaded again as soon as it is used up
template <int D>
struct RawTile {
    u32x4 k[2][D / 64];                                  // key lane % 16 of each 16: 16 codes a chunk
    std::conditional_t<D == 128, uint2, uint32_t> v[8];  // keys 4 g + i, 16 + 4 g + i: D / 16 channels
    uint32_t ke[2], ve[2];                               // E of v's four keys each; of k's key, or those four
    int bad;                                             // bits: a 16-key group's page is not in the cache
};

// Codes without their scale as pairs of 16-bit values: K of int8, whose scale the scores
// take (8 products a lane and tile instead of 64).
template <bool BF>
__device__ __forceinline__ uint2 decode_int8_pairs(uint32_t w) {
    if constexpr (BF) {
        const v4f f = {static_cast<float>(static_cast<int8_t>(w)), static_cast<float>(static_cast<int8_t>(w >> 8)),
                       static_cast<float>(static_cast<int8_t>(w >> 16)), static_cast<float>(static_cast<int8_t>(w >> 24))};
        return make_uint2(__builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u),
                          __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u));
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const uint32_t u = w ^ 0x80808080u;
        const h2 lo = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
        const h2 hi = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
        const h2 c = {1152, 1152};
        return make_uint2(__builtin_bit_cast(uint32_t, lo - c), __builtin_bit_cast(uint32_t, hi - c));
    }
}

template <int D>
constexpr int kPitch = D + 4;  // floats per row of the joined O

template <class T, class C, int D, int NR>
__device__ __forceinline__ void few_item(const AttnCacheArgs& a, const RowTile& t, int hk, float* lds) {
    using frag = typename T::frag;
    constexpr int KS = D / 32, DT = D / 16, CH = D / 16;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int rows = t.lq * a.group;  // < 2^31: the host bounds total_q * Hq

    int kmax[NR];
    frag qf[NR][KS];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int row = min(t.row0 + 16 * r + c, rows - 1);
        const int token = row / a.group, head = hk * a.group + row % a.group;
        kmax[r] = visible(a, t, token);
        const uint16_t* qp = a.q + (static_cast<int64_t>(t.q0) + token) * a.q_t + head * a.q_h + 16 * g;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[r][s] = *reinterpret_cast<const frag*>(qp + 64 * (s / 2) + 8 * (s % 2));
    }
    const int kend = visible(a, t, (min(t.row0 + 16 * NR, rows) - 1) / a.group);
    const int kfull = visible(a, t, t.row0 / a.group);
    const int ntile = (kend + SK - 1) / SK, range = range_steps((t.lk + SK - 1) / SK, t.splits);
    const int tile0 = min(t.split * range, ntile), tile1 = min(tile0 + range, ntile);
    const int n = tile1 - tile0 > wave ? (tile1 - tile0 - wave + SW - 1) / SW : 0;

    const bool own = t.b < a.batch;
    const int* table = own ? a.table + static_cast<int64_t>(t.b) * a.max_blocks : a.prefix_table;
    const int blocks = (t.lk + (1 << a.c.page_shift) - 1) >> a.c.page_shift;  // that hold keys in use

    // K's scale is the scores'. (V's is not P's: P carries 2^kPBias, and times a small scale, below
    // 2^-126, would lose its digits or vanish. That took 180.2 to 179.2 us of one token of 64 long
    // int8 caches, 151 to 145 of 64 tokens over 4096 keys of 16 sequences.)
    constexpr bool kScores = C::kDtype == QIMG_INT8;

    // Pages of the wave's tiles, 32 at a time: lane l holds that of 16-key group l % 2 of
    // tile l / 2.
    // Addresses are a uniform row of the cache and these lane offsets.
    const uint32_t koff = c * D + 16 * g, voff = 4 * g * D + CH * c;
    RawTile<D> x;
    int ids = 0, next_bad = 0;
    int64_t rows16[2] = {0, 0};  // cache rows of the tile that is being loaded
    const auto load_k = [&](int i) __attribute__((always_inline)) {
        if ((i & 31) == 0) {
            const int group16 = 2 * (tile0 + wave + SW * (i + (lane >> 1))) + (lane & 1);
            ids = table[min(group16 >> (a.c.page_shift - 4), blocks - 1)];
            // waited for here: behind the branch the compiler would wait in every tile, and
            // for every load in flight
            asm volatile("" : "+v"(ids));
        }
        next_bad = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int page = __builtin_amdgcn_readlane(ids, 2 * (i & 31) + h);
            const bool in = page >= 0 && page < a.c.n_pages;
            next_bad |= in ? 0 : 1 << h;
            page = in ? page : 0;
            const int group16 = 2 * (tile0 + wave + SW * i) + h;
            const int64_t row = ((static_cast<int64_t>(page) * a.c.hk + hk) << a.c.page_shift) +
                                16 * (group16 & ((1 << (a.c.page_shift - 4)) - 1));
            rows16[h] = row;
            const Buffer k(a.c.k + row * D, 16 * D), e(a.c.ke + row, 16);
#pragma unroll
            for (int s = 0; s < D / 64; ++s) x.k[h][s] = k.load<u32x4>(koff, 64 * s);
            if constexpr (kScores) x.ke[h] = e.load<uint32_t>(4 * g);
            else x.ke[h] = e.load<uint8_t>(c);
        }
    };
    // of the tile whose K was loaded last
    const auto load_v = [&]() __attribute__((always_inline)) {
        x.bad = next_bad;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const Buffer v(a.c.v + rows16[h] * D, 16 * D), e(a.c.ve + rows16[h], 16);
            x.ve[h] = e.load<uint32_t>(4 * g);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x.v[4 * h + j] = v.load<std::remove_reference_t<decltype(x.v[0])>>(voff, j * D);
        }
    };

    v4f o[NR][DT], sum[NR];
    float m[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
        sum[r] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};  // all four the same
        m[r] = kNegInf;
    }
    const frag ones = as_frag<T>(T::kOnes, T::kOnes, T::kOnes, T::kOnes);

    if (n > 0) {
        load_k(0);
        load_v();
    }
    for (int i = 0; i < n; ++i) {
        const int key0 = (tile0 + wave + SW * i) * SK;
        v4f s[NR][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int r = 0; r < NR; ++r) s[r][h] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int d = 0; d < D / 64; ++d) {
                uint2 w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (kScores) w[j] = decode_int8_pairs<T::kBf>(x.k[h][d][j]);
                    else w[j] = decode_pairs<C, T::kBf>(x.k[h][d][j], exp_scale(x.ke[h]));
                }
                const frag k0 = as_frag<T>(w[0].x, w[0].y, w[1].x, w[1].y);
                const frag k1 = as_frag<T>(w[2].x, w[2].y, w[3].x, w[3].y);
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    s[r][h] = T::mma16(k0, qf[r][2 * d], s[r][h]);
                    s[r][h] = T::mma16(k1, qf[r][2 * d + 1], s[r][h]);
                }
            }
            if constexpr (kScores) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float scale = exp_scale(x.ke[h] >> 8 * j & 0xffu);
#pragma unroll
                    for (int r = 0; r < NR; ++r) s[r][h][j] *= scale;
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (i + 1 < n) load_k(i + 1);
        __builtin_amdgcn_sched_barrier(0);
        const bool hidden = key0 + SK > kfull || x.bad != 0;  // some row does not see some key, or not as it lies there
        if (hidden) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = key0 + 16 * h + 4 * g + j;
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        if (x.bad >> h & 1) s[r][h][j] = __builtin_nanf("");  // keys of a page outside the cache
                        if (key >= kmax[r]) s[r][h][j] = kNegInf;
                    }
                    // what lies there is not a number anybody wrote
                    if (key >= t.lk || (x.bad >> h & 1)) {
                        x.v[4 * h + j] = {};
                        x.ve[h] = (x.ve[h] & ~(0xffu << 8 * j)) | 127u << 8 * j;
                    }
                }
        }
        frag pf[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float mt = s[r][0][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) mt = fmaxf(mt, s[r][j >> 2][j & 3]);
            mt = quarter_max(mt) * a.scale_log2;
            const bool bump = mt > m[r] + kSlack;
            const float m_new = bump ? mt : m[r];
            if (__ballot(bump)) {
                const float f = bump ? __builtin_amdgcn_exp2f(m[r] - m_new) : 1.0f;
                sum[r] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[r][d] *= f;
            }
            m[r] = m_new;
            const float neg = (m_new == kNegInf ? 0.0f : -m_new) + T::kPBias;
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][j >> 2][j & 3], a.scale_log2, neg));
            uint32_t pk[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) pk[j] = T::pack(p[2 * j], p[2 * j + 1]);
            pf[r] = as_frag<T>(pk[0], pk[1], pk[2], pk[3]);
            sum[r] = T::mma16(ones, pf[r], sum[r]);
        }
        // four channels at a time: pairs of two channels of the eight keys, crosswise
#pragma unroll
        for (int d4 = 0; d4 < CH / 4; ++d4) {
            uint2 w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t raw;
                if constexpr (D == 128) raw = d4 == 0 ? x.v[j].x : x.v[j].y;
                else raw = x.v[j];
                w[j] = decode_pairs<C, T::kBf>(raw, exp_scale(x.ve[j / 4] >> 8 * (j & 3) & 0xffu));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t f[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t lo = e < 2 ? w[2 * j].x : w[2 * j].y, hi = e < 2 ? w[2 * j + 1].x : w[2 * j + 1].y;
                    f[j] = __builtin_amdgcn_perm(hi, lo, e % 2 == 0 ? 0x05040100u : 0x07060302u);
                }
                const frag vf = as_frag<T>(f[0], f[1], f[2], f[3]);
#pragma unroll
                for (int r = 0; r < NR; ++r) o[r][4 * d4 + e] = T::mma16(vf, pf[r], o[r][4 * d4 + e]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (i + 1 < n) load_v();
        __builtin_amdgcn_sched_barrier(0);
    }

    // the waves' shares, 16 rows at a time: O into the wave's own LDS, m and sum behind all of it
    float* osh = lds + wave * 16 * kPitch<D>;
    float(*ml)[16][2] = reinterpret_cast<float(*)[16][2]>(lds + SW * 16 * kPitch<D>);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        if (t.row0 + 16 * r >= rows) break;
        // channel CH (4 g + j) + d of query c
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int d = 0; d < DT; d += 4)
                *reinterpret_cast<v4f*>(osh + c * kPitch<D> + CH * (4 * g + j) + d) =
                    (v4f){o[r][d][j], o[r][d + 1][j], o[r][d + 2][j], o[r][d + 3][j]};
        if (g == 0) {
            ml[wave][c][0] = m[r];
            ml[wave][c][1] = sum[r][0];
        }
        __syncthreads();
        constexpr int E = D / 16;
        const int jr = threadIdx.x >> 4, c0 = (threadIdx.x & 15) * E;
        const int row = t.row0 + 16 * r + jr;
        if (row < rows) {
            float mm = ml[0][jr][0];
#pragma unroll
            for (int w = 1; w < SW; ++w) mm = fmaxf(mm, ml[w][jr][0]);
            float tot = 0.0f, acc[E];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = 0.0f;
#pragma unroll
            for (int w = 0; w < SW; ++w) {
                // no finite score: O is zero there, the sum zero or NaN
                const float mw = ml[w][jr][0];
                const float f = mw == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(mw - mm);
                tot += f * ml[w][jr][1];
                const float* src = lds + (w * 16 + jr) * kPitch<D> + c0;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += f * src[e];
            }
            const int64_t token = static_cast<int64_t>(t.q0) + row / a.group;
            const int head = hk * a.group + row % a.group;
            if (t.splits > 1 || a.prefix_splits > 0) {
                const int parts = a.own_splits + a.prefix_splits;
                const int64_t at = (token * a.hq + head) * parts + (own ? 0 : a.own_splits) + t.split;
                float* po = a.part_o + at * D + c0;
#pragma unroll
                for (int e = 0; e < E; e += 4)
                    *reinterpret_cast<v4f*>(po + e) = (v4f){acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
                if (c0 == 0) {
                    a.part_ml[2 * at] = mm;
                    a.part_ml[2 * at + 1] = tot;
                }
            } else {
                store_row<T, E>(a.out + token * a.o_t + head * a.o_h + c0, acc, tot, tot == 0.0f);
            }
        }
        __syncthreads();  // the next rows take the place of O
    }
}

template <int D>
constexpr int kFewLds = SW * 16 * (kPitch<D> + 2);  // floats

// Workgroup `block` of `blocks` walks over the items.
template <class T, class C, int D, int NR>
__device__ __forceinline__ void few_items(const AttnCacheArgs& a, const Part& part, int block, int blocks, float* lds) {
    Walk w = {part.lo, 0, load_sequence(a, part.lo + (threadIdx.x & 63), part.hi)};
    const int per = range_length(a, w.s, part);
    for (int item = block;; item += blocks) {
        const RowTile t = find_tile(a, w, part, item / a.c.hk, per);
        if (!t.found) return;
        few_item<T, C, D, NR>(a, t, item % a.c.hk, lds);
    }
}

template <class T, class C, int D, int NR>
__global__ __launch_bounds__(SW * 64, NR == 1 ? 3 : 2) void attn_cache_few_kernel(AttnCacheArgs a, Part part) {
    __shared__ __attribute__((aligned(16))) float lds[kFewLds<D>];
    few_items<T, C, D, NR>(a, part, blockIdx.x, gridDim.x, lds);
}

// ---- many rows: 128 of them, four waves over one ring -----------------------
// Codes decoded once: attn_cache_decode_kernel writes a part's keys to scratch as 16-bit
// rows, head by head, and the work on them is attention_varlen.hip's (its tiles, waves
// and phases, of which attention_tiles.h holds what both share). Decoding on the way into
// LDS instead, 64 codes a thread and step, took no pass of its own, but each tile of rows
// does it anew: with seven tiles a head (128 tokens of 28/4 heads over 16000 int8 keys)
// the loop took 52 us (45 here, and 11 for the decoding, beside the own keys' tiles), with
// fifty (1024 tokens over 8192 e4m3 keys and 333 over 2381) 169 (133 and 9).
//
// Bound by the softmax's vector instructions and the matrix unit in turn, which work about
// half of the time each: 2.0 us a step of two workgroups, 1.07 PFLOP/s in the steps (a
// large product 1.3). A launch in shares also starts, and writes and joins partial
// results, 64 KB a workgroup: 18 us of the 45 and of the 133, 12 and 16 of the joins.
//
// Where the CUs want more than whole tiles (range_length), the tiles' steps are dealt out
// in equal shares and a tile's parts joined.

// Rows of a sequence's slot in scratch: whole 64-key tiles of what its table holds.
__device__ __forceinline__ int64_t slot_rows(const AttnCacheArgs& a, int b) {
    const int64_t keys = static_cast<int64_t>(b < a.batch ? a.max_blocks : a.prefix_blocks) << a.c.page_shift;
    return (keys + MK - 1) / MK * MK;
}

// One tile of 64 keys of one head a workgroup. Keys of a page outside the cache are NaN.
// Bound by memory: 8192 and 2381 e4m3 keys of 4 heads, 54 MB, 9 us.
template <class T, class C, int D>
__device__ __forceinline__ void decode_tile(const AttnCacheArgs& a, const Part& part, int tiles, int block) {
    const int tile = block % tiles, at = block / tiles;
    const int head = at % part.heads, slot = at / part.heads, b = part.lo + slot;
    const Sequence s = load_sequence(a, b, part.hi);
    if (s.lq == 0 || tile * MK >= s.lk) return;
    const int* table = b < a.batch ? a.table + static_cast<int64_t>(b) * a.max_blocks : a.prefix_table;
    const int last = ((s.lk + (1 << a.c.page_shift) - 1) >> a.c.page_shift) - 1;
    constexpr int TPR = D / 16, N = MK * TPR / 256;
    int page[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
        page[i] = table[min((tile * MK + static_cast<int>(threadIdx.x) / TPR + 256 / TPR * i) >> a.c.page_shift, last)];
    const int64_t base = (static_cast<int64_t>(slot) * part.heads + head) * slot_rows(a, b) * D;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int key = tile * MK + static_cast<int>(threadIdx.x) / TPR + 256 / TPR * i, c = 16 * (threadIdx.x % TPR);
        const bool in = page[i] >= 0 && page[i] < a.c.n_pages;
        const int64_t row = ((static_cast<int64_t>(in ? page[i] : 0) * a.c.hk + part.h0 + head) << a.c.page_shift) +
                            (key & ((1 << a.c.page_shift) - 1));
        const u32x4 kw = *reinterpret_cast<const u32x4*>(a.c.k + row * D + c), vw = *reinterpret_cast<const u32x4*>(a.c.v + row * D + c);
        const float ks = exp_scale(a.c.ke[row]), vs = exp_scale(a.c.ve[row]);
        u32x4 r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint2 k = decode_pairs<C, T::kBf>(kw[j], ks), v = decode_pairs<C, T::kBf>(vw[j], vs);
            r[j / 2][j % 2 * 2] = in ? k.x : T::kNans, r[j / 2][j % 2 * 2 + 1] = in ? k.y : T::kNans;
            r[2 + j / 2][j % 2 * 2] = in ? v.x : 0u, r[2 + j / 2][j % 2 * 2 + 1] = in ? v.y : 0u;
        }
        uint16_t* ko = a.dense_k + base + static_cast<int64_t>(key) * D + c;
        uint16_t* vo = a.dense_v + base + static_cast<int64_t>(key) * D + c;
        *reinterpret_cast<u32x4*>(ko) = r[0];
        *reinterpret_cast<u32x4*>(ko + 8) = r[1];
        *reinterpret_cast<u32x4*>(vo) = r[2];
        *reinterpret_cast<u32x4*>(vo + 8) = r[3];
    }
}

template <class T, class C, int D>
__global__ __launch_bounds__(256) void attn_cache_decode_kernel(AttnCacheArgs a, Part part, int tiles, int first) {
    decode_tile<T, C, D>(a, part, tiles, first + blockIdx.x);
}

// The first `few` workgroups work on the sequences' own keys in tiles of few rows, the
// others decode the prefix for its tiles of MR, mostly behind them where they are as many as
// run at once: a launch less. 16000 int8 keys beside 128 sequences of 1 to 509: 20 us; in two
// launches, the decoding first, 23, and in the launch of the prefix' tiles instead the own
// keys took 9 to 10 besides the 11.
template <class T, class C, int D, int NR>
__global__ __launch_bounds__(SW * 64, NR == 1 ? 3 : 2) void attn_cache_mixed_kernel(AttnCacheArgs a, Part own, int few,
                                                                                    Part prefix, int tiles) {
    __shared__ __attribute__((aligned(16))) float lds[kFewLds<D>];
    if (static_cast<int>(blockIdx.x) < few)
        few_items<T, C, D, NR>(a, own, blockIdx.x, few, lds);
    else
        decode_tile<T, C, D>(a, prefix, tiles, static_cast<int>(blockIdx.x) - few);
}

template <int D>
constexpr int kManyLds = MSLOT * 2 * MK * D * 2;  // bytes

// Key tiles [tile0, tile0 + n) of a row tile.
template <class T, int D>
__device__ __forceinline__ void many_item(const AttnCacheArgs& a, const Part& part, const RowTile& t, int hk, int tile0, int n,
                                          uint8_t* lds) {
    using W = Many<T, D>;
    constexpr int PAIR = 2 * W::TB;
    static_assert(MSLOT * PAIR == kManyLds<D>, "LDS of the kernels");

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, half = lane >> 5;
    const int rows = t.lq * a.group;
    const int row = min(t.row0 + 32 * wave + l32, rows - 1);
    const bool valid = t.row0 + 32 * wave + l32 < rows;
    const int token = row / a.group, head = hk * a.group + row % a.group;
    const int kmax = visible(a, t, token), kfull = visible(a, t, t.row0 / a.group);
    const bool own = t.b < a.batch;

    W w;
#pragma unroll
    for (int d = 0; d < W::DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) w.o[d][r] = 0.0f;
    w.m = kNegInf;
    w.sum = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    if (n > 0) {
        const int64_t room = slot_rows(a, t.b);
        const int64_t base = (static_cast<int64_t>(t.b - part.lo) * part.heads + hk - part.h0) * room * D;
        TileStream<D, false> ks;
        TileStream<D, true> vs;
        ks.init(a.dense_k + base, D, t.lk, tile0, 1, wave);
        ks.issue(lds + W::TB, wave);
        {
            const uint16_t* qp = a.q + (static_cast<int64_t>(t.q0) + token) * a.q_t + head * a.q_h + 8 * half;
#pragma unroll
            for (int i = 0; i < W::KS; ++i) w.qf[i] = *reinterpret_cast<const typename T::frag*>(qp + 16 * i);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < W::DT; ++d) w.voff[d] = v_lane_off<D>(d);
#pragma unroll
        for (int c = 0; c < W::KS; ++c) w.koff[c] = l32 * (2 * D) + swz_k<D>(l32, 2 * c + half) * 16;
#pragma unroll
        for (int r = 0; r < 16 * W::KB; ++r) w.s[r >> 4][r & 15] = 0.0f;
        vs.init(a.dense_v + base, D, t.lk, tile0, 1, wave);
        __builtin_amdgcn_sched_barrier(0);
        vs.issue(lds + PAIR, wave);
        ks.issue(lds + PAIR + W::TB, wave);
        wait_vmcnt<W::PER>();
        phase_barrier();
        w.template first_scores<W::NPV>(lds);
        // V(p) and M(p + 1): behind the barrier every wave has done M(p), whose slot takes pair p + 2
        // during V(p), and pair p + 1, sent during V(p - 1), has landed
        const auto step = [&](int p, const uint8_t* __restrict src, uint8_t* __restrict dst) __attribute__((always_inline)) {
            wait_vmcnt<0>();
            phase_barrier();
            w.template read_group<0>(src, w.buf[0]);
            __builtin_amdgcn_sched_barrier(0);
            w.softmax((tile0 + p) * MK, kfull, kmax, a.scale_log2, [&](int i) {
                if (i < W::PER / 2)
                    vs.issue_one(i, dst, wave);
                else
                    ks.issue_one(i - W::PER / 2, dst + W::TB, wave);
            });
#pragma unroll
            for (int i = 0; i < 8 * W::KB; ++i) asm volatile("" : "+v"(w.pk[i]));  // P is made in this phase
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            bool none = false;
            w.template m_groups<0, false>(src, none);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
        };
        for (int p = 0; p < n; ++p) step(p, lds + ((p + 1) % MSLOT) * PAIR, lds + (p % MSLOT) * PAIR);
        wait_vmcnt<0>();  // the loads past the last tile no longer write the ring
    }
    const float tot = half_sum(w.sum[0]);
    constexpr int CHUNKS = D / 8;
    if (t.splits > 1 || a.prefix_splits > 0) {
        if (!valid) return;
        const int64_t at = ((static_cast<int64_t>(t.q0) + token) * a.hq + head) * (a.own_splits + a.prefix_splits) +
                           (own ? 0 : a.own_splits) + t.split;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            *reinterpret_cast<v4f*>(a.part_o + at * D + 32 * (c / 4) + 8 * (c % 4) + 4 * half) =
                (v4f){w.o[c / 4][c % 4 * 4], w.o[c / 4][c % 4 * 4 + 1], w.o[c / 4][c % 4 * 4 + 2],
                      w.o[c / 4][c % 4 * 4 + 3]};
        if (half == 0) {
            a.part_ml[2 * at] = w.m;
            a.part_ml[2 * at + 1] = tot;
        }
        return;
    }
    if (!valid) return;
    const float inv = 1.0f / tot;
    // channels 8 (g + half) .. of block d after the lane halves have exchanged
    // their four of g and g + 1
    uint16_t* op = a.out + (static_cast<int64_t>(t.q0) + token) * a.o_t + head * a.o_h + 8 * half;
#pragma unroll
    for (int d = 0; d < W::DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t x = T::pack(w.o[d][4 * g + 2 * i] * inv, w.o[d][4 * g + 2 * i + 1] * inv);
                const uint32_t y = T::pack(w.o[d][4 * g + 4 + 2 * i] * inv, w.o[d][4 * g + 4 + 2 * i + 1] * inv);
                const auto sw = __builtin_amdgcn_permlane32_swap(x, y, false, false);
                v[i] = tot == 0.0f ? 0u : sw[0];
                v[2 + i] = tot == 0.0f ? 0u : sw[1];
            }
            *reinterpret_cast<u32x4*>(op + 32 * d + 8 * g) = (u32x4){v[0], v[1], v[2], v[3]};
        }
}

// Workgroup `block`: a tile, or its share of the steps.
template <class T, int D>
__device__ __forceinline__ void many_items(const AttnCacheArgs& a, const Part& part, int block, uint8_t* lds) {
    const Sequence first = load_sequence(a, part.lo + (threadIdx.x & 63), part.hi);
    const int share = range_length(a, first, part);
    // Neighbours, which read the same keys, on one XCD; whole causal tiles, longest first, over
    // all of them.
    const bool spread = share == 0 && a.causal && part.lo < a.batch;
    int total = 0, me = block;
    if (!spread) {
        total = share == 0 ? count_tiles(a, first, part) * part.heads : count_steps(a, first, part, part.hi);
        const int blocks = share == 0 ? total : (total + share - 1) / share;
        if (block >= blocks) return;
        me = xcd_remap(block, blocks);
    }
    const int end = share == 0 ? 1 : min((me + 1) * share, total);
    for (int x = share == 0 ? 0 : me * share; x < end;) {
        int hk = 0, step = 0;
        RowTile t;
        if (share == 0) {
            const int tiles = total / part.heads;
            hk = part.h0 + (spread ? me % part.heads : me / tiles);
            Walk w = {part.lo, 0, first};
            t = find_tile(a, w, part, spread ? me / part.heads : me % tiles, 0);
        } else {
            t = find_step(a, first, part, x, share, me, hk, step);
        }
        if (!t.found) return;
        const int all = (t.lk + MK - 1) / MK;
        const int seen = (visible(a, t, (min(t.row0 + MR, t.lq * a.group) - 1) / a.group) + MK - 1) / MK;
        const int n = share == 0 ? all : min(all - step, end - x);
        many_item<T, D>(a, part, t, hk, step, min(n, seen - step), lds);
        if (share == 0) return;
        x += n;
        if (x < end) __syncthreads();  // (the next tile's keys take the place of this one's)
    }
}

template <class T, int D>
__global__ __launch_bounds__(MW * 64, 2) void attn_cache_many_kernel(AttnCacheArgs a, Part part) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kManyLds<D>];
    many_items<T, D>(a, part, blockIdx.x, lds);
}

// Partial results of a row: 16 threads add every G-th of them in order, eight parts' loads
// going out together, and the G sums meet in the wave; tiles of 16 / G rows of one sequence
// and kv head. Bound by latency, or the parts' bytes: 1357 tokens of 28 heads in up to four
// parts 16.5 us. G = 4 where tiles of 16 rows would leave CUs idle: 16 tokens of 28/4 heads
// in up to 32 parts 5.2 us (7.5 with G = 1), but 128 tokens 17 (12).
template <class T, int D, int G>
__device__ __forceinline__ void join_item(const AttnCacheArgs& a, const RowTile& t, int hk, int own, int shared) {
    constexpr int E = D / 16, U = 8;
    typedef float v2f __attribute__((ext_vector_type(2)));
    const int row = t.row0 + threadIdx.x / (16 * G), c0 = (threadIdx.x & 15) * E, g = (threadIdx.x >> 4) % G;
    if (row >= t.lq * a.group) return;
    const int64_t token = static_cast<int64_t>(t.q0) + row / a.group;
    const int head = hk * a.group + row % a.group;
    const int64_t at = (token * a.hq + head) * (a.own_splits + a.prefix_splits);
    const int n = own + shared;
    float mm = kNegInf, tot = 0.0f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    for (int s0 = g; s0 < n; s0 += U * G) {
        v2f ml[U];
        v4f v[U][E / 4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = min(s0 + u * G, n - 1);
            const int64_t p = at + (s < own ? s : a.own_splits + s - own);
            ml[u] = *reinterpret_cast<const v2f*>(a.part_ml + 2 * p);
#pragma unroll
            for (int e = 0; e < E / 4; ++e) v[u][e] = *reinterpret_cast<const v4f*>(a.part_o + p * D + c0 + 4 * e);
        }
        float top = mm;
#pragma unroll
        for (int u = 0; u < U; ++u) top = fmaxf(top, ml[u][0]);
        const float old = mm == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(mm - top);
        mm = top;
        tot *= old;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= old;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u * G >= n) continue;
            // no finite score: O is zero there, the sum zero or NaN
            const float f = ml[u][0] == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(ml[u][0] - mm);
            tot += f * ml[u][1];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += f * v[u][e / 4][e % 4];
        }
    }
#pragma unroll
    for (int step = 16; step < 16 * G; step *= 2) {
        const float top = fmaxf(mm, __shfl_xor(mm, step));
        const float f = mm == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(mm - top);
        mm = top;
        tot *= f;
        tot += __shfl_xor(tot, step);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            acc[e] *= f;
            acc[e] += __shfl_xor(acc[e], step);
        }
    }
    if (g != 0) return;
    store_row<T, E>(a.out + token * a.o_t + head * a.o_h + c0, acc, tot, tot == 0.0f);
}

template <class T, int D, int G>
__global__ __launch_bounds__(256) void attn_cache_join_kernel(AttnCacheArgs a, Part own_part, Part prefix_part) {
    const int lane = threadIdx.x & 63;
    const Sequence first = load_sequence(a, lane, own_part.hi);
    const int per = range_length(a, first, own_part);
    Sequence p = {0, 0, 0};
    int prefix_per = 0;
    if (a.prefix_splits > 0) {
        p = load_sequence(a, a.batch, a.batch + 1);
        // (one launch of both has one length of ranges)
        prefix_per = own_part.hi > a.batch ? per : range_length(a, load_sequence(a, a.batch + lane, prefix_part.hi), prefix_part);
    }
    const Part rows = {0, a.batch, 16 / G, 0, a.c.hk};
    Walk w = {0, 0, first};
    for (int item = blockIdx.x;; item += gridDim.x) {
        const int hk = item % a.c.hk;
        const RowTile t = find_tile(a, w, rows, item / a.c.hk, 0);
        if (!t.found) return;
        const int n = steps_of(own_part, t.lk);
        int own = 1, shared = 0;
        if (own_part.rows != MR) {
            own = key_ranges(n, per, max(a.own_splits, 1));
        } else if (per != 0) {
            const int tiles = row_tiles(a, t.lq, MR), before = count_steps(a, first, own_part, t.b);
            own = tile_shares(before + (hk * tiles + t.row0 / MR) * n, n, per).count;
        }
        if (a.prefix_splits == 0) {
            if (own == 1) continue;  // complete already
        } else if (prefix_part.rows != MR) {
            shared = key_ranges(steps_of(prefix_part, p.lk), prefix_per, a.prefix_splits);
        } else {
            // a row's tile of the prefix, whose rows are those of all sequences
            const int np = steps_of(prefix_part, p.lk), tiles = row_tiles(a, p.lq, MR);
            const int row = min(t.row0 + static_cast<int>(threadIdx.x / (16 * G)), t.lq * a.group - 1);
            const int tile = static_cast<int>(((static_cast<int64_t>(t.q0) - p.q0) * a.group + row) / MR);
            shared = prefix_per == 0 ? 1 : tile_shares((hk * tiles + tile) * np, np, prefix_per).count;
        }
        join_item<T, D, G>(a, t, hk, own, shared);
    }
}

// upper bound on the tiles of `rows` rows that the sequences have
int64_t tile_bound(int total_q, int batch, int group, int rows) {
    const int64_t seqs = batch < total_q ? batch : total_q;
    return (static_cast<int64_t>(total_q) * group + seqs * (rows - 1)) / rows;
}

}  // namespace

constexpr int kMostSplits = 32;
constexpr int kCus = 256, kJoinGrid = 4096;
constexpr int kFewTiles = 320;  // of 32 rows that the card works on without those of MR
constexpr int kWorkTogether = 24000, kWorkOf32 = 40000;  // products of 16 rows and 32 keys behind a prefix
constexpr int kMostBlocks = 1 << 22;  // of a launch (a grid has less than 2^32 threads)
constexpr int64_t kMostDense = int64_t{1} << 30;  // bytes of 16-bit rows at a time, of one head of a sequence at least

AttnCachePlan attn_cache_plan(int total_q, int batch, int hq, int hk, int D, int64_t own_keys, int64_t prefix_keys) {
    AttnCachePlan p{};
    if (total_q <= 0 || batch <= 0) return p;
    const int group = hq / hk;
    // Rows of a tile. Rows of MR have their keys decoded into scratch first, which pays once some
    // hundred rows use them and there are tiles for the workgroups; 28/4 heads of 128, e4m3, MR
    // rows and 32, in us: 16 tokens at 4096 keys 27.4, 15.2, of 32 sequences 159, 68; 64 tokens
    // at 4096 of 16 sequences 135, 116; 300 at 300 keys 15.8, 15.4, of 4 sequences 20.3, 32.9;
    // 200 at 2000 of 8 sequences 70, 95; 512 at 4096 58.9, 58.5.
    const auto fits = [&](int rows, int seqs) { return tile_bound(total_q, seqs, group, rows) * hk < kMostBlocks; };
    const int64_t rows = (static_cast<int64_t>(total_q) * group + batch - 1) / batch;  // of a sequence, on average
    if (rows <= 16)
        p.own_rows = 16;
    else if (rows <= 512 || tile_bound(total_q, batch, group, 32) * hk <= kFewTiles || !fits(MR, batch))
        p.own_rows = 32;
    else
        p.own_rows = MR;
    // Behind a prefix by the products of 16 rows and 32 keys. One launch for both parts is best
    // while they are few, then tiles of 32 rows, then MR; one token each with 40 keys of its
    // own, MR rows, 32, and the own part's 16, in us: 16 tokens behind 4096 keys 30.8, 21.5,
    // 15.9; 64 behind 4096 35.1, 30.2, 28.5; 128 behind 4096 43.1, 39.3, 48.7; 256 behind 4096
    // 61.3, 64.7, 81.7; 128 behind 16384 72.7, 90.6, 114.7; int8 256 behind 4096 62.2, 73.5.
    const int64_t work = (static_cast<int64_t>(total_q) * group + 15) / 16 * ((prefix_keys + 31) / 32) * hk;
    p.prefix_rows = work <= kWorkTogether && p.own_rows != MR ? p.own_rows : work <= kWorkOf32 || !fits(MR, 1) ? 32 : MR;
    // Most ranges of a sequence: eight steps each at least, and 2^13 row tiles times ranges; of
    // MR rows the shares that may meet in a tile, up to 1.5 tiles a workgroup.
    const auto splits = [&](int64_t keys, int rows, int seqs) -> int {
        const int64_t tiles = std::max<int64_t>(tile_bound(total_q, seqs, group, rows) * hk, 1);
        if (rows == MR) {
            const int64_t steps = (keys + MK - 1) / MK;
            const bool pays = shares_pay(static_cast<float>(tiles * steps) / kManyGrid, static_cast<float>(tiles),
                                         static_cast<float>((tiles + kManyGrid - 1) / kManyGrid * steps));
            return tiles > kManyGrid * 3 / 2 || !pays
                       ? 1
                       : static_cast<int>(std::min<int64_t>({kManyGrid / tiles + 2, (steps + 3) / 4 + 1, kMostSplits}));
        }
        const int64_t most = std::min<int64_t>((keys + 8 * SK - 1) / (8 * SK), 8192 / tiles);
        return static_cast<int>(std::max<int64_t>(std::min<int64_t>(most, kMostSplits), 1));
    };
    p.own_splits = splits(own_keys, p.own_rows, batch);
    p.prefix_splits = prefix_keys > 0 ? splits(prefix_keys, p.prefix_rows, 1) : 0;
    // The 16-bit rows of a part in tiles of MR: as many heads, or sequences, at a time as
    // kMostDense holds. Where that is not all there are no shares.
    const auto dense = [&](int64_t keys, int rows, int seqs, int& slots, int& heads, int& splits) {
        slots = seqs, heads = hk;
        if (rows != MR || keys == 0) return;
        const int64_t slot = (keys + MK - 1) / MK * MK, each = slot * D * 4, most = std::max<int64_t>(kMostDense / each, 1);
        if (most < static_cast<int64_t>(seqs) * hk) {
            splits = std::min(splits, 1);
            heads = static_cast<int>(std::clamp<int64_t>(most / seqs, 1, hk));
            slots = static_cast<int>(std::min<int64_t>(most / heads, seqs));
        }
        p.dense_rows = std::max(p.dense_rows, slot * slots * heads);
    };
    int one = 1;
    dense(own_keys, p.own_rows, batch, p.own_slots, p.own_heads, p.own_splits);
    dense(prefix_keys, p.prefix_rows, 1, one, p.prefix_heads, p.prefix_splits);
    if (p.own_splits > 1 || p.prefix_splits > 0)
        p.part_rows = static_cast<int64_t>(total_q) * hq * (p.own_splits + p.prefix_splits);
    return p;
}

AttnCacheScratch attn_cache_scratch(const AttnCachePlan& plan, int D) {
    const auto align = [](int64_t n) { return (n + 255) / 256 * 256; };
    return {align(plan.part_rows * D * 4), align(plan.part_rows * 8), align(plan.dense_rows * D * 2)};
}

template <class T, class C, int D>
static hipError_t launch_attn(const AttnCacheArgs& a, const AttnCachePlan& plan, hipStream_t stream) {
    const bool prefix = plan.prefix_splits > 0;
    // few rows of both: one launch over them all
    const bool together = prefix && plan.prefix_rows == plan.own_rows && plan.own_rows != MR;
    const Part own = {0, a.batch + (together ? 1 : 0), plan.own_rows, 0, a.c.hk};
    const Part shared = {a.batch, a.batch + 1, plan.prefix_rows, 0, a.c.hk};
    const dim3 block(MW * 64);
    static_assert(MW == SW && SW == 4, "workgroups of 256 for all");
    // workgroups of MR rows: the tiles, or the shares of those that run at once
    const auto many = [&](int seqs, int heads, int splits) {
        const int64_t tiles = tile_bound(a.total_q, seqs, a.group, MR) * heads;
        return static_cast<unsigned>(splits > 1 ? std::max<int64_t>(tiles, kManyGrid) : tiles);
    };
    // of few rows: they walk over the items
    const auto few = [&](bool with_own, bool with_prefix, int rows) {
        int64_t items = with_own ? tile_bound(a.total_q, a.batch, a.group, rows) * a.own_splits : 0;
        if (with_prefix) items += tile_bound(a.total_q, 1, a.group, rows) * a.prefix_splits;
        return static_cast<unsigned>(std::min<int64_t>(items * a.c.hk, few_grid(rows)));
    };
    // the codes of a part as 16-bit rows in scratch; with the own part's few rows if they are asked for
    const auto decode = [&](const Part& part, bool with_own) {
        const int64_t keys = static_cast<int64_t>(part.lo < a.batch ? a.max_blocks : a.prefix_blocks) << a.c.page_shift;
        const int tiles = static_cast<int>((keys + MK - 1) / MK);
        // (scratch bounds them: below 2^25)
        const int blocks = static_cast<int>(static_cast<int64_t>(tiles) * part.heads * (part.hi - part.lo));
        int first = 0;
        if (const int more = with_own ? static_cast<int>(few(true, false, own.rows)) : 0; more > 0) {
            first = std::min(blocks, kMostBlocks);
            if (own.rows == 16)
                hipLaunchKernelGGL((attn_cache_mixed_kernel<T, C, D, 1>), dim3(more + first), block, 0, stream, a, own, more,
                                   part, tiles);
            else
                hipLaunchKernelGGL((attn_cache_mixed_kernel<T, C, D, 2>), dim3(more + first), block, 0, stream, a, own, more,
                                   part, tiles);
        }
        for (; first < blocks; first += kMostBlocks)
            hipLaunchKernelGGL((attn_cache_decode_kernel<T, C, D>), dim3(std::min(blocks - first, kMostBlocks)), block, 0, stream,
                               a, part, tiles, first);
        return hipGetLastError();
    };
    bool own_done = false;
    hipError_t e = hipSuccess;
    if (prefix && shared.rows == MR) {
        for (int h = 0; h < a.c.hk && e == hipSuccess; h += plan.prefix_heads) {
            Part part = shared;
            part.h0 = h, part.heads = std::min(plan.prefix_heads, a.c.hk - h);
            e = decode(part, h == 0 && own.rows != MR);
            if (e != hipSuccess) break;
            own_done = own.rows != MR;
            hipLaunchKernelGGL((attn_cache_many_kernel<T, D>), dim3(many(1, part.heads, a.prefix_splits)), block, 0, stream, a,
                               part);
            e = hipGetLastError();
        }
    } else if (prefix && !together) {  // of 32 rows, where the sequences' own tiles have 16
        hipLaunchKernelGGL((attn_cache_few_kernel<T, C, D, 2>), dim3(few(false, true, 32)), block, 0, stream, a, shared);
        e = hipGetLastError();
    }
    if (e == hipSuccess && own.rows == MR) {
        for (int b = 0; b < a.batch; b += plan.own_slots) {
            for (int h = 0; h < a.c.hk; h += plan.own_heads) {
                const Part part = {b, std::min(b + plan.own_slots, a.batch), MR, h, std::min(plan.own_heads, a.c.hk - h)};
                e = decode(part, false);
                if (e != hipSuccess) return e;
                hipLaunchKernelGGL((attn_cache_many_kernel<T, D>), dim3(many(part.hi - part.lo, part.heads, a.own_splits)),
                                   block, 0, stream, a, part);
                e = hipGetLastError();
                if (e != hipSuccess) return e;
            }
        }
    } else if (e == hipSuccess && !own_done) {
        if (own.rows == 16)
            hipLaunchKernelGGL((attn_cache_few_kernel<T, C, D, 1>), dim3(few(true, together, 16)), block, 0, stream, a, own);
        else
            hipLaunchKernelGGL((attn_cache_few_kernel<T, C, D, 2>), dim3(few(true, together, 32)), block, 0, stream, a, own);
        e = hipGetLastError();
    }
    if (e != hipSuccess || plan.part_rows == 0) return e;
    const auto join = [&](auto g) {
        constexpr int G = decltype(g)::value;
        const int64_t tiles = std::min<int64_t>(tile_bound(a.total_q, a.batch, a.group, 16 / G) * a.c.hk, kJoinGrid);
        hipLaunchKernelGGL((attn_cache_join_kernel<T, D, G>), dim3(static_cast<unsigned>(tiles)), dim3(256), 0, stream, a, own,
                           shared);
    };
    if (tile_bound(a.total_q, a.batch, a.group, 16) * a.c.hk > kCus)
        join(std::integral_constant<int, 1>{});
    else
        join(std::integral_constant<int, 4>{});
    return hipGetLastError();
}

hipError_t launch_attention_cache(const AttnCacheArgs& a, const AttnCachePlan& plan, int dtype, int codes, int D,
                                  hipStream_t stream) {
    const auto with_codes = [&](auto t, auto d) {
        using T = decltype(t);
        constexpr int HD = decltype(d)::value;
        return codes == QIMG_INT8 ? launch_attn<T, Int8Codes, HD>(a, plan, stream)
                                  : launch_attn<T, E4m3Codes, HD>(a, plan, stream);
    };
    const auto with_type = [&](auto d) { return dtype == QIMG_BF16 ? with_codes(Bf16{}, d) : with_codes(Fp16{}, d); };
    return D == 128 ? with_type(std::integral_constant<int, 128>{}) : with_type(std::integral_constant<int, 64>{});
}

}  // namespace qimg
