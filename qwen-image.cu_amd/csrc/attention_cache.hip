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
// key ranges of about `per` tiles of SK keys, equally long, that lk keys are cut into
constexpr int SK = 32;
__device__ __forceinline__ int key_ranges(int lk, int per) {
    if (per == 0) return 1;
    const int n = (lk + SK - 1) / SK;
    return max((2 * n + per) / (2 * per), 1);
}

// Item `idx` of the sequences [lo, hi): in order, each with its tiles of `rows` rows
// times its key ranges of about `per` key tiles. A lane takes one sequence, a wave
// scans 64 at a time, the first 64 (`first`, of which some may lie behind hi) loaded once
// by the caller.
__device__ __forceinline__ RowTile find_tile(const AttnCacheArgs& a, const Sequence& first, int lo, int hi, int idx,
                                             int rows, int per) {
    const int lane = threadIdx.x & 63;
    RowTile t;
    t.found = false;
    t.b = t.q0 = t.lq = t.lk = t.row0 = t.split = 0;
    t.splits = 1;
    int before = 0;
    for (int b0 = lo; b0 < hi; b0 += 64) {
        const Sequence s = b0 == lo ? first : load_sequence(a, b0 + lane, hi);
        const int n = b0 + lane < hi ? row_tiles(a, s.lq, rows) : 0, parts = key_ranges(s.lk, per);
        const int incl = wave_scan(n * parts);
        const int total = __builtin_amdgcn_readlane(incl, 63);
        const uint64_t hit = __ballot(before + incl > idx);
        if (idx < before + total && hit != 0) {
            const int src = __builtin_ctzll(hit);
            t.b = b0 + src;
            t.q0 = __builtin_amdgcn_readlane(s.q0, src);
            t.lq = __builtin_amdgcn_readlane(s.lq, src);
            t.lk = __builtin_amdgcn_readlane(s.lk, src);
            t.splits = __builtin_amdgcn_readlane(parts, src);
            const int cnt = __builtin_amdgcn_readlane(n, src);
            const int i = idx - (before + __builtin_amdgcn_readlane(incl, src) - cnt * t.splits);
            if (i < 0 || i >= cnt * t.splits) return t;  // (sums past 2^31: offsets that overlap many times)
            const int tile = i / t.splits;
            t.split = i - tile * t.splits;
            // (inside a causal sequence the last, longest tile first)
            t.row0 = (rows == MR && a.causal && t.b != a.batch ? cnt - 1 - tile : tile) * rows;
            t.found = true;
            return t;
        }
        before += total;
    }
    return t;
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
constexpr int SW = 4;
constexpr int kFewGrid = 1024;  // workgroups of the launch at most

// Key tiles per range, about: as many as make the launch one item a workgroup, at least
// two a wave, at most a.own_splits (prefix_splits) ranges a sequence. 0: no ranges.
__device__ __forceinline__ int range_tiles(const AttnCacheArgs& a, const Sequence& first, int lo, int hi, int rows) {
    if (a.own_splits <= 1 && a.prefix_splits <= 1) return 0;
    const int lane = threadIdx.x & 63;
    int least = 1;
    float work = 0.0f, tiles = 0.0f;  // key tiles of all row tiles, row tiles: sums that need no last digit
    for (int b0 = lo; b0 < hi; b0 += 64) {
        const Sequence s = b0 == lo ? first : load_sequence(a, b0 + lane, hi);
        const int kt = (s.lk + SK - 1) / SK;
        const float n = static_cast<float>(row_tiles(a, s.lq, rows));
        work += wave_sum_dpp(n * static_cast<float>(kt));
        tiles += wave_sum_dpp(n);
        const int most = max(b0 + lane == a.batch ? a.prefix_splits : a.own_splits, 1);
        least = max(least, wave_reduce_dpp((kt + most - 1) / most, [](int x, int y) { return max(x, y); }));
    }
    work *= static_cast<float>(a.c.hk);
    tiles *= static_cast<float>(a.c.hk);
    // (offsets that overlap may sum to any number)
    const int per = static_cast<int>(fminf(work / fmaxf(kFewGrid, 1.25f * tiles), 0x1p25f)) + 1;
    return __builtin_amdgcn_readfirstlane(max(max(per, 2 * SW), least));
}

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
    const int ntile = (kend + SK - 1) / SK, range = ((t.lk + SK - 1) / SK + t.splits - 1) / t.splits;
    const int tile0 = min(t.split * range, ntile), tile1 = min(tile0 + range, ntile);
    const int n = tile1 - tile0 > wave ? (tile1 - tile0 - wave + SW - 1) / SW : 0;

    const bool own = t.b < a.batch;
    const int* table = own ? a.table + static_cast<int64_t>(t.b) * a.max_blocks : a.prefix_table;
    const int blocks = (t.lk + (1 << a.c.page_shift) - 1) >> a.c.page_shift;  // that hold keys in use

    constexpr bool kScores = C::kDtype == QIMG_INT8;             // K's scale is the scores'
    constexpr bool kWeights = kScores && T::kBf;                 // V's scale is P's (bf16 has fp32's range)

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
        const bool hidden = key0 + SK > kfull || x.bad != 0;  // some row does not see some key
        if (hidden) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = key0 + 16 * h + 4 * g + j;
#pragma unroll
                    for (int r = 0; r < NR; ++r)
                        if (key >= kmax[r] || (x.bad >> h & 1)) s[r][h][j] = kNegInf;
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
            if constexpr (kWeights) {
                // the same roundings, as a power of two changes none
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    pk[j] = T::pack(p[2 * j] * exp_scale(x.ve[j / 2] >> 16 * (j & 1) & 0xffu),
                                    p[2 * j + 1] * exp_scale(x.ve[j / 2] >> (16 * (j & 1) + 8) & 0xffu));
                pf[r] = as_frag<T>(pk[0], pk[1], pk[2], pk[3]);
            }
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
                if constexpr (kWeights) w[j] = decode_int8_pairs<true>(raw);
                else w[j] = decode_pairs<C, T::kBf>(raw, exp_scale(x.ve[j / 4] >> 8 * (j & 3) & 0xffu));
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

template <class T, class C, int D, int NR>
__global__ __launch_bounds__(SW * 64, NR == 1 ? 3 : 2) void attn_cache_few_kernel(AttnCacheArgs a, int lo, int hi) {
    __shared__ __attribute__((aligned(16))) float lds[SW * 16 * (kPitch<D> + 2)];
    const Sequence first = load_sequence(a, lo + (threadIdx.x & 63), hi);
    const int per = range_tiles(a, first, lo, hi, 16 * NR);
    for (int item = blockIdx.x;; item += gridDim.x) {
        const RowTile t = find_tile(a, first, lo, hi, item / a.c.hk, 16 * NR, per);
        if (!t.found) return;
        few_item<T, C, D, NR>(a, t, item % a.c.hk, lds);
    }
}

// ---- many rows: 128 of them, four waves over one ring -----------------------
// The work of a wave and its phases are attention_varlen.hip's (Many, its 64-key tiles
// and the ring of two slots that hold V of tile p - 1 beside K of tile p); what differs is
// how a tile gets there: codes come to registers, a step ahead of their use, and go to
// LDS as 16-bit values, once for the four waves. Per step and thread that is 64 codes,
// between the exponentials of the softmax. Page numbers are loaded a further step ahead.
// Tiles too few for the CUs have their keys cut into ranges, a workgroup each.
constexpr int kManyGrid = 512;  // workgroups that run at once, two a CU

// A tile's key ranges of `per` 64-key tiles each, of `n` in all.
struct TileRanges {
    int n, per, count;
};
__device__ __forceinline__ TileRanges many_ranges(const AttnCacheArgs& a, const RowTile& t, int row0) {
    const int rows = t.lq * a.group;
    TileRanges r;
    r.n = (visible(a, t, (min(row0 + MR, rows) - 1) / a.group) + MK - 1) / MK;
    const int most = max(t.b < a.batch ? a.own_splits : a.prefix_splits, 1);
    r.per = most == 1 ? max(r.n, 1) : max((r.n + most - 1) / most, 4);
    r.count = max((r.n + r.per - 1) / r.per, 1);
    return r;
}

// V tiles in LDS have their 16-byte chunks also swapped in pairs by bit 2 of the row: the
// stores of 16 lanes then take 256 bytes of banks (they hold chunks of one parity of
// two rows, or four, that differ in that bit; with swz_v alone every second one waits).
template <int D>
__device__ __forceinline__ int swz_vc(int row, int c) {
    return swz_v<D>(row, c) ^ ((row >> 2) & 1);
}
// (v_lane_off with these chunks)
template <int D>
__device__ __forceinline__ int vc_lane_off(int dt) {
    const int lane = threadIdx.x & 63, i = lane & 15;
    const int row = 4 * (lane >> 5) + (i >> 2);
    const int chunk = 4 * dt + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    return row * (2 * D) + swz_vc<D>(row, chunk) * 16 + (i & 1) * 8;
}

// The codes of K or V tiles on their way to LDS: a thread holds 16 codes of N rows. A
// wave's rows of one load lie in one 16-key group, so its page and the address of the
// load are uniform.
template <class T, class C, int D, bool VTILE>
struct CodeStream {
    static constexpr int N = D / 64, TPR = D / 16, RPW = 64 / TPR;  // loads of a thread a tile; threads a row, rows a load
    int row, off;  // a lane's row and offset behind the load's first row
    int dst[2];    // and its two chunks' places in LDS
    u32x4 raw[N];
    uint32_t e[N];
    __device__ __forceinline__ void init(int wave) {
        const int lane = threadIdx.x & 63, q = lane / TPR, c = lane % TPR;
        if constexpr (!VTILE) row = q;
        else if constexpr (D == 128) row = (q & 1) * 4 + (q >> 1);                             // rows r, r + 4 side by side
        else row = (q & 1) + (q >> 1 & 1) * 4 + (q >> 2 & 1) * 2 + (q >> 3) * 8;  // r, r + 1, r + 4, r + 5
        off = row * D + 16 * c;
        const int at = RPW * wave + row;
#pragma unroll
        for (int j = 0; j < 2; ++j) dst[j] = at * (2 * D) + (VTILE ? swz_vc<D>(at, 2 * c + j) : swz_k<D>(at, 2 * c + j)) * 16;
    }
    // load i of the tile: the wave's rows begin at these addresses
    __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* exps, int i) {
        raw[i] = Buffer(codes, RPW * D).load<u32x4>(off);
        e[i] = Buffer(exps, RPW).load<uint8_t>(row);
    }
    // codes 8 j .. 8 j + 7 of load i as 16-bit values to their place in the tile. `left`: rows of
    // the load that hold keys in use; V of the others is zeros, whatever lies there.
    __device__ __forceinline__ void store(int i, int j, uint8_t* tile, int left) {
        float scale = exp_scale(e[i]);
        uint32_t x = raw[i][2 * j], y = raw[i][2 * j + 1];
        if (VTILE && left < RPW) {
            const bool none = row >= left;
            scale = none ? 0.0f : scale;
            x = none ? 0u : x;
            y = none ? 0u : y;
        }
        const uint2 p = decode_pairs<C, T::kBf>(x, scale), q = decode_pairs<C, T::kBf>(y, scale);
        *reinterpret_cast<u32x4*>(tile + dst[j] + 64 / N * i * (2 * D)) = (u32x4){p.x, p.y, q.x, q.y};
    }
};

template <class T, class C, int D>
__global__ __launch_bounds__(MW * 64, 2) void attn_cache_many_kernel(AttnCacheArgs a, int lo, int hi, int tiles, int splits) {
    using W = Many<T, D>;
    using KStream = CodeStream<T, C, D, false>;
    using VStream = CodeStream<T, C, D, true>;
    constexpr int PAIR = 2 * W::TB, N = KStream::N, RPW = KStream::RPW;
    static_assert(W::PER == 4 * N, "stores of a thread a pair");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[MSLOT * PAIR];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, half = lane >> 5;
    // The row tiles that share a range of a head's keys side by side on one XCD.
    const int logical = xcd_remap(blockIdx.x, gridDim.x);
    const int split = logical / tiles % splits, hk = logical / (tiles * splits);
    const RowTile t = find_tile(a, load_sequence(a, lo + lane, hi), lo, hi, logical % tiles, MR, 0);
    if (!t.found) return;
    const TileRanges ranges = many_ranges(a, t, t.row0);
    if (split >= ranges.count) return;
    const int tile0 = split * ranges.per, n = min(ranges.per, ranges.n - tile0);

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
        // Where the keys of 16 tiles lie: lane l holds the first cache row of 16-key group l behind
        // tile `base`, `bad` a bit for each group whose page is outside the cache (row 0 stands for
        // it). kTurn tiles further on those of the 16 tiles from there take their place, whose
        // page numbers are loaded by then: a step reaches three tiles ahead. (Rows worked out anew
        // from the page number for every load took a fifth of the loop: the wave issues nothing
        // else meanwhile.)
        constexpr int kTurn = 12;
        const int* table = own ? a.table + static_cast<int64_t>(t.b) * a.max_blocks : a.prefix_table;
        const int last = ((t.lk + (1 << a.c.page_shift) - 1) >> a.c.page_shift) - 1;  // page of the last key in use
        const auto pages_from = [&](int tile) { return table[min((4 * tile + lane) >> (a.c.page_shift - 4), last)]; };
        int ids_next = pages_from(tile0), base = tile0, row_lo = 0, row_hi = 0;
        uint64_t bad = 0;
        const auto turn = [&](int tile) {
            const bool in = ids_next >= 0 && ids_next < a.c.n_pages;
            const int64_t first = ((static_cast<int64_t>(in ? ids_next : 0) * a.c.hk + hk) << a.c.page_shift) +
                                  (16 * (4 * tile + lane) & ((1 << a.c.page_shift) - 1));
            row_lo = static_cast<int>(first);
            row_hi = static_cast<int>(first >> 32);
            bad = __ballot(!in);
            base = tile;
            ids_next = pages_from(tile + kTurn);
        };
        turn(tile0);
        KStream ks;
        VStream vs;
        ks.init(wave);
        vs.init(wave);
        // the wave's rows of load i: group RPW * wave / 16 of four (D 64) or of two of them
        const int sub = RPW * wave / 16, in_group = RPW * wave % 16;
        const auto row_of = [&](int i, int tile) __attribute__((always_inline)) {
            const int g = 4 * (tile - base) + 4 / N * i + sub;
            return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(row_hi, g))) << 32 |
                                        static_cast<uint32_t>(__builtin_amdgcn_readlane(row_lo, g)));
        };
        const uint8_t *kc = a.c.k + in_group * D, *kx = a.c.ke + in_group, *vc = a.c.v + in_group * D, *vx = a.c.ve + in_group;
        const auto load_k = [&](int i, int tile) __attribute__((always_inline)) {
            const int64_t at = row_of(i, tile);
            ks.load(kc + at * D, kx + at, i);
        };
        const auto load_v = [&](int i, int tile) __attribute__((always_inline)) {
            const int64_t at = row_of(i, tile);
            vs.load(vc + at * D, vx + at, i);
        };
        // rows of load i that hold keys in use: none in a page outside the cache
        const auto left_of = [&](int i, int tile) __attribute__((always_inline)) {
            return bad >> (4 * (tile - base) + 4 / N * i + sub) & 1 ? 0 : t.lk - (tile * MK + 64 / N * i + RPW * wave);
        };
#pragma unroll
        for (int i = 0; i < N; ++i) load_k(i, tile0);
        {
            const uint16_t* qp = a.q + (static_cast<int64_t>(t.q0) + token) * a.q_t + head * a.q_h + 8 * half;
#pragma unroll
            for (int i = 0; i < W::KS; ++i) w.qf[i] = *reinterpret_cast<const typename T::frag*>(qp + 16 * i);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) load_v(i, tile0);
#pragma unroll
        for (int d = 0; d < W::DT; ++d) w.voff[d] = vc_lane_off<D>(d);
#pragma unroll
        for (int c = 0; c < W::KS; ++c) w.koff[c] = l32 * (2 * D) + swz_k<D>(l32, 2 * c + half) * 16;
#pragma unroll
        for (int r = 0; r < 16 * W::KB; ++r) w.s[r >> 4][r & 15] = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) ks.store(i, j, lds + W::TB, 0);
#pragma unroll
        for (int i = 0; i < N; ++i) load_k(i, tile0 + 1);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) vs.store(i, j, lds + PAIR, left_of(i, tile0));
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) ks.store(i, j, lds + PAIR + W::TB, 0);
#pragma unroll
        for (int i = 0; i < N; ++i) {  // pair 2: V of tile 1, K of tile 2
            load_v(i, tile0 + 1);
            load_k(i, tile0 + 2);
        }
        wait_lgkmcnt0();
        phase_barrier();
        w.template first_scores<W::NPV>(lds);
        for (int p = 0; p < n; ++p) {
            const uint8_t* src = lds + ((p + 1) % MSLOT) * PAIR;
            uint8_t* dst = lds + (p % MSLOT) * PAIR;
            const int tile = tile0 + p;
            if (tile == base + kTurn) turn(tile);
            wait_lgkmcnt0();  // pair p + 1 is in LDS, this wave's part of it
            phase_barrier();
            w.template read_group<0>(src, w.buf[0]);
            __builtin_amdgcn_sched_barrier(0);
            if (const int odd = static_cast<int>(bad >> 4 * (tile - base)) & 15) {  // keys of a page outside the cache are not seen
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    if (odd >> g & 1)
#pragma unroll
                        for (int r = 0; r < 8; ++r) w.s[g / 2][8 * (g % 2) + r] = kNegInf;
            }
            w.softmax(tile * MK, kfull, kmax, a.scale_log2, [&](int i) {
                // Two stores of each load, then the next one into its registers (behind the last
                // tile too: with loads under a condition the compiler waits for all of them).
                const int l = i % (2 * N) / 2, j = i % 2;
                if (i < 2 * N) {
                    vs.store(l, j, dst, left_of(l, tile + 1));
                    if (j == 1) load_v(l, tile + 2);
                } else {
                    ks.store(l, j, dst + W::TB, 0);
                    if (j == 1) load_k(l, tile + 3);
                }
            });
#pragma unroll
            for (int i = 0; i < 8 * W::KB; ++i) asm volatile("" : "+v"(w.pk[i]));  // P is made in this phase
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            bool bad = false;
            w.template m_groups<0, false>(src, bad);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
        }
    }
    const float tot = half_sum(w.sum[0]);
    constexpr int CHUNKS = D / 8;
    if (ranges.count > 1 || a.prefix_splits > 0) {
        if (!valid) return;
        const int64_t at = ((static_cast<int64_t>(t.q0) + token) * a.hq + head) * (a.own_splits + a.prefix_splits) +
                           (own ? 0 : a.own_splits) + split;
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

// Partial results of a row, added in order: 16 threads a row, tiles of 16 rows of one
// sequence and kv head. Eight parts' loads go out together.
template <class T, int D>
__device__ __forceinline__ void join_item(const AttnCacheArgs& a, const AttnCachePlan& plan, const RowTile& t, int hk, int per,
                                          bool together) {
    constexpr int E = D / 16, U = 8;
    typedef float v2f __attribute__((ext_vector_type(2)));
    const int own = plan.own_rows == MR ? many_ranges(a, t, t.row0 / MR * MR).count : key_ranges(t.lk, per);
    int shared = 0;
    if (a.prefix_splits > 0) {
        const Sequence p = load_sequence(a, a.batch, a.batch + 1);
        if (plan.prefix_rows == MR) {
            RowTile pt = t;
            pt.b = a.batch, pt.q0 = p.q0, pt.lq = p.lq, pt.lk = p.lk;
            shared = many_ranges(a, pt, 0).count;
        } else {
            shared = key_ranges(p.lk, together ? per : range_tiles(a, load_sequence(a, a.batch + (threadIdx.x & 63), a.batch + 1), a.batch,
                                                                    a.batch + 1, plan.prefix_rows));
        }
    }
    const int row = t.row0 + (threadIdx.x >> 4), c0 = (threadIdx.x & 15) * E;
    if (own + shared == 1 || row >= t.lq * a.group) return;
    const int64_t token = static_cast<int64_t>(t.q0) + row / a.group;
    const int head = hk * a.group + row % a.group;
    const int64_t at = (token * a.hq + head) * (a.own_splits + a.prefix_splits);
    const int n = own + shared;
    float mm = kNegInf, tot = 0.0f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    for (int s0 = 0; s0 < n; s0 += U) {
        v2f ml[U];
        v4f v[U][E / 4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = min(s0 + u, n - 1);
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
            if (s0 + u >= n) continue;
            // no finite score: O is zero there, the sum zero or NaN
            const float f = ml[u][0] == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(ml[u][0] - mm);
            tot += f * ml[u][1];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += f * v[u][e / 4][e % 4];
        }
    }
    store_row<T, E>(a.out + token * a.o_t + head * a.o_h + c0, acc, tot, tot == 0.0f);
}

template <class T, int D>
__global__ __launch_bounds__(256) void attn_cache_join_kernel(AttnCacheArgs a, AttnCachePlan plan) {
    const int lane = threadIdx.x & 63;
    const bool together = plan.prefix_splits > 0 && plan.prefix_rows == plan.own_rows && plan.own_rows != MR;
    const int hi = a.batch + (together ? 1 : 0);
    const Sequence first = load_sequence(a, lane, hi);
    const int per = plan.own_rows == MR ? 0 : range_tiles(a, first, 0, hi, plan.own_rows);
    for (int item = blockIdx.x;; item += gridDim.x) {
        const int hk = item % a.c.hk;
        const RowTile t = find_tile(a, first, 0, a.batch, item / a.c.hk, 16, 0);
        if (!t.found) return;
        join_item<T, D>(a, plan, t, hk, per, together);
    }
}

// upper bound on the tiles of `rows` rows that the sequences have
int64_t tile_bound(int total_q, int batch, int group, int rows) {
    const int64_t seqs = batch < total_q ? batch : total_q;
    return (static_cast<int64_t>(total_q) * group + seqs * (rows - 1)) / rows;
}

}  // namespace

constexpr int kMostSplits = 32;
constexpr int kMostBlocks = 1 << 22;  // of a launch (a grid has less than 2^32 threads)

// Key ranges of each of `tiles` tiles of 128 rows over `steps` key tiles, so that time is
// least: rounds of workgroups times a range's steps, each with the start of a range, and
// what the ranges' float results cost. Lengths are on the device: the table's room stands
// for them here, which decides the time, not the result.
static int many_splits(int64_t tiles, int64_t steps) {
    int best = 1;
    double least = 0.0;
    for (int s = 1; s <= kMostSplits && (s == 1 || 4 * s <= steps); ++s) {
        const int64_t items = tiles * s;
        const double pace = items <= kManyGrid / 2 ? 1.5 : 1.7, rounds = static_cast<double>((items + kManyGrid - 1) / kManyGrid);
        const double t = rounds * pace * (static_cast<double>(steps) / s + 3.0) + (s > 1 ? 4.0 + 0.026 * static_cast<double>(items) : 0.0);
        if (s == 1 || t < least) best = s, least = t;
    }
    return best;
}

AttnCachePlan attn_cache_plan(int total_q, int batch, int hq, int hk, int D, int64_t own_keys, int64_t prefix_keys) {
    AttnCachePlan p{};
    if (total_q <= 0 || batch <= 0) return p;
    const int group = hq / hk;
    // rows of a tile, by the average number of a sequence
    const auto tile_rows = [&](int64_t rows, int seqs) {
        return rows <= 16 ? 16 : rows <= 64 || tile_bound(total_q, seqs, group, MR) * hk >= kMostBlocks ? 32 : MR;
    };
    p.own_rows = tile_rows((static_cast<int64_t>(total_q) * group + batch - 1) / batch, batch);
    p.prefix_rows = tile_rows(static_cast<int64_t>(total_q) * group, 1);
    // most ranges: at least eight key tiles each, and 2^13 row tiles times ranges; of 128
    // rows as many as run at once
    const auto splits = [&](int64_t keys, int rows, int seqs) {
        const int64_t tiles = std::max<int64_t>(tile_bound(total_q, seqs, group, rows) * hk, 1);
        if (rows == MR) return many_splits(tiles, (keys + MK - 1) / MK);
        const int64_t most = std::min<int64_t>((keys + 8 * SK - 1) / (8 * SK), 8192 / tiles);
        return static_cast<int>(std::max<int64_t>(std::min<int64_t>(most, kMostSplits), 1));
    };
    p.own_splits = splits(own_keys, p.own_rows, batch);
    p.prefix_splits = prefix_keys > 0 ? splits(prefix_keys, p.prefix_rows, 1) : 0;
    if (p.own_splits > 1 || p.prefix_splits > 0)
        p.part_rows = static_cast<int64_t>(total_q) * hq * (p.own_splits + p.prefix_splits);
    return p;
}

// The sequences [lo, hi) in tiles of `rows` rows.
template <class T, class C, int D>
static hipError_t launch_part(const AttnCacheArgs& a, int rows, int lo, int hi, hipStream_t stream) {
    const int64_t own = lo < a.batch ? tile_bound(a.total_q, a.batch, a.group, rows) : 0;
    const int64_t shared = hi > a.batch ? tile_bound(a.total_q, 1, a.group, rows) : 0;
    if (rows == MR) {
        const int splits = lo < a.batch ? a.own_splits : a.prefix_splits;
        const int tiles = static_cast<int>(own + shared);
        hipLaunchKernelGGL((attn_cache_many_kernel<T, C, D>), dim3(static_cast<unsigned>(tiles) * splits * a.c.hk),
                           dim3(MW * 64), 0, stream, a, lo, hi, tiles, splits);
        return hipGetLastError();
    }
    const int64_t items = (own * a.own_splits + shared * a.prefix_splits) * a.c.hk;
    const dim3 grid(static_cast<unsigned>(items < kFewGrid ? items : kFewGrid));
    if (rows == 16)
        hipLaunchKernelGGL((attn_cache_few_kernel<T, C, D, 1>), grid, dim3(SW * 64), 0, stream, a, lo, hi);
    else
        hipLaunchKernelGGL((attn_cache_few_kernel<T, C, D, 2>), grid, dim3(SW * 64), 0, stream, a, lo, hi);
    return hipGetLastError();
}

template <class T, class C, int D>
static hipError_t launch_attn(const AttnCacheArgs& a, const AttnCachePlan& plan, hipStream_t stream) {
    const bool prefix = plan.prefix_splits > 0;
    const bool together = prefix && plan.prefix_rows == plan.own_rows && plan.own_rows != MR;
    hipError_t e = launch_part<T, C, D>(a, plan.own_rows, 0, a.batch + (together ? 1 : 0), stream);
    if (e == hipSuccess && prefix && !together)
        e = launch_part<T, C, D>(a, plan.prefix_rows, a.batch, a.batch + 1, stream);
    if (e != hipSuccess || plan.part_rows == 0) return e;
    const int64_t tiles = std::min<int64_t>(tile_bound(a.total_q, a.batch, a.group, 16) * a.c.hk, kMostBlocks);
    hipLaunchKernelGGL((attn_cache_join_kernel<T, D>), dim3(static_cast<unsigned>(tiles)), dim3(256), 0, stream, a, plan);
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
