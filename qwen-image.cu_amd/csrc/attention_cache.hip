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

#include "cache_codes.h"
#include "qimg_internal.h"

namespace qimg {

namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr float kNegInf = -__builtin_inff();
constexpr float kSlack = 8.0f;

// element type: fragment vector, MFMA, P pair packing
struct Bf16 {
    using frag = v8bf;
    static constexpr bool kBf = true;
    static constexpr float kPBias = -38.0f;
    static constexpr uint32_t kOnes = 0x3f803f80u;
    __device__ static __forceinline__ v4f mma(frag a, frag b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    __device__ static __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
};
struct Fp16 {
    using frag = v8h;
    static constexpr bool kBf = false;
    static constexpr float kPBias = 7.0f;
    static constexpr uint32_t kOnes = 0x3c003c00u;
    __device__ static __forceinline__ v4f mma(frag a, frag b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    __device__ static __forceinline__ uint32_t pack(float a, float b) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        typedef float f2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, h2));
    }
};

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

// inclusive sum over the wave's lanes
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
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
            t.row0 = tile * rows;
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

// A wave's 32-key tile as it lies in the cache
template <int D>
struct RawTile {
    u32x4 k[2][D / 64];                                       // key lane % 16 of each 16: 16 codes a chunk
    std::conditional_t<D == 128, uint2, uint32_t> v[8];       // keys 4 g + i, 16 + 4 g + i: D / 16 channels
    uint32_t ke[2], ve[2];                                    // E of k's key, of v's four keys each
    int bad;                                                  // bits: a 16-key group's page is not in the cache
};

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

    // Pages of the wave's tiles, 32 at a time: lane l holds that of 16-key group l % 2 of
    // tile l / 2.
    int ids = 0;
    const auto load = [&](RawTile<D>& x, int i) __attribute__((always_inline)) {
        if ((i & 31) == 0) {
            const int group16 = 2 * (tile0 + wave + SW * (i + (lane >> 1))) + (lane & 1);
            ids = table[min(group16 >> (a.c.page_shift - 4), blocks - 1)];
        }
        x.bad = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int page = __builtin_amdgcn_readlane(ids, 2 * (i & 31) + h);
            const bool in = page >= 0 && page < a.c.n_pages;
            x.bad |= in ? 0 : 1 << h;
            page = in ? page : 0;
            const int group16 = 2 * (tile0 + wave + SW * i) + h;
            const int64_t row = ((static_cast<int64_t>(page) * a.c.hk + hk) << a.c.page_shift) +
                                16 * (group16 & ((1 << (a.c.page_shift - 4)) - 1));
            const uint8_t* kp = a.c.k + row * D + c * D + 16 * g;
            const uint8_t* vp = a.c.v + row * D + 4 * g * D + CH * c;
#pragma unroll
            for (int s = 0; s < D / 64; ++s) x.k[h][s] = *reinterpret_cast<const u32x4*>(kp + 64 * s);
            x.ke[h] = a.c.ke[row + c];
            x.ve[h] = *reinterpret_cast<const uint32_t*>(a.c.ve + row + 4 * g);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x.v[4 * h + j] = *reinterpret_cast<const std::remove_reference_t<decltype(x.v[0])>*>(vp + j * D);
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

    const auto step = [&](RawTile<D>& x, int i) __attribute__((always_inline)) {
        const int key0 = (tile0 + wave + SW * i) * SK;
        v4f s[NR][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float scale = exp_scale(x.ke[h]);
#pragma unroll
            for (int r = 0; r < NR; ++r) s[r][h] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int d = 0; d < D / 64; ++d) {
                uint2 w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = decode_pairs<C, T::kBf>(x.k[h][d][j], scale);
                const frag k0 = as_frag<T>(w[0].x, w[0].y, w[1].x, w[1].y);
                const frag k1 = as_frag<T>(w[2].x, w[2].y, w[3].x, w[3].y);
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    s[r][h] = T::mma(k0, qf[r][2 * d], s[r][h]);
                    s[r][h] = T::mma(k1, qf[r][2 * d + 1], s[r][h]);
                }
            }
        }
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
            uint32_t pk[4];
#pragma unroll
            for (int j = 0; j < 8; j += 2)
                pk[j / 2] = T::pack(__builtin_amdgcn_exp2f(__builtin_fmaf(s[r][j >> 2][j & 3], a.scale_log2, neg)),
                                    __builtin_amdgcn_exp2f(__builtin_fmaf(s[r][j >> 2][(j & 3) + 1], a.scale_log2, neg)));
            pf[r] = as_frag<T>(pk[0], pk[1], pk[2], pk[3]);
            sum[r] = T::mma(ones, pf[r], sum[r]);
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
                for (int r = 0; r < NR; ++r) o[r][4 * d4 + e] = T::mma(vf, pf[r], o[r][4 * d4 + e]);
            }
        }
    };

    if (n > 0) {
        RawTile<D> x, y;
        load(x, 0);
        for (int i = 0; i < n; i += 2) {
            if (i + 1 < n) load(y, i + 1);
            step(x, i);
            if (i + 1 < n) {
                if (i + 2 < n) load(x, i + 2);
                step(y, i + 1);
            }
        }
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
__global__ __launch_bounds__(SW * 64, NR == 4 ? 1 : 2) void attn_cache_few_kernel(AttnCacheArgs a, int lo, int hi) {
    __shared__ __attribute__((aligned(16))) float lds[SW * 16 * (kPitch<D> + 2)];
    const Sequence first = load_sequence(a, lo + (threadIdx.x & 63), hi);
    const int per = range_tiles(a, first, lo, hi, 16 * NR);
    for (int item = blockIdx.x;; item += gridDim.x) {
        const RowTile t = find_tile(a, first, lo, hi, item / a.c.hk, 16 * NR, per);
        if (!t.found) return;
        few_item<T, C, D, NR>(a, t, item % a.c.hk, lds);
    }
}

// Partial results of a row, added in order: 16 threads a row, tiles of 16 rows of one
// sequence and kv head. Eight parts' loads go out together.
template <class T, int D>
__global__ __launch_bounds__(256) void attn_cache_join_kernel(AttnCacheArgs a, AttnCachePlan plan) {
    constexpr int E = D / 16, U = 8;
    typedef float v2f __attribute__((ext_vector_type(2)));
    const int lane = threadIdx.x & 63;
    const bool together = plan.prefix_splits > 0 && plan.prefix_rows == plan.own_rows;
    const int hi = a.batch + (together ? 1 : 0);
    const Sequence first = load_sequence(a, lane, hi);
    const int per = range_tiles(a, first, 0, hi, plan.own_rows);
    const int hk = blockIdx.x % a.c.hk;
    const RowTile t = find_tile(a, first, 0, a.batch, blockIdx.x / a.c.hk, 16, 0);
    if (!t.found) return;
    const int own = key_ranges(t.lk, per);
    int shared = 0;
    if (a.prefix_splits > 0) {
        const Sequence p = load_sequence(a, a.batch, a.batch + 1);
        shared = key_ranges(p.lk, together ? per : range_tiles(a, load_sequence(a, a.batch + lane, a.batch + 1), a.batch,
                                                                a.batch + 1, plan.prefix_rows));
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

// upper bound on the tiles of `rows` rows that the sequences have
int64_t tile_bound(int total_q, int batch, int group, int rows) {
    const int64_t seqs = batch < total_q ? batch : total_q;
    return (static_cast<int64_t>(total_q) * group + seqs * (rows - 1)) / rows;
}

}  // namespace

constexpr int kMostSplits = 32;

AttnCachePlan attn_cache_plan(int total_q, int batch, int hq, int hk, int D, int64_t own_keys, int64_t prefix_keys) {
    AttnCachePlan p{};
    if (total_q <= 0 || batch <= 0) return p;
    const int group = hq / hk;
    const auto few_rows = [](int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; };
    p.own_rows = few_rows((static_cast<int64_t>(total_q) * group + batch - 1) / batch);
    p.prefix_rows = few_rows(static_cast<int64_t>(total_q) * group);
    // most ranges: at least eight key tiles each, and 2^13 row tiles times ranges
    const auto splits = [&](int64_t keys, int64_t tiles) {
        const int64_t most = std::min<int64_t>((keys + 8 * SK - 1) / (8 * SK), kMostSplits);
        return static_cast<int>(std::max<int64_t>(std::min(most, 8192 / std::max<int64_t>(tiles, 1)), 1));
    };
    p.own_splits = splits(own_keys, tile_bound(total_q, batch, group, p.own_rows) * hk);
    p.prefix_splits = prefix_keys > 0 ? splits(prefix_keys, tile_bound(total_q, 1, group, p.prefix_rows) * hk) : 0;
    if (p.own_splits > 1 || p.prefix_splits > 0)
        p.part_rows = static_cast<int64_t>(total_q) * hq * (p.own_splits + p.prefix_splits);
    return p;
}

template <class T, class C, int D>
static hipError_t launch_few(const AttnCacheArgs& a, int rows, int lo, int hi, hipStream_t stream) {
    const int64_t own = lo < a.batch ? tile_bound(a.total_q, a.batch, a.group, rows) * a.own_splits : 0;
    const int64_t shared = hi > a.batch ? tile_bound(a.total_q, 1, a.group, rows) * a.prefix_splits : 0;
    const int64_t items = (own + shared) * a.c.hk;
    const dim3 grid(static_cast<unsigned>(items < kFewGrid ? items : kFewGrid));
    if (rows == 16)
        hipLaunchKernelGGL((attn_cache_few_kernel<T, C, D, 1>), grid, dim3(SW * 64), 0, stream, a, lo, hi);
    else if (rows == 32)
        hipLaunchKernelGGL((attn_cache_few_kernel<T, C, D, 2>), grid, dim3(SW * 64), 0, stream, a, lo, hi);
    else
        hipLaunchKernelGGL((attn_cache_few_kernel<T, C, D, 4>), grid, dim3(SW * 64), 0, stream, a, lo, hi);
    return hipGetLastError();
}

template <class T, class C, int D>
static hipError_t launch_attn(const AttnCacheArgs& a, const AttnCachePlan& plan, hipStream_t stream) {
    const bool prefix = plan.prefix_splits > 0, together = prefix && plan.prefix_rows == plan.own_rows;
    hipError_t e = launch_few<T, C, D>(a, plan.own_rows, 0, a.batch + (together ? 1 : 0), stream);
    if (e == hipSuccess && prefix && !together)
        e = launch_few<T, C, D>(a, plan.prefix_rows, a.batch, a.batch + 1, stream);
    if (e != hipSuccess || plan.part_rows == 0) return e;
    const int64_t tiles = tile_bound(a.total_q, a.batch, a.group, 16) * a.c.hk;
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
