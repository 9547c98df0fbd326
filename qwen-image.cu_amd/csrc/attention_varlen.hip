// attention_varlen.hip — unquantized attention over packed sequences:
//   s_ij = sm_scale * q_i . k_j             (j visible to i)
//   o_i  = sum_j e^(s_ij - m_i) v_j / sum_j e^(s_ij - m_i)
// for sequences of different lengths that lie one behind the other, grouped
// heads (Hq a multiple of Hk, query head h reads kv head h / (Hq / Hk)), bf16
// or fp16. Key j of a sequence with lq queries and lk keys is visible to
// query i when j < lk and, if causal, j <= i + lk - lq (the last query sees
// the last key). A query that sees no key gives zeros.
//
// Rows: a tile's rows are (token, head of the group) pairs of one sequence
// and one kv head, row = token * group + head, so the heads of a group share
// the K and V they read (one token of 7 heads is 7 rows of a tile, not 7
// tiles), and a causal tile spans few tokens.
//
// Arithmetic: v_mfma_f32_32x32x16 on both products, fp32 accumulation, base-2
// online softmax with the running maximum and sum in fp32. Scores are computed
// transposed (S^T = K Q^T), so a lane holds one query row's scores and the P
// registers are the second product's operand as they are: with O^T = V^T P^T
// element e of lane half h stands for key 16 t + 8 (e / 4) + 4 h + e % 4 of a
// 16-key group t, and V^T comes from row-major V in LDS through
// ds_read_b64_tr_b16, whose four values are 4 consecutive keys of one channel.
// P is rounded to the inputs' type for the second product, as the matrix unit takes
// no others at its rate (in two parts they would be half as many products again): with u half
// a step of the type (2^-8 in bf16, 2^-11 in fp16) an error of at most
// sum_j u p_j |v_j - o|, since the row sum adds the rounded values (a constant V is
// returned exactly); against 64 bits 1.15 to 1.4 times what rounding the result alone
// leaves. The maximum moves, and O and the sum are rescaled, only when a tile exceeds
// it by more than kSlack (log2 units): P then reaches 2^kSlack, which changes no
// relative rounding. fp16 P carries a further factor 2^kBias16 (at most 2^15 in all):
// weights below 2^-21 of the maximum are then subnormal, off by up to 2^-32 of it each
// (the bound above grows by sum_j 2^-32 |v_j - o|), and vanish below 2^-32. bf16 V
// reaches as far as the fp32 sums of P V: with a factor 2^kBiasBf fewer than 2^30 keys
// of the largest V, each weighing 2^kSlack, stay below 2^128 (without it 4 keys of 1e38
// gave infinity). For that P vanishes below 2^-88 of the maximum, and V whose average is
// below 2^-79 loses digits; the fp32 exponent's own rounding is 2^-19 of P, a thousandth
// of what bf16 leaves.
//
// K and V tiles go to LDS by buffer loads whose descriptor ends at the
// sequence's last key: rows behind it arrive as zeros, so nothing that lies
// there (another sequence, an unused part of a cache) reaches the result, NaN
// included. Every tile has a descriptor of its own (64-bit base), so offsets
// inside one stay small however long the cache is.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "qimg_device.h"
#include "qimg_internal.h"

namespace qimg {

namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

constexpr float kNegInf = -__builtin_inff();
constexpr float kSlack = 8.0f;   // lazy-rescale threshold of the running maximum (log2 units)
constexpr float kBias16 = 7.0f;  // log2 of the factor on fp16 P
constexpr float kBiasBf = -38.0f;  // and on bf16 P
constexpr int kRsrcWord3 = 0x00020000;  // raw unswizzled buffer (gfx9 family)

// element type: fragment vector, MFMA, P pair packing and its row sum, and
// the mask of a value's exponent bits (all ones: infinity or NaN). The row sum is
// a matrix product as well: with A = 1 an element of 4x4x4's column j is the sum of
// the four values that lane j of its group of four holds. (16 dot products of pairs a
// tile, v_dot2, take 107 cycles alone, but 620 beside another wave's MFMAs, which they
// wait for; eight of these 4x4x4 take 88. Together 1-3% of the kernel's time.)
struct Bf16 {
    using frag = v8bf;
    static constexpr float kPBias = kBiasBf;
    static constexpr uint32_t kExp = 0x7f80u, kMant = 0x007fu;
    __device__ static __forceinline__ v16f mma(frag a, frag b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    __device__ static __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
    __device__ static __forceinline__ v4f add4(uint32_t p0, uint32_t p1, v4f s) {
        constexpr short one = 0x3f80;
        return __builtin_amdgcn_mfma_f32_4x4x4bf16_1k((v4s){one, one, one, one},
                                                      __builtin_bit_cast(v4s, static_cast<uint64_t>(p1) << 32 | p0), s,
                                                      0, 0, 0);
    }
};
struct Fp16 {
    using frag = v8h;
    static constexpr float kPBias = kBias16;
    static constexpr uint32_t kExp = 0x7c00u, kMant = 0x03ffu;
    __device__ static __forceinline__ v16f mma(frag a, frag b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    __device__ static __forceinline__ uint32_t pack(float a, float b) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        typedef float f2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, h2));
    }
    __device__ static __forceinline__ v4f add4(uint32_t p0, uint32_t p1, v4f s) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        constexpr _Float16 one = 1;
        return __builtin_amdgcn_mfma_f32_4x4x4f16((h4){one, one, one, one},
                                                  __builtin_bit_cast(h4, static_cast<uint64_t>(p1) << 32 | p0), s, 0, 0,
                                                  0);
    }
};

// max of the two lane halves' values (lanes l and l ^ 32)
__device__ __forceinline__ float half_max(float v) {
    const unsigned u = __float_as_uint(v);
    const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const unsigned u = __float_as_uint(v);
    const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}

// LDS tiles of ROWS keys x D channels, rows unpadded, 16-byte chunks swizzled
// by row: a K fragment read takes one logical chunk of 16 consecutive rows
// (ds_read_b128, 16 lanes a cycle over 256 bytes of banks), so those need 16
// different bank groups; a transposing V read takes 64 bytes of each of 4
// consecutive rows per half wave, which need 4 different quarters of the
// banks.
template <int D>
__device__ __forceinline__ int swz_k(int row, int c) {
    return D == 128 ? c ^ (row & 15) : c ^ ((row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int swz_v(int row, int c) {
    return D == 128 ? c ^ (4 * (row & 3)) : c ^ (4 * ((row >> 1) & 1));
}

// One sequence's tile of rows.
struct RowTile {
    int q0, lq, k0, lk;  // first query and key row, their numbers
    int row0;            // first (token, head) row of the tile in the sequence
    int split, splits;   // key range of it, and into how many the sequence's keys are cut
    bool found;
};

// A lane's sequence b: first query and key row, numbers of both. Offsets
// outside [0, total] or falling ones are clamped, so no tile reaches past the
// tensors.
struct Sequence {
    int q0, lq, k0, lk;
};
__device__ __forceinline__ Sequence load_sequence(const AttnVarlenArgs& a, int b) {
    Sequence s = {0, 0, 0, 0};
    if (b < a.batch) {
        s.q0 = min(max(a.cu_q[b], 0), a.total_q);
        s.lq = min(max(a.cu_q[b + 1], s.q0), a.total_q) - s.q0;
        s.k0 = min(max(a.cu_k[b], 0), a.total_k);
        s.lk = min(max(a.cu_k[b + 1], s.k0), a.total_k) - s.k0;
        if (a.k_lens != nullptr) s.lk = min(s.lk, max(a.k_lens[b], 0));
    }
    return s;
}
__device__ __forceinline__ int row_tiles(const AttnVarlenArgs& a, int lq, int rows) {
    return static_cast<int>((static_cast<int64_t>(lq) * a.group + rows - 1) / rows);
}
// key ranges of about `per` tiles of SK keys, equally long, that lk keys are cut into
// (per = 0: one). Rounded to the nearest number: rounded up, 240 tiles of 8192 keys went
// into 121, 121 and 14 each and took 220 us, in halves 188.
constexpr int SK = 32;
__device__ __forceinline__ int key_ranges(int lk, int per) {
    if (per == 0) return 1;
    const int n = (lk + SK - 1) / SK;
    return max((2 * n + per) / (2 * per), 1);
}

// inclusive sum over the wave's lanes: shifts by 1, 2, 4 and 8 inside rows of
// 16, then the rows' last lanes broadcast to the rows behind them
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

// Item `idx` of the launch: the sequences in order, each with its tiles of
// `rows` rows (inside a causal sequence the last, longest one first) times its
// key ranges of `per` tiles. Each lane takes one sequence; a wave scans 64 of
// them at a time, the first 64 (`first`) loaded once by the caller.
__device__ __forceinline__ RowTile find_tile(const AttnVarlenArgs& a, const Sequence& first, int idx, int rows,
                                             int per) {
    const int lane = threadIdx.x & 63;
    RowTile t;
    t.found = false;
    t.q0 = t.lq = t.k0 = t.lk = t.row0 = t.split = 0;
    t.splits = 1;
    int before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const Sequence s = b0 == 0 ? first : load_sequence(a, b0 + lane);
        const int n = row_tiles(a, s.lq, rows), parts = key_ranges(s.lk, per);
        const int incl = wave_scan(n * parts);
        const int total = __builtin_amdgcn_readlane(incl, 63);
        const uint64_t hit = __ballot(before + incl > idx);
        if (idx < before + total && hit != 0) {
            const int src = __builtin_ctzll(hit);
            t.q0 = __builtin_amdgcn_readlane(s.q0, src);
            t.lq = __builtin_amdgcn_readlane(s.lq, src);
            t.k0 = __builtin_amdgcn_readlane(s.k0, src);
            t.lk = __builtin_amdgcn_readlane(s.lk, src);
            t.splits = __builtin_amdgcn_readlane(parts, src);
            const int cnt = __builtin_amdgcn_readlane(n, src);
            const int i = idx - (before + __builtin_amdgcn_readlane(incl, src) - cnt * t.splits);
            if (i < 0 || i >= cnt * t.splits) return t;  // (sums past 2^31: offsets that overlap many times)
            const int tile = per == 0 ? i : i / t.splits;
            t.split = i - tile * t.splits;
            t.row0 = (a.causal ? cnt - 1 - tile : tile) * rows;
            t.found = true;
            return t;
        }
        before += total;
    }
    return t;
}

// number of keys that the query of `token` sees
__device__ __forceinline__ int visible(const AttnVarlenArgs& a, const RowTile& t, int token) {
    if (!a.causal) return t.lk;
    return min(max(token + 1 + t.lk - t.lq, 0), t.lk);
}

// DMA of keys [key, key + ROWS) of one kv head to LDS by one wave, 1 KB = 512 / D
// rows an instruction. Rows from the sequence's end on are zeros.
template <int D, int ROWS, bool VTILE>
__device__ __forceinline__ void dma_tile(const uint16_t* base, int64_t stride, int key, int lk, uint8_t* lds) {
    constexpr int RPI = 512 / D, CPR = D / 8;
    const int lane = threadIdx.x & 63;
    const int left = min(lk - key, ROWS);
    const int bytes = left > 0 ? static_cast<int>(((left - 1) * stride + D) * 2) : 0;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(base + static_cast<int64_t>(key) * stride), 0, bytes, kRsrcWord3);
#pragma unroll
    for (int j = 0; j < ROWS / RPI; ++j) {
        const int row = j * RPI + lane / CPR;
        const int c = VTILE ? swz_v<D>(row, lane % CPR) : swz_k<D>(row, lane % CPR);
        const uint32_t off = static_cast<uint32_t>(row) * static_cast<uint32_t>(stride) * 2u + c * 16;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            r, (__attribute__((address_space(3))) void*)(lds + j * 1024), 16, off, 0, 0, 0);
    }
}

// A lane's byte offsets into a V tile for the transposing reads of channel
// block dt (rows 16 t + 8 e + 4 half + lane % 16 / 4 add (16 t + 8 e) * 2 D)
template <int D>
__device__ __forceinline__ int v_lane_off(int dt) {
    const int lane = threadIdx.x & 63, i = lane & 15;
    const int row = 4 * (lane >> 5) + (i >> 2);
    const int chunk = 4 * dt + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    return row * (2 * D) + swz_v<D>(row, chunk) * 16 + (i & 1) * 8;
}
// The V^T fragments of 16-key group t, one per 32 channels: two transposing
// reads each (4 keys a lane), waited for in the same statement. (Through the
// builtin the compiler orders the reads behind every load in flight, the next
// tiles' DMA included.)
template <class T, int D, int t>
__device__ __forceinline__ void read_v(const uint8_t* vt, const int (&off)[D / 32], typename T::frag (&f)[D / 32]) {
    typedef int v2i __attribute__((ext_vector_type(2)));
    constexpr int O0 = 16 * t * 2 * D, O1 = O0 + 8 * 2 * D;
    const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) const uint8_t*)vt));
    v2i r[D / 16];
    if constexpr (D == 128) {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
            "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
            "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
            "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
            : "v"(base + off[0]), "v"(base + off[1]), "v"(base + off[2]), "v"(base + off[3]), "n"(O0), "n"(O1)
            : "memory");
    } else {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
            "ds_read_b64_tr_b16 %2, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
            : "v"(base + off[0]), "v"(base + off[1]), "n"(O0), "n"(O1)
            : "memory");
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
        f[d] = __builtin_bit_cast(typename T::frag, __builtin_shufflevector(r[2 * d], r[2 * d + 1], 0, 1, 2, 3));
}

// An infinite or NaN value of V at a key that some row does not see would
// reach that row as 0 * inf. In a tile with hidden keys the fragments are
// looked over, such values are taken out of the product (sanitize) and, once
// the loop is done, added to the rows that see them (add_nonfinite).
template <class T>
__device__ __forceinline__ bool has_nonfinite(typename T::frag f) {
    const v4i w = __builtin_bit_cast(v4i, f);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = static_cast<uint32_t>(w[i]);
        bad |= (u & T::kExp) == T::kExp;
        bad |= (u & (T::kExp << 16)) == (T::kExp << 16);
    }
    return bad;
}
template <class T>
__device__ __forceinline__ typename T::frag sanitize(typename T::frag f) {
    v4i w = __builtin_bit_cast(v4i, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t u = static_cast<uint32_t>(w[i]);
        u = (u & T::kExp) == T::kExp ? u & 0xffff0000u : u;
        u = (u & (T::kExp << 16)) == (T::kExp << 16) ? u & 0xffffu : u;
        w[i] = static_cast<int>(u);
    }
    return __builtin_bit_cast(typename T::frag, w);
}
// o (channels 32 d + 8 g + 4 half + c of the lane's row) += the infinite and NaN
// values of keys [key0, kmax)
template <class T, int DT>
__device__ __forceinline__ void add_nonfinite(const uint16_t* v, int64_t stride, int key0, int kmax, v16f (&o)[DT]) {
    const int half = (threadIdx.x & 63) >> 5;
    for (int key = key0; key < kmax; ++key) {
        const uint16_t* vr = v + key * stride + 4 * half;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint2 u = *reinterpret_cast<const uint2*>(vr + 32 * d + 8 * g);
                const uint32_t h[4] = {u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float inf = (h[c] & 0x8000u) ? -__builtin_inff() : __builtin_inff();
                    const float bad = (h[c] & T::kMant) ? __builtin_nanf("") : inf;
                    o[d][4 * g + c] += (h[c] & T::kExp) == T::kExp ? bad : 0.0f;
                }
            }
    }
}

// ---- few rows: 32 of them, the keys over the waves --------------------------
// Four waves share a tile of 32 rows and take its 32-key tiles in turn, each
// with K and V slots of its own (no barrier in the loop; a slot is refilled as
// soon as its fragments are in registers). Their (O, m, sum) are joined through
// LDS in wave order. Two workgroups a CU (64 KB of tiles each). With a.splits > 1
// long sequences' keys are further cut into ranges, whose partial results
// attn_join_kernel adds in order. The launch is at most two workgroups a CU,
// which walk over the items that the lengths on the device give: a grid sized by
// the host's bound on them would mostly be workgroups without work, 2.5 us each.
constexpr int SR = 32, SW = 4;
constexpr int kFewGrid = 512;  // workgroups of the launch at most, two a CU

// Key tiles per range, about; 0: no ranges. As many as make the launch one item a
// workgroup, or a quarter more items than row tiles; at least four a wave, at most
// a.splits ranges a sequence. Where row tiles alone take more than a quarter of the
// workgroups and are about as long, each stays whole: they keep the memory busy by
// themselves, and ranges only add their join (us, 24 heads, tokens, whole / in ranges: 6
// of 1000 keys 26 / 29, 8 of 8192 keys 161 / 176; of unlike lengths, 8192 and 5 of 64 100
// / 34, 10 random ones up to 8192 135 / 114).
__device__ __forceinline__ int range_tiles(const AttnVarlenArgs& a, const Sequence& first) {
    if (a.splits == 1) return 0;
    const int lane = threadIdx.x & 63;
    int longest = 0;
    float work = 0.0f, tiles = 0.0f;  // key tiles of all row tiles, row tiles: sums that need no last digit
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const Sequence s = b0 == 0 ? first : load_sequence(a, b0 + lane);
        const int kt = (s.lk + SK - 1) / SK;
        const float n = static_cast<float>(row_tiles(a, s.lq, SR));
        work += wave_sum_dpp(n * static_cast<float>(kt));
        tiles += wave_sum_dpp(n);
        longest = max(longest, wave_reduce_dpp(kt, [](int x, int y) { return max(x, y); }));
    }
    tiles *= static_cast<float>(a.hk);
    work *= static_cast<float>(a.hk);
    const bool alike = tiles > kFewGrid / 4 && static_cast<float>(longest) * tiles < 1.5f * work;
    // (a sequence has at most 2^25 key tiles; offsets that overlap may sum to any number)
    int per = alike ? longest : static_cast<int>(fminf(work / fmaxf(kFewGrid, 1.25f * tiles), 0x1p25f)) + 1;
    per = max(max(per, 4 * SW), (longest + a.splits - 1) / a.splits);
    return __builtin_amdgcn_readfirstlane(min(per, max(longest, 1)));
}

// E channels of an output row: acc / tot, zeros where the row sees no key
template <class T, int E>
__device__ __forceinline__ void store_row(uint16_t* op, const float (&acc)[E], float tot, bool none) {
    const float inv = 1.0f / tot;
#pragma unroll
    for (int e = 0; e < E; e += 8) {
        u32x4 st;
#pragma unroll
        for (int c = 0; c < 4; ++c) st[c] = none ? 0u : T::pack(acc[e + 2 * c] * inv, acc[e + 2 * c + 1] * inv);
        *reinterpret_cast<u32x4*>(op + e) = st;
    }
}

// LDS bytes of a wave: its tiles, later its share of O
template <int D>
struct Few {
    static constexpr int TILES = (D == 128 ? 2 : 4) * SK * D * 2, O = SR * (D + 4) * 4;
    static constexpr int WB = O > TILES ? O : TILES;
};

template <class T, int D>
__device__ __forceinline__ void few_item(const AttnVarlenArgs& a, const RowTile& t, int hk, uint8_t* ring) {
    using frag = typename T::frag;
    constexpr int KS = D / 16, DT = D / 32;
    constexpr int TB = SK * D * 2;       // bytes of a K or V tile
    constexpr int P = TB / 1024;         // DMA instructions per tile
    constexpr int NS = D == 128 ? 1 : 2;  // K and V slots of a wave
    constexpr int PITCH = D + 4;         // floats per row of the joined O
    constexpr int WB = SR * PITCH * 4 > 2 * NS * TB ? SR * PITCH * 4 : 2 * NS * TB;  // LDS bytes of a wave
    static_assert(WB == Few<D>::WB, "LDS of the kernel");
    float(*ml)[SR][2] = reinterpret_cast<float(*)[SR][2]>(ring + SW * WB);

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, half = lane >> 5;
    const int rows = t.lq * a.group;  // < 2^31: the host bounds total_q * Hq
    const int row = min(t.row0 + l32, rows - 1);
    const int token = row / a.group;
    const int head = hk * a.group + row % a.group;
    const int kmax = visible(a, t, token);
    const int kend = visible(a, t, (min(t.row0 + SR, rows) - 1) / a.group);
    const int kfull = visible(a, t, t.row0 / a.group);
    // 32-key tiles of this range
    const int ntile = (kend + SK - 1) / SK, range = ((t.lk + SK - 1) / SK + t.splits - 1) / t.splits;
    const int tile0 = min(t.split * range, ntile);
    const int tile1 = min(tile0 + range, ntile);

    frag qf[KS];
    {
        const uint16_t* qp = a.q + (static_cast<int64_t>(t.q0) + token) * a.q_t + head * a.q_h + 8 * half;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const frag*>(qp + 16 * s);
    }
    const uint16_t* kbase = a.k + static_cast<int64_t>(t.k0) * a.k_t + hk * a.k_h;
    const uint16_t* vbase = a.v + static_cast<int64_t>(t.k0) * a.v_t + hk * a.v_h;
    uint8_t* kring = ring + wave * WB;
    uint8_t* vring = kring + NS * TB;

    v16f o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    float m = kNegInf;
    v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};  // all four the same
    int nonfinite = -1;  // first of this wave's tiles whose V was sanitized
    int voff[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) voff[d] = v_lane_off<D>(d);

    auto key_of = [&](int i) { return (tile0 + wave + SW * i) * SK; };
    auto issue_k = [&](int i) { dma_tile<D, SK, false>(kbase, a.k_t, key_of(i), t.lk, kring + i % NS * TB); };
    auto issue_v = [&](int i) { dma_tile<D, SK, true>(vbase, a.v_t, key_of(i), t.lk, vring + i % NS * TB); };
    const int n = tile1 - tile0 > wave ? (tile1 - tile0 - wave + SW - 1) / SW : 0;
    if (n > 0) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            issue_k(i);
            issue_v(i);
        }
    }
    for (int i = 0; i < n; ++i) {
        const int key0 = key_of(i);
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<(2 * NS - 1) * P>();  // K of tile i
        __builtin_amdgcn_sched_barrier(0);
        v16f s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
        const uint8_t* kt = kring + i % NS * TB;
        frag kf[KS];
#pragma unroll
        for (int c = 0; c < KS; ++c)
            kf[c] = *reinterpret_cast<const frag*>(kt + l32 * (2 * D) + swz_k<D>(l32, 2 * c + half) * 16);
#pragma unroll
        for (int c = 0; c < KS; ++c) s = T::mma(kf[c], qf[c], s);
        __builtin_amdgcn_sched_barrier(0);
        wait_lgkmcnt0();  // the slot's fragments are in registers
        __builtin_amdgcn_sched_barrier(0);
        issue_k(i + NS);

        const bool hidden = key0 + SK > kfull;  // some row does not see some key
        float p[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = s[r] * a.scale_log2;
        if (hidden) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (key0 + 8 * (r >> 2) + 4 * half + (r & 3) >= kmax) p[r] = kNegInf;
        }
        float mt = p[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mt = fmaxf(mt, p[r]);
        mt = half_max(mt);
        const bool bump = mt > m + kSlack;
        const float m_new = bump ? mt : m;
        if (__ballot(bump)) {
            const float f = bump ? __builtin_amdgcn_exp2f(m - m_new) : 1.0f;
            sum *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= f;
        }
        m = m_new;
        const float neg = (m == kNegInf ? 0.0f : -m) + T::kPBias;
        uint32_t pk[8];
#pragma unroll
        for (int r = 0; r < 16; r += 2)
            pk[r / 2] = T::pack(__builtin_amdgcn_exp2f(p[r] + neg), __builtin_amdgcn_exp2f(p[r + 1] + neg));
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<(2 * NS - 1) * P>();  // V of tile i
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t* vt = vring + i % NS * TB;
        frag vf[2][DT];
        read_v<T, D, 0>(vt, voff, vf[0]);
        read_v<T, D, 1>(vt, voff, vf[1]);
        __builtin_amdgcn_sched_barrier(0);
        issue_v(i + NS);
        if (hidden) {
            bool bad = false;
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int d = 0; d < DT; ++d) bad |= has_nonfinite<T>(vf[g][d]);
            if (__ballot(bad)) {
                if (nonfinite < 0) nonfinite = i;
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int d = 0; d < DT; ++d) vf[g][d] = sanitize<T>(vf[g][d]);
            }
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const frag pf = __builtin_bit_cast(frag, (v4i){static_cast<int>(pk[4 * g]), static_cast<int>(pk[4 * g + 1]),
                                                           static_cast<int>(pk[4 * g + 2]), static_cast<int>(pk[4 * g + 3])});
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] = T::mma(vf[g][d], pf, o[d]);
            sum = T::add4(pk[4 * g], pk[4 * g + 1], sum);
            sum = T::add4(pk[4 * g + 2], pk[4 * g + 3], sum);
        }
    }
    wait_vmcnt<0>();  // the loads past the last tile no longer write the ring
    if (nonfinite >= 0)
        for (int i = nonfinite; i < n; ++i)
            add_nonfinite<T, DT>(vbase, a.v_t, key_of(i), min(key_of(i) + SK, kmax), o);

    // the waves' shares: O into the wave's own LDS, m and sum behind all of it
    const float own = half_sum(sum[0]);
    float* osh = reinterpret_cast<float*>(ring + wave * WB);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<v4f*>(osh + l32 * PITCH + 32 * d + 8 * g + 4 * half) =
                (v4f){o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (half == 0) {
        ml[wave][l32][0] = m;
        ml[wave][l32][1] = own;
    }
    __syncthreads();

    // thread: row tid / 8, channels (tid % 8) * D / 8 ..
    const int jr = threadIdx.x >> 3;
    const int jrow = t.row0 + jr;
    if (jrow < rows) {
        constexpr int E = D / 8;
        const int c0 = (threadIdx.x & 7) * E;
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
            const float* src = reinterpret_cast<const float*>(ring + w * WB) + jr * PITCH + c0;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += f * src[e];
        }
        const int64_t jtoken = static_cast<int64_t>(t.q0) + jrow / a.group;
        const int jhead = hk * a.group + jrow % a.group;
        if (t.splits > 1) {
            const int64_t at = (jtoken * a.hq + jhead) * a.splits + t.split;
            float* po = a.part_o + at * D + c0;
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<v4f*>(po + e) = (v4f){acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
            if (c0 == 0) {
                a.part_ml[2 * at] = mm;
                a.part_ml[2 * at + 1] = tot;
            }
        } else {
            store_row<T, E>(a.out + jtoken * a.o_t + jhead * a.o_h + c0, acc, tot,
                            visible(a, t, jrow / a.group) == 0);
        }
    }
    __syncthreads();  // the next item's tiles take the place of O
}

template <class T, int D>
__global__ __launch_bounds__(SW * 64, 2) void attn_few_kernel(AttnVarlenArgs a) {
    // One LDS object: with two, the compiler orders every read of the tiles
    // behind all DMA in flight.
    __shared__ __attribute__((aligned(1024))) uint8_t ring[SW * Few<D>::WB + SW * SR * 8];
    const Sequence first = load_sequence(a, threadIdx.x & 63);
    const int per = range_tiles(a, first);
    for (int item = blockIdx.x;; item += gridDim.x) {
        const RowTile t = find_tile(a, first, item / a.hk, SR, per);
        if (!t.found) return;
        few_item<T, D>(a, t, item % a.hk, ring);
    }
}

// Partial results of one row, added in order: those of range u lie at row
// at + u * step of part_o and part_ml. Eight ranges' loads go out together (one
// after the other, 16 tokens over up to 8192 keys took 7 us here, most of it
// waiting).
template <class T, int E>
__device__ __forceinline__ void join_row(const AttnVarlenArgs& a, int64_t at, int64_t step, int splits, int c0,
                                         uint16_t* op, bool none) {
    constexpr int D = 8 * E, U = 8;
    typedef float v2f __attribute__((ext_vector_type(2)));
    float mm = kNegInf, tot = 0.0f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    for (int s0 = 0; s0 < splits; s0 += U) {
        v2f ml[U];
        v4f v[U][E / 4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t p = at + min(s0 + u, splits - 1) * step;
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
            if (s0 + u >= splits) continue;
            // no finite score: O is zero there, the sum zero or NaN
            const float f = ml[u][0] == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(ml[u][0] - mm);
            tot += f * ml[u][1];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += f * v[u][e / 4][e % 4];
        }
    }
    store_row<T, E>(op + c0, acc, tot, none);
}

// The key ranges of a tile of 32 rows: thread: row tid / 8, channels
// (tid % 8) * D / 8 .. Sequences of one range are complete already.
template <class T, int D>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnVarlenArgs a) {
    const Sequence first = load_sequence(a, threadIdx.x & 63);
    const int per = range_tiles(a, first);
    const int hk = blockIdx.x % a.hk;
    const RowTile t = find_tile(a, first, blockIdx.x / a.hk, SR, 0);
    if (!t.found) return;
    const int splits = key_ranges(t.lk, per);
    const int row = t.row0 + (threadIdx.x >> 3);
    if (splits == 1 || row >= t.lq * a.group) return;
    const int64_t token = static_cast<int64_t>(t.q0) + row / a.group;
    const int head = hk * a.group + row % a.group;
    join_row<T, D / 8>(a, (token * a.hq + head) * a.splits, 1, splits, (threadIdx.x & 7) * (D / 8),
                       a.out + token * a.o_t + head * a.o_h, visible(a, t, row / a.group) == 0);
}

// ---- many rows: 128 of them, four waves over one ring -----------------------
// Wave w owns rows 32 w .. of the tile; 64-key tiles stream through an LDS ring
// of two slots and serve all four waves, so a tile's bytes are read once for 128
// rows. A slot holds what one matrix phase reads: V of tile p - 1 and K of tile
// p ("pair" p). Work alternates between a vector phase, V(p): the softmax of
// tile p, and a matrix phase, M(p): O += V P of tile p - 1, then the scores of
// tile p. Two workgroups share a CU (64 KB of LDS, two waves a SIMD), so one's
// exponentials run beside the other's MFMAs. V begins with the fragment reads of
// the next M's first MFMAs, M reads a group of four fragments ahead. (Two groups
// ahead, with a third buffer, measured 1-2% slower, without the matrix phase's
// priority 2 x 24 heads of 4352 took 2% more, 1301 tokens 20% more.) The DMA
// instructions are spread over V's exponentials: sent in one go a wave's eight
// took 460 cycles of the step's 3070, 16 each of the CU's address unit (2 x 24
// heads of 4352 and 4173 tokens, bf16: 462 -> 450 us; one barrier a step instead
// of two: 441). A tile now takes a wave 1330 cycles of V, 1290 of M (1104 of
// them MFMA) and 200 at the barrier, two workgroups' together 2890.
constexpr int MR = 128, MW = 4, MK = 64, MSLOT = 2;

// The K or V tiles of one head in turn: `p` the next tile's first row, `left`
// the bytes from there to the end of the sequence's last row (not positive
// behind it). Each tile's descriptor starts at its own row, so offsets stay
// below a tile's bytes however long the sequence is, and ends with the
// sequence: rows behind it arrive as zeros.
template <int D, bool VTILE>
struct TileStream {
    const uint8_t* p;
    int64_t left, step;
    uint32_t off[MK * D * 2 / 1024 / MW];  // a lane's byte offsets in a tile, one per DMA instruction
    // every `every`-th tile from tile `first` on
    __device__ __forceinline__ void init(const uint16_t* base, int64_t stride, int lk, int first, int every, int wave) {
        p = reinterpret_cast<const uint8_t*>(base + first * MK * stride);
        step = 2 * MK * stride * every;
        left = lk > first * MK ? 2 * ((lk - first * MK - 1) * stride + D) : 0;
        constexpr int RPI = 512 / D, CPR = D / 8;
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < MK / RPI / MW; ++i) {
            const int row = (wave + MW * i) * RPI + lane / CPR;
            const int c = VTILE ? swz_v<D>(row, lane % CPR) : swz_k<D>(row, lane % CPR);
            off[i] = static_cast<uint32_t>(row) * static_cast<uint32_t>(stride) * 2u + c * 16;
        }
    }
    static constexpr int N = MK * D * 2 / 1024 / MW;  // DMA instructions of a wave
    // instruction i of the next tile; the last one moves on
    __device__ __forceinline__ void issue_one(int i, uint8_t* dst, int wave) {
#if defined(__HIP_DEVICE_COMPILE__)  // (the host pass rejects the builtin, and with it the kernels that share this)
        const int64_t n = left < 0 ? 0 : left > 0x7fffffff ? 0x7fffffff : left;
        const __amdgpu_buffer_rsrc_t r =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, static_cast<int>(n), kRsrcWord3);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            r, (__attribute__((address_space(3))) void*)(dst + (wave + MW * i) * 1024), 16, off[i], 0, 0, 0);
        if (i == N - 1) {
            p += step;
            left -= step;
        }
#endif
    }
    __device__ __forceinline__ void issue(uint8_t* dst, int wave) {
#pragma unroll
        for (int i = 0; i < N; ++i) issue_one(i, dst, wave);
    }
};

template <class T, int D>
struct Many {
    using frag = typename T::frag;
    static constexpr int KB = MK / 32;
    static constexpr int KS = D / 16, DT = D / 32;
    static constexpr int TB = MK * D * 2;           // bytes of a K or V tile
    static constexpr int PER = 2 * TB / 1024 / MW;  // DMA instructions per wave and pair
    static constexpr int NPV = 2 * KB * DT / 4, NG = NPV + KB * KS / 4;  // groups of four MFMAs: PV, all
    v16f o[DT], s[KB];
    frag qf[KS], buf[2][4];
    uint32_t pk[8 * KB];  // P: 16-key group g at pk[4 g ..]
    int voff[DT], koff[KS];  // lane offsets of V reads (channel block), K reads (k-step)
    float m;
    v4f sum;  // all four the same

    // fragments of group j: PV units (16-key group u / DT, channel block
    // u % DT), then score units (k-step u / KB, key block u % KB)
    template <int j>
    __device__ __forceinline__ void read_group(const uint8_t* src, frag (&f)[4]) {
        using as3 = __attribute__((address_space(3))) v4s*;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (j < NPV) {
                const int u = 4 * j + i;
                const uint8_t* p = src + voff[u % DT] + 16 * (u / DT) * (2 * D);
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((as3)(p));
                const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((as3)(p + 8 * (2 * D)));
                f[i] = __builtin_bit_cast(frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            } else {
                const int u = 4 * (j - NPV) + i;
                f[i] = *reinterpret_cast<const frag*>(src + TB + koff[u / KB] + 32 * (u % KB) * (2 * D));
            }
        }
    }
    __device__ __forceinline__ frag p_frag(int g) const {
        return __builtin_bit_cast(frag, (v4i){static_cast<int>(pk[4 * g]), static_cast<int>(pk[4 * g + 1]),
                                              static_cast<int>(pk[4 * g + 2]), static_cast<int>(pk[4 * g + 3])});
    }
    template <int j>
    __device__ __forceinline__ void mma_group(const frag (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (j < NPV) {
                const int u = 4 * j + i;
                o[u % DT] = T::mma(f[i], p_frag(u / DT), o[u % DT]);
                if (u % (DT / 2) == 0) {
                    const int r = 4 * (u / DT) + 2 * (u % DT != 0);
                    sum = T::add4(pk[r], pk[r + 1], sum);
                }
            } else {
                const int u = 4 * (j - NPV) + i;
                s[u % KB] = T::mma(f[i], qf[u / KB], s[u % KB]);
            }
        }
    }
    template <int j, bool CLEAN>
    __device__ __forceinline__ void m_groups(const uint8_t* src, bool& bad) {
        if constexpr (j < NG) {
            if constexpr (j + 1 < NG) read_group<j + 1>(src, buf[(j + 1) % 2]);
            if constexpr (CLEAN && j < NPV) {
                bool b = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) b |= has_nonfinite<T>(buf[j % 2][i]);
                if (__ballot(b)) {
                    bad = true;
#pragma unroll
                    for (int i = 0; i < 4; ++i) buf[j % 2][i] = sanitize<T>(buf[j % 2][i]);
                }
            }
            if constexpr (j == NPV) {
#pragma unroll
                for (int r = 0; r < 16 * KB; ++r) s[r >> 4][r & 15] = 0.0f;
            }
            mma_group<j>(buf[j % 2]);
            __builtin_amdgcn_sched_barrier(0);
            m_groups<j + 1, CLEAN>(src, bad);
        }
    }
    template <int j>
    __device__ __forceinline__ void first_scores(const uint8_t* src) {
        if constexpr (j < NG) {
            read_group<j>(src, buf[j % 2]);
            mma_group<j>(buf[j % 2]);
            first_scores<j + 1>(src);
        }
    }

    // dma(i), i < PER: the next DMA instructions, spread over the exponentials
    template <class Dma>
    __device__ __forceinline__ void softmax(int key0, int kfull, int kmax, float c, Dma&& dma) {
        const int half = (threadIdx.x & 63) >> 5;
        if (key0 + MK > kfull) {  // some row of the tile does not see some key
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (key0 + 32 * b + 8 * (r >> 2) + 4 * half + (r & 3) >= kmax) s[b][r] = kNegInf;
        }
        float mt = s[0][0];
#pragma unroll
        for (int r = 1; r < 16 * KB; ++r) mt = fmaxf(mt, s[r >> 4][r & 15]);
        mt = half_max(mt) * c;
        const bool bump = mt > m + kSlack;
        const float m_new = bump ? mt : m;
        if (__ballot(bump)) {
            const float f = bump ? __builtin_amdgcn_exp2f(m - m_new) : 1.0f;
            sum *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= f;
        }
        m = m_new;
        const float neg = (m == kNegInf ? 0.0f : -m) + T::kPBias;
#pragma unroll
        for (int r = 0; r < 16 * KB; r += 2) {
            if (r % (16 * KB / PER) == 0) {
                __builtin_amdgcn_sched_barrier(0);
                dma(r / (16 * KB / PER));
                __builtin_amdgcn_sched_barrier(0);
            }
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r >> 4][r & 15], c, neg));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r >> 4][(r & 15) + 1], c, neg));
            pk[r / 2] = T::pack(p0, p1);
        }
    }
};

__device__ __forceinline__ void phase_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");  // no LDS read or DMA moves across, whatever the compiler thinks of aliasing
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// V(p) and M(p + 1) of one wave. Behind the barrier every wave has done M(p),
// whose slot takes pair p + 2 during V(p), and pair p + 1, sent during V(p - 1),
// has landed. The slots come as restrict pointers, which tells the compiler that
// the reads of `src` do not depend on the DMA into `dst`: the waits and barriers
// see to that. PHASED: a second barrier between V and M. CLEAN: infinities and
// NaN of V are taken out and the first tile that had some is noted.
template <class T, int D, bool CLEAN, bool PHASED>
__device__ __forceinline__ void many_step(Many<T, D>& w, const uint8_t* __restrict src, uint8_t* __restrict dst,
                                          TileStream<D, false>& ks, TileStream<D, true>& vs, float scale, int tile,
                                          int wave, int kfull, int kmax, int& nonfinite) {
    using W = Many<T, D>;
    wait_vmcnt<0>();
    phase_barrier();
    w.template read_group<0>(src, w.buf[0]);
    __builtin_amdgcn_sched_barrier(0);
    w.softmax(tile * MK, kfull, kmax, scale, [&](int i) {
        if (i < W::PER / 2)
            vs.issue_one(i, dst, wave);
        else
            ks.issue_one(i - W::PER / 2, dst + W::TB, wave);
    });
    // P is made in this phase: left to itself the compiler moves the
    // exponentials next to the MFMAs that read them
#pragma unroll
    for (int i = 0; i < 8 * W::KB; ++i) asm volatile("" : "+v"(w.pk[i]));
    __builtin_amdgcn_sched_barrier(0);
    if (PHASED) phase_barrier();
    __builtin_amdgcn_s_setprio(1);
    bool bad = false;
    w.template m_groups<0, CLEAN>(src, bad);
    if (CLEAN && bad && nonfinite < 0) nonfinite = tile;
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
}

// KG = 1: as above. KG = 2, for launches of few tiles, whose workgroups have a CU
// each: eight waves, two groups of four that take the 64-key tiles in turn, each
// with a ring of its own, a phase apart: the second barrier keeps one group's V
// beside the other's M; the groups' (O, m, sum) are joined through LDS (the
// lanes of waves w and w + 4 hold the same rows and channels).
//
// Without a causal mask all tiles take equally long, and a last round of
// workgroups that fills few of the CUs takes nearly as long as a full one. The
// tiles from a.tail on are then cut into a.splits key ranges, a workgroup each
// (KG = 1), and attn_tail_join_kernel adds what these leave in scratch.
template <class T, int D, int KG>
__global__ __launch_bounds__(KG * MW * 64, 2) void attn_many_kernel(AttnVarlenArgs a, int tiles) {
    using W = Many<T, D>;
    constexpr int PAIR = 2 * W::TB, RING = MSLOT * PAIR, CHUNKS = D / 8;
    constexpr int JOIN = KG == 2 ? MW * 64 * (D / 2 + 2) * 4 : 0;  // a group's O, m and sum
    constexpr int RINGS = KG * RING > JOIN ? KG * RING : JOIN;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[RINGS + KG * MW * 4];  // and a flag of every wave

    const int lane = threadIdx.x & 63;
    const int wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = KG == 1 ? wave_all : wave_all % MW, kg = KG == 1 ? 0 : wave_all / MW;
    uint8_t* const ring = lds + kg * RING;
    const int l32 = lane & 31, half = lane >> 5;
    // Causal: the sequences' last, longest tiles first, the heads of one tile
    // side by side (a head stays on few XCDs as workgroups go round-robin over
    // them). Otherwise all tiles of a head on one XCD.
    const int piece = KG == 1 ? static_cast<int>(blockIdx.x) - a.tail : -1;  // not negative: a range of a tile
    int hk, idx;
    if (a.causal) {
        hk = blockIdx.x % a.hk;
        idx = blockIdx.x / a.hk;
    } else {
        const int logical = xcd_remap(piece < 0 ? blockIdx.x : a.tail + piece % a.tail_tiles, tiles * a.hk);
        hk = logical / tiles;
        idx = logical % tiles;
    }
    const RowTile t = find_tile(a, load_sequence(a, lane), idx, MR, 0);
    if (!t.found) return;

    const int rows = t.lq * a.group;
    const int row = min(t.row0 + 32 * wave + l32, rows - 1);
    const bool valid = t.row0 + 32 * wave + l32 < rows;
    const int token = row / a.group;
    const int head = hk * a.group + row % a.group;
    const int kmax = visible(a, t, token);
    const int kend = visible(a, t, (min(t.row0 + MR, rows) - 1) / a.group);  // of the whole tile
    int n = (kend + MK * KG - 1) / (MK * KG);                         // steps
    const int kfull = visible(a, t, t.row0 / a.group);                // of every row
    int tile0 = kg;                                                   // the first 64-key tile
    if (piece >= 0) {
        const int per = (n + a.splits - 1) / a.splits;
        tile0 = min(piece / a.tail_tiles * per, n);
        n = min(per, n - tile0);
    }

    W w;
    const uint16_t* kbase = a.k + static_cast<int64_t>(t.k0) * a.k_t + hk * a.k_h;
    const uint16_t* vbase = a.v + static_cast<int64_t>(t.k0) * a.v_t + hk * a.v_h;
    int nonfinite = -1;  // first of this wave's tiles whose V was sanitized

    const auto pass = [&](auto clean) __attribute__((always_inline)) {
        constexpr bool CLEAN = decltype(clean)::value;
        // The scores of the first tile need its K and Q: these loads go out first,
        // the registers are set up beside them, then follows pair 1. (Q, the registers
        // and then all loads: 1000 cycles more.)
        TileStream<D, false> ks;
        TileStream<D, true> vs;
        ks.init(kbase, a.k_t, t.lk, tile0, KG, wave);
        ks.issue(ring + W::TB, wave);
        if constexpr (!CLEAN) {
            const uint16_t* qp = a.q + (static_cast<int64_t>(t.q0) + token) * a.q_t + head * a.q_h + 8 * half;
#pragma unroll
            for (int i = 0; i < W::KS; ++i) w.qf[i] = *reinterpret_cast<const typename T::frag*>(qp + 16 * i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < W::DT; ++d) w.voff[d] = v_lane_off<D>(d);
#pragma unroll
            for (int c = 0; c < W::KS; ++c) w.koff[c] = l32 * (2 * D) + swz_k<D>(l32, 2 * c + half) * 16;
        }
#pragma unroll
        for (int d = 0; d < W::DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) w.o[d][r] = 0.0f;
#pragma unroll
        for (int r = 0; r < 16 * W::KB; ++r) w.s[r >> 4][r & 15] = 0.0f;
        w.m = kNegInf;
        w.sum = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
        vs.init(vbase, a.v_t, t.lk, tile0, KG, wave);
        __builtin_amdgcn_sched_barrier(0);
        vs.issue(ring + PAIR, wave);
        ks.issue(ring + PAIR + W::TB, wave);
        wait_vmcnt<W::PER>();
        phase_barrier();
        w.template first_scores<W::NPV>(ring);
        if (KG == 2 && kg == 1) phase_barrier();
        for (int p = 0; p < n; ++p)
            many_step<T, D, CLEAN, KG == 2>(w, ring + ((p + 1) % MSLOT) * PAIR, ring + (p % MSLOT) * PAIR, ks, vs,
                                            a.scale_log2, KG * p + tile0, wave, kfull, kmax, nonfinite);
        if (KG == 2 && kg == 0) phase_barrier();
        wait_vmcnt<0>();  // the loads past the last tile no longer write the ring
    };
    pass(std::false_type{});
    // An infinity or NaN of V in a place that some row does not see has made that
    // row's product 0 * inf: if O holds any such value the tile is done again with
    // them taken out, and added to the rows that see them. (Looking V over in every
    // masked step took 3600 of its 6700 cycles, and a second copy of the loop.)
    if (a.causal && n > 0) {
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int d = 0; d < W::DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r & 3] = __builtin_fmaf(w.o[d][r], 0.0f, x[r & 3]);
        const bool bad = __ballot(x[0] + x[1] + x[2] + x[3] != 0.0f) != 0;
        int* const flags = reinterpret_cast<int*>(lds + RINGS);
        if (lane == 0) flags[wave_all] = bad;
        __syncthreads();
        int any = 0;
#pragma unroll
        for (int i = 0; i < KG * MW; ++i) any |= flags[i];
        if (__builtin_amdgcn_readfirstlane(any)) {
            __syncthreads();  // (every wave has left the ring)
            pass(std::true_type{});
            if (nonfinite >= 0)
                for (int tile = nonfinite; tile * MK < kmax; tile += KG)
                    add_nonfinite<T, W::DT>(vbase, a.v_t, tile * MK, min(tile * MK + MK, kmax), w.o);
        }
    }
    float tot = half_sum(w.sum[0]);

    if constexpr (KG == 2) {
        __syncthreads();
        float* const part = reinterpret_cast<float*>(lds) + wave * 64 * (D / 2 + 2);
        if (kg == 1) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
                *reinterpret_cast<v4f*>(part + (c * 64 + lane) * 4) =
                    (v4f){w.o[c / 4][c % 4 * 4], w.o[c / 4][c % 4 * 4 + 1], w.o[c / 4][c % 4 * 4 + 2],
                          w.o[c / 4][c % 4 * 4 + 3]};
            part[64 * (D / 2) + lane] = w.m;
            part[64 * (D / 2) + 64 + lane] = tot;
        }
        __syncthreads();
        if (kg == 1) return;
        const float m1 = part[64 * (D / 2) + lane], t1 = part[64 * (D / 2) + 64 + lane];
        const float top = fmaxf(w.m, m1);
        // no finite score in a group: its O is zero, its sum zero or NaN
        const float f0 = w.m == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(w.m - top);
        const float f1 = m1 == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m1 - top);
        tot = tot * f0 + t1 * f1;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const v4f x = *reinterpret_cast<const v4f*>(part + (c * 64 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w.o[c / 4][c % 4 * 4 + e] = w.o[c / 4][c % 4 * 4 + e] * f0 + x[e] * f1;
        }
    }

    if (piece >= 0) {
        const int64_t at = static_cast<int64_t>(piece) * MR + 32 * wave + l32;
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
                v[i] = kmax == 0 ? 0u : sw[0];
                v[2 + i] = kmax == 0 ? 0u : sw[1];
            }
            *reinterpret_cast<u32x4*>(op + 32 * d + 8 * g) = (u32x4){v[0], v[1], v[2], v[3]};
        }
}

// The key ranges of the last tiles: 32 rows of one a workgroup.
template <class T, int D>
__global__ __launch_bounds__(256) void attn_tail_join_kernel(AttnVarlenArgs a, int tiles) {
    const int tile = blockIdx.x / (MR / 32), row0 = blockIdx.x % (MR / 32) * 32 + (threadIdx.x >> 3);
    const int logical = xcd_remap(a.tail + tile, tiles * a.hk), hk = logical / tiles;
    const RowTile t = find_tile(a, load_sequence(a, threadIdx.x & 63), logical % tiles, MR, 0);
    if (!t.found) return;
    const int row = t.row0 + row0;
    if (row >= t.lq * a.group) return;
    const int64_t token = static_cast<int64_t>(t.q0) + row / a.group;
    const int head = hk * a.group + row % a.group;
    join_row<T, D / 8>(a, static_cast<int64_t>(tile) * MR + row0, static_cast<int64_t>(a.tail_tiles) * MR, a.splits,
                       (threadIdx.x & 7) * (D / 8), a.out + token * a.o_t + head * a.o_h,
                       visible(a, t, row / a.group) == 0);
}

// upper bound on the tiles of `rows` rows that the sequences have
int64_t tile_bound(int total_q, int batch, int group, int rows) {
    const int64_t seqs = batch < total_q ? batch : total_q;
    return (static_cast<int64_t>(total_q) * group + seqs * (rows - 1)) / rows;
}

}  // namespace

constexpr int kGroupTiles = 256;  // workgroups of two groups that run at once, one a CU

// Tiles of 128 rows, or of 32: the latter while they are one round of workgroups
// (us, 32 / 128 rows; 28 heads, causal: 120 tiles of 128 14.0 / 16.9, 144 19.5 / 18.1,
// 192 23.2 / 19.8; 4 heads, all of 500 keys: 104 14.6 / 14.9, 136 20.5 / 15.2; of 8000
// keys: 72 78 / 84, 136 145 / 90). A token or a few over caches fill few rows of
// either tile, and there the keys of a long sequence have to go into ranges, which the
// tiles of 32 do by the lengths on the device: up to 1024 of those (us, 32 / 128 rows: one
// of 8192 keys beside 5 of 64, 24 heads, 34 / 101, beside 31, 28 on 4 heads, 17 / 138,
// 127 24.6 / 142; 32 random lengths up to 8192 55 / 106; all alike, 6 x 8192 139 / 136, 64 x
// 300 16.3 / 14.7, the launch that joins; 16 on 8 heads of 64, 32 x 8192 114 / 97). More
// keep every CU busy whatever their lengths (of 2048 tiles, random, 885 / 819). A few: at
// most 8 queries and 32 rows a sequence on average, as a prompt among tokens wants its
// large tiles (6 heads, 512 tokens and 31 single ones over 4000 keys each 105 / 78).
constexpr int kManyTiles = kFewGrid * SR / MR + 1;

// The tail of a launch of `tiles` equal tiles of 128 rows without a causal mask:
// how many tiles its last round has (a multiple of eight where there are as many, so
// that a tile's ranges run on one XCD), and into how many key ranges they go, one
// round of them. The gain in us: a round of few workgroups takes a us a step (64
// keys), ranges c for their start and the join, and for each of their tiles b a step
// and d for its float results. Fitted to 24 heads over 1500 and 5000 keys with 16 to
// 208 tiles in the last round (us, whole / in ranges; D 128, 5000 keys: 16 tiles
// 227 / 169, 64 228 / 187, 160 232 / 218, 208 234 / 238; 1500 keys: 16 81 / 71, 64
// 80 / 78, 112 81 / 82; D 64, 5000 keys: 16 127 / 111, 160 138 / 129, 208 141 / 149;
// 1500 keys: 16 equal, 64 46 / 47). In two ranges, or where a tile has a CU
// (two wave groups), nothing is gained: power then bounds the last round too. Lengths
// are on the device: the keys' average stands for them here, which decides the time,
// not the result.
static void plan_tail(AttnVarlenPlan& p, int tiles, int total_k, int batch, int D) {
    const int slots = 2 * kGroupTiles, tail = std::min((tiles % slots + 7) / 8 * 8, tiles);
    if (p.groups == 2 || tail == 0) return;
    const double a = D == 128 ? 0.97 : 0.33, b = D == 128 ? 0.0038 : 0.0012, c = D == 128 ? 11.4 : 8.0,
                 d = D == 128 ? 0.034 : 0.01;
    const double steps = static_cast<double>(total_k) / batch / MK;
    const int s = std::min({16, slots / tail, static_cast<int>(steps / 4)});
    if (s < 3 || steps * a - c <= tail * (steps * b + d)) return;
    p.splits = s;
    p.tail_tiles = tail;
    p.tail = tiles - tail;
}

AttnVarlenPlan attn_varlen_plan(int total_q, int total_k, int batch, int hq, int hk, int D, bool causal) {
    AttnVarlenPlan p{};
    p.splits = 1;
    if (total_q <= 0 || batch <= 0 || total_k <= 0) return p;
    const int64_t many = tile_bound(total_q, batch, hq / hk, MR) * hk;
    const int64_t few = tile_bound(total_q, batch, hq / hk, SR) * hk;
    const int64_t seqs = std::min(batch, total_q), rows = static_cast<int64_t>(total_q) * (hq / hk);
    const bool cached = few <= 2 * kFewGrid && total_k / 8 >= total_q && total_q <= 8 * seqs && rows <= SR * seqs;
    // (a workgroup a tile, and a grid has less than 2^32 threads: beyond, the kernel that walks)
    p.many = many >= kManyTiles && many < (1 << 22) && !cached;
    if (p.many) {
        p.tail = static_cast<int>(many);
        // Two groups a tile for one round of workgroups, or two with a causal mask (the
        // tiles have half the keys on average), where the keys repay the join, about 2 us
        // a round (us, one group / two, 28 heads, causal: 3 x 300 tokens 14.0 / 15.7, 3 x
        // 350 15.4 / 15.9, 2 x 400 15.4 / 16.3, 2 x 430 15.7 / 16.3, 2 x 450 16.4 / 16.5, 2 x
        // 480 17.1 / 16.8, 1100 28.9 / 24.3, 4 x 500, 452 tiles, 21.8 / 28.2, 2 x 1000, 444,
        // 30.1 / 31.4, 1200, 264, 30.4 / 25.6, 2048, 448, 47.3 / 43.8, 3000, 660, 76 / 81; all
        // keys: 2 x 400 16.2 / 17.1, 2 x 450 17.5 / 16.9, 1301 tokens of 24 heads, 264, 35.6 /
        // 46.9). Lengths are on the device: the average decides, of the slots with k_lens.
        // Unlike lengths would have two groups pay from a lower one (512 + 269 tokens 16.5 /
        // 16.1, 600 + 180 18.5 / 17.3).
        const int keys = total_k / batch;
        p.groups = (many <= kGroupTiles && keys >= 448) || (causal && many <= 2 * kGroupTiles && keys >= 1100) ? 2 : 1;
        if (!causal) plan_tail(p, p.tail, total_k, batch, D);
        p.part_rows = p.splits > 1 ? static_cast<int64_t>(p.tail_tiles) * p.splits * MR : 0;
        return p;
    }
    // Most key ranges a sequence may be cut into: where the tiles of 32 rows alone
    // do not fill half of the launch's workgroups, or over caches, and the keys are more
    // than 1024 (one token of 28 heads over 600 keys, us, whole / in ranges with their join:
    // 11.1 / 13.2; 1000: 13.6 / 13.6; 1500: 17.3 / 13.4; 3000: 28 / 13.8). The ranges'
    // length is found on the device.
    if (total_k <= 8 * SW * SK || (few > kFewGrid / 2 && !cached)) return p;
    const int64_t most = std::min((total_k + 4 * SW * SK - 1) / (4 * SW * SK), 32);
    p.splits = static_cast<int>(std::min(most, 8192 / few));  // (parts of 140 MB at most)
    p.part_rows = static_cast<int64_t>(total_q) * hq * p.splits;
    return p;
}

template <class T, int D>
static hipError_t launch_few(const AttnVarlenArgs& a, hipStream_t stream) {
    const int64_t tiles = tile_bound(a.total_q, a.batch, a.group, SR) * a.hk;
    const int64_t items = tiles * a.splits;
    hipLaunchKernelGGL((attn_few_kernel<T, D>), dim3(static_cast<unsigned>(items < kFewGrid ? items : kFewGrid)),
                       dim3(SW * 64), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    hipLaunchKernelGGL((attn_join_kernel<T, D>), dim3(static_cast<unsigned>(tiles)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

template <class T, int D>
static hipError_t launch_many(const AttnVarlenArgs& a, hipStream_t stream) {
    const int tiles = static_cast<int>(tile_bound(a.total_q, a.batch, a.group, MR));
    const unsigned grid = a.tail + a.tail_tiles * a.splits;
    if (a.groups == 2)
        hipLaunchKernelGGL((attn_many_kernel<T, D, 2>), dim3(grid), dim3(2 * MW * 64), 0, stream, a, tiles);
    else
        hipLaunchKernelGGL((attn_many_kernel<T, D, 1>), dim3(grid), dim3(MW * 64), 0, stream, a, tiles);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.tail_tiles == 0) return e;
    hipLaunchKernelGGL((attn_tail_join_kernel<T, D>), dim3(a.tail_tiles * (MR / 32)), dim3(256), 0, stream, a, tiles);
    return hipGetLastError();
}

template <class T, int D>
static hipError_t launch_attn(const AttnVarlenArgs& a, hipStream_t stream) {
    return a.many ? launch_many<T, D>(a, stream) : launch_few<T, D>(a, stream);
}

hipError_t launch_attention_varlen(const AttnVarlenArgs& a, int dtype, int D, hipStream_t stream) {
    if (dtype == QIMG_BF16)
        return D == 128 ? launch_attn<Bf16, 128>(a, stream) : launch_attn<Bf16, 64>(a, stream);
    return D == 128 ? launch_attn<Fp16, 128>(a, stream) : launch_attn<Fp16, 64>(a, stream);
}

}  // namespace qimg
