// attention_tiles.h — what the attention kernels over row-major K and V tiles in LDS share:
// element types, the LDS layout, and the work of a wave on 32 rows and 64-key tiles
// (attention_varlen.hip describes the arithmetic and the phases).
#pragma once

#include "qimg_device.h"

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
    static constexpr bool kBf = true;
    static constexpr uint32_t kOnes = 0x3f803f80u, kNans = 0x7fc07fc0u;
    __device__ static __forceinline__ v4f mma16(frag a, frag b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
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
    static constexpr bool kBf = false;
    static constexpr uint32_t kOnes = 0x3c003c00u, kNans = 0x7e007e00u;
    __device__ static __forceinline__ v4f mma16(frag a, frag b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
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

// A lane's byte offsets into a V tile for the transposing reads of channel
// block dt (rows 16 t + 8 e + 4 half + lane % 16 / 4 add (16 t + 8 e) * 2 D)
template <int D>
__device__ __forceinline__ int v_lane_off(int dt) {
    const int lane = threadIdx.x & 63, i = lane & 15;
    const int row = 4 * (lane >> 5) + (i >> 2);
    const int chunk = 4 * dt + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    return row * (2 * D) + swz_v<D>(row, chunk) * 16 + (i & 1) * 8;
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

// rows of a workgroup's tile, its waves, keys of a step, slots of the ring
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

}  // namespace

}  // namespace qimg
