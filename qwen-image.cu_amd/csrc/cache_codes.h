// cache_codes.h — the codes of a quantized key/value cache: a row (token, kv
// head) of D values is D codes, int8 or OCP e4m3, and one byte E, the power of
// two 2^(E - 127) that they count. E is the least for which the largest
// magnitude of the row is at most 127 (int8) or 448 (e4m3) times it, 1 at least.
//
// Powers of two, not amax / 127: a code times one is exact in bf16 and in fp32
// (7 bits of an int8 code, 4 of e4m3), so K and V enter the matrix unit and come
// back from the cache without a rounding of their own, scores and softmax weights
// carry no scale, and a row's scale is one byte instead of four. It costs e4m3
// nothing (its step follows the value; the smallest step alone moves) and int8 at
// most one bit: its step is amax / 127 to amax / 64.
//
// A token whose k or v of a head holds an infinity or a NaN gets E = 255 for that
// head's k, which makes its scores NaN for every row that sees it and for no
// other; such a v is stored as zeros, so codes of V are always finite.
#pragma once

#include "qimg_device.h"
#include "qimg_internal.h"

namespace qimg {

struct Int8Codes {
    static constexpr int kDtype = QIMG_INT8;
    static constexpr int kTopExp = 6;  // 127 = (1 + kTopMant / 2^23) 2^kTopExp
    static constexpr uint32_t kTopMant = 0x7e0000u;
    static constexpr uint32_t kNanCode = 0u;  // (0 times the scale of E = 255)
    __device__ static __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
        return i8x4_rne_sat(a, b, c, d);
    }
    __device__ static __forceinline__ v4f decode4(uint32_t w, float scale) {
        return (v4f){static_cast<float>(static_cast<int8_t>(w)) * scale,
                     static_cast<float>(static_cast<int8_t>(w >> 8)) * scale,
                     static_cast<float>(static_cast<int8_t>(w >> 16)) * scale,
                     static_cast<float>(static_cast<int8_t>(w >> 24)) * scale};
    }
};
struct E4m3Codes {
    static constexpr int kDtype = QIMG_FP8_E4M3;
    static constexpr int kTopExp = 8;  // 448
    static constexpr uint32_t kTopMant = 0x600000u;
    static constexpr uint32_t kNanCode = 0x7f7f7f7fu;
    __device__ static __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
        return e4m3x4(a, b, c, d);
    }
    __device__ static __forceinline__ v4f decode4(uint32_t w, float scale) {
        typedef float v2f __attribute__((ext_vector_type(2)));
        const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
        const v2f hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
        return (v4f){lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
    }
};

// 2^(E - 127); E = 255 gives infinity, E = 0 (which no writer leaves) zero
__device__ __forceinline__ float exp_scale(uint32_t e) { return __uint_as_float(e << 23); }

// E of a row whose largest magnitude has these bits (finite)
template <class C>
__device__ __forceinline__ int row_exp(uint32_t amax_bits) {
    const int e = static_cast<int>(amax_bits >> 23) - C::kTopExp + ((amax_bits & 0x7fffffu) > C::kTopMant ? 1 : 0);
    return e < 1 ? 1 : e;
}

// Four codes (a dword, the first in the low byte) as two pairs of 16-bit values.
template <class C, bool BF>
__device__ __forceinline__ uint2 decode_pairs(uint32_t w, float scale) {
    if constexpr (C::kDtype == E4m3Codes::kDtype) {
        if constexpr (BF) {
            return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false)),
                              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true)));
        } else {
            return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false)),
                              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true)));
        }
    } else if constexpr (BF) {
        // exact in the upper half of an fp32 value
        const v4f f = Int8Codes::decode4(w, scale);
        return make_uint2(__builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u),
                          __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u));
    } else {
        // code + 128 in the low byte of 1024 makes fp16 1024 + code + 128; then times the
        // scale in two factors, as fp16 alone holds no 2^-25 and below: one rounding, and
        // none where the value is an fp16 value
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const uint32_t u = w ^ 0x80808080u;
        const h2 lo = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
        const h2 hi = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
        const float first = fmaxf(scale, 0x1p-14f);
        const _Float16 s1 = static_cast<_Float16>(first), s2 = static_cast<_Float16>(scale < 0x1p-14f ? scale * 0x1p14f : 1.0f);
        const h2 c = {1152, 1152}, f1 = {s1, s1}, f2 = {s2, s2};
        return make_uint2(__builtin_bit_cast(uint32_t, (lo - c) * f1 * f2), __builtin_bit_cast(uint32_t, (hi - c) * f1 * f2));
    }
}

}  // namespace qimg
