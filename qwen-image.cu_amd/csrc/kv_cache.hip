// kv_cache.hip — the heads of a packed projection on their way into attention:
// RMS norm of each q and k head, y = x (mean(x^2) + eps)^-1/2 w, its rotary
// positions, (a, b) -> (a cos - b sin, b cos + a sin), and either all heads to a
// packed output or k and v as codes into their cache pages, in one pass; and the
// rows of a cache read back.
//
// Bound by memory: each value is read and written once. A head is G lanes of eight
// values (G = 8, 16 or 32: its sum of squares and largest magnitude are reduced
// within a wave by DPP, nothing goes through LDS), a lane holds both values of each
// of its pairs, and a whole head is in registers before any of it is written, so a
// packed output may be x. Statistics, norm and rotation are fp32, with one rounding
// to out's type, or to the code. k and v of a (token, kv head) are the same lanes'
// work where they become codes: a NaN in one marks the other. 10816 tokens of 28 + 4 + 4
// heads of 128, fp32 to bf16, 57.5 us (5.2 TB/s; a large copy reaches 4.9, part of this
// stays in the caches); 10751 tokens with k and v into e4m3 pages 65 us (4.4 TB/s); a few
// tokens 3.5 to 4.5 us, one chain of loads (position, table and x, or slot and x).
#include <algorithm>
#include <type_traits>

#include "cache_codes.h"
#include "qimg_internal.h"

namespace qimg {

namespace {

// four neighbouring values of the type
template <int DT>
__device__ __forceinline__ v4f load4(const void* p, int64_t i) {
    if constexpr (DT == QIMG_FP32) {
        return *reinterpret_cast<const v4f*>(static_cast<const float*>(p) + i);
    } else {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        const uint16_t h[4] = {static_cast<uint16_t>(u.x), static_cast<uint16_t>(u.x >> 16), static_cast<uint16_t>(u.y),
                               static_cast<uint16_t>(u.y >> 16)};
        v4f f;
#pragma unroll
        for (int c = 0; c < 4; ++c) f[c] = DT == QIMG_BF16 ? bf16_to_f32(h[c]) : f16_to_f32(h[c]);
        return f;
    }
}
__device__ __forceinline__ void store4(void* p, int64_t i, v4f f, int dtype) {
    if (dtype == QIMG_FP32) {
        *reinterpret_cast<v4f*>(static_cast<float*>(p) + i) = f;
    } else if (dtype == QIMG_BF16) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) =
            make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
    } else {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) =
            make_uint2(f32_to_f16(f[0]) | (static_cast<uint32_t>(f32_to_f16(f[1])) << 16),
                       f32_to_f16(f[2]) | (static_cast<uint32_t>(f32_to_f16(f[3])) << 16));
    }
}

// reduction over groups of G neighbouring lanes (wave_reduce_dpp's first steps)
template <int G, typename T, typename Op>
__device__ __forceinline__ T group_reduce(T v, Op op) {
    v = op(v, dpp32<0xB1>(v));
    v = op(v, dpp32<0x4E>(v));
    v = op(v, dpp32<0x141>(v));
    if constexpr (G >= 16) v = op(v, dpp32<0x140>(v));
    if constexpr (G >= 32) {
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const auto sw = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        v = op(__builtin_bit_cast(T, static_cast<unsigned>(sw[0])), __builtin_bit_cast(T, static_cast<unsigned>(sw[1])));
    }
    return v;
}

struct Eight {
    v4f p, q;  // values i0 .. i0 + 3 and i1 .. i1 + 3 of the head
};

// Norm and rotation of a lane's eight values; `w` the norm's weights or null.
template <int G>
__device__ __forceinline__ void norm_turn(const HeadsArgs& a, Eight& x, const uint16_t* w, const float* cs, int e,
                                          int i0, int i1, bool valid) {
    if (w != nullptr) {
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) s = __builtin_fmaf(x.p[c], x.p[c], s);
#pragma unroll
        for (int c = 0; c < 4; ++c) s = __builtin_fmaf(x.q[c], x.q[c], s);
        s = group_reduce<G>(s, [](float u, float v) { return u + v; });
        const float r = 1.0f / sqrtf(s / static_cast<float>(a.d) + a.eps);
        v4f wp = {0.0f, 0.0f, 0.0f, 0.0f}, wq = wp;
        if (valid) {
            wp = load4<QIMG_BF16>(w, i0);
            wq = load4<QIMG_BF16>(w, i1);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            x.p[c] = x.p[c] * r * wp[c];
            x.q[c] = x.q[c] * r * wq[c];
        }
    }
    if (cs != nullptr && e < a.r / 8) {
        // (cos, sin) of pairs 4 e .. 4 e + 3
        const v4f lo = *reinterpret_cast<const v4f*>(cs + 8 * e), hi = *reinterpret_cast<const v4f*>(cs + 8 * e + 4);
        const float co[4] = {lo[0], lo[2], hi[0], hi[2]}, si[4] = {lo[1], lo[3], hi[1], hi[3]};
        const v4f u = x.p, v = x.q;
        if (!a.interleaved) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                x.p[c] = __builtin_fmaf(u[c], co[c], -(v[c] * si[c]));
                x.q[c] = __builtin_fmaf(v[c], co[c], u[c] * si[c]);
            }
        } else {
            x.p[0] = __builtin_fmaf(u[0], co[0], -(u[1] * si[0]));
            x.p[1] = __builtin_fmaf(u[1], co[0], u[0] * si[0]);
            x.p[2] = __builtin_fmaf(u[2], co[1], -(u[3] * si[1]));
            x.p[3] = __builtin_fmaf(u[3], co[1], u[2] * si[1]);
            x.q[0] = __builtin_fmaf(v[0], co[2], -(v[1] * si[2]));
            x.q[1] = __builtin_fmaf(v[1], co[2], v[0] * si[2]);
            x.q[2] = __builtin_fmaf(v[2], co[3], -(v[3] * si[3]));
            x.q[3] = __builtin_fmaf(v[3], co[3], v[2] * si[3]);
        }
    }
}

template <int IN>
__device__ __forceinline__ Eight load8(const void* x, int64_t at, int i0, int i1, bool valid) {
    Eight r;
    r.p = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    r.q = r.p;
    if (valid) {
        r.p = load4<IN>(x, at + i0);
        r.q = load4<IN>(x, at + i1);
    }
    return r;
}

// bits of the largest magnitude of the head; 0x7f800000 and more: not finite
template <int G>
__device__ __forceinline__ uint32_t head_amax(const Eight& x) {
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        m = max(m, __float_as_uint(x.p[c]) & 0x7fffffffu);
        m = max(m, __float_as_uint(x.q[c]) & 0x7fffffffu);
    }
    return group_reduce<G>(m, [](uint32_t u, uint32_t v) { return u > v ? u : v; });
}

// Codes of a head with largest magnitude `amax` (bits). Two kinds of values must not come
// back as infinities: finite ones as 2^128, and those of fp16 rows as 65536, which is
// infinite there. That happens to rows whose largest code would be the first of the next
// power of two (int8 64 times 2^122 and 2^10, e4m3 256 times 2^120 and 2^8); the code below
// replaces it.
template <class C, int IN>
__device__ __forceinline__ void store_codes(uint8_t* codes, uint8_t* exps, int64_t row, int d, int e, int i0, int i1,
                                            const Eight& x, uint32_t amax) {
    const int exp = row_exp<C>(amax);
    const float inv = __uint_as_float(static_cast<uint32_t>(254 - exp) << 23);
    v4f p = x.p * inv, q = x.q * inv;
    constexpr bool kInt8 = C::kDtype == QIMG_INT8;
    constexpr int kTop = kInt8 ? 127 + 122 : 127 + 120, kTop16 = kInt8 ? 127 + 10 : 127 + 8;
    if (exp == kTop || (IN == QIMG_FP16 && exp == kTop16 && amax <= 0x477fe000u)) {  // 65504
        constexpr float kMost = kInt8 ? 63.0f : 240.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            p[c] = __builtin_amdgcn_fmed3f(p[c], -kMost, kMost);
            q[c] = __builtin_amdgcn_fmed3f(q[c], -kMost, kMost);
        }
    }
    *reinterpret_cast<uint32_t*>(codes + row * d + i0) = C::encode4(p[0], p[1], p[2], p[3]);
    *reinterpret_cast<uint32_t*>(codes + row * d + i1) = C::encode4(q[0], q[1], q[2], q[3]);
    if (e == 0) exps[row] = static_cast<uint8_t>(exp);
}

// Lane group: one head of one token; with a cache (C not void) the k and v heads of
// one kv head. The first r / 8 lanes of a turned head take pairs (halves: values
// 4 e .. and r / 2 + 4 e ..), the others and interleaved ones 8 e ...
template <int IN, int G, class C>
__global__ __launch_bounds__(256) void heads_kernel(HeadsArgs a) {
    constexpr bool CACHE = !std::is_same_v<C, void>;
    const uint32_t units = CACHE ? a.nq + a.nk : a.nq + 2 * a.nk;
    const uint32_t total = static_cast<uint32_t>(a.tokens) * units;
    const uint32_t u = blockIdx.x * (256 / G) + threadIdx.x / G;
    const int e = threadIdx.x % G;
    if (u >= total) return;  // (a lane group leaves whole)
    const uint32_t t = u / units;
    const int head = static_cast<int>(u - t * units);
    const bool turned = head < a.nq + a.nk;
    const float* cs = nullptr;
    if (a.table != nullptr) {
        const int pos = a.positions[t];
        if (pos < 0 || pos >= a.table_rows) return;  // such a token is left alone
        if (turned) cs = a.table + static_cast<int64_t>(pos) * a.r;
    }
    const bool valid = 8 * e < a.d;
    const bool halves = cs != nullptr && !a.interleaved && e < a.r / 8;
    const int i0 = halves ? 4 * e : 8 * e, i1 = halves ? a.r / 2 + 4 * e : 8 * e + 4;
    if (!CACHE || head < a.nq) {
        Eight x = load8<IN>(a.x, t * a.x_t + head * a.x_h, i0, i1, valid);
        if (turned) norm_turn<G>(a, x, head < a.nq ? a.wq : a.wk, cs, e, i0, i1, valid);
        if (valid) {
            const int64_t o = t * a.o_t + head * a.o_h;
            store4(a.out, o + i0, x.p, a.out_dtype);
            store4(a.out, o + i1, x.q, a.out_dtype);
        }
    }
    if constexpr (CACHE) {
        if (head >= a.nq) {
            const int kv = head - a.nq;
            const int slot = a.slots[t];
            if (slot < 0 || slot >= a.n_slots) return;
            Eight k = load8<IN>(a.k, t * a.k_t + kv * a.k_h, i0, i1, valid);
            Eight v = load8<IN>(a.v, t * a.v_t + kv * a.v_h, 8 * e, 8 * e + 4, valid);
            norm_turn<G>(a, k, a.wk, cs, e, i0, i1, valid);
            const uint32_t km = head_amax<G>(k), vm = head_amax<G>(v);
            const bool v_bad = vm >= 0x7f800000u, bad = km >= 0x7f800000u || v_bad;
            const int64_t page = slot >> a.page_shift;
            const int64_t row = (((page * a.nk + kv) << a.page_shift) | (slot & ((1 << a.page_shift) - 1)));
            if (!valid) return;
            if (bad) {
                *reinterpret_cast<uint2*>(a.ck + row * a.d + 8 * e) = make_uint2(C::kNanCode, C::kNanCode);
                if (e == 0) a.cke[row] = 255;
            } else {
                store_codes<C, IN>(a.ck, a.cke, row, a.d, e, i0, i1, k, km);
            }
            if (v_bad) {
                *reinterpret_cast<uint2*>(a.cv + row * a.d + 8 * e) = make_uint2(0u, 0u);
                if (e == 0) a.cve[row] = 127;
            } else {
                store_codes<C, IN>(a.cv, a.cve, row, a.d, e, 8 * e, 8 * e + 4, v, vm);
            }
        }
    }
}

constexpr int kMostBlocks = 1 << 22;  // of a launch (a grid has less than 2^32 threads)

// `a` from token t on
template <int IN>
HeadsArgs from_token(HeadsArgs a, int t) {
    const auto ahead = [](auto p, int64_t bytes) {
        if (p != nullptr) p = (decltype(p))((uintptr_t)p + bytes);
        return p;
    };
    constexpr int64_t in = IN == QIMG_FP32 ? 4 : 2;
    a.x = ahead(a.x, in * t * a.x_t), a.k = ahead(a.k, in * t * a.k_t), a.v = ahead(a.v, in * t * a.v_t);
    a.out = ahead(a.out, (a.out_dtype == QIMG_FP32 ? 4 : 2) * t * a.o_t);
    a.positions = ahead(a.positions, int64_t{4} * t), a.slots = ahead(a.slots, int64_t{4} * t);
    a.tokens -= t;
    return a;
}

template <int IN, class C>
void launch_heads_in(const HeadsArgs& all, hipStream_t stream) {
    const int g = all.d <= 64 ? 8 : all.d <= 128 ? 16 : 32;
    const int64_t units = std::is_same_v<C, void> ? all.nq + 2 * all.nk : all.nq + all.nk;  // of a token, < 2^24
    const int64_t most = kMostBlocks * (256 / g) / units;                                   // tokens of a launch
    for (int64_t t = 0; t < all.tokens; t += most) {
        HeadsArgs a = from_token<IN>(all, static_cast<int>(t));
        a.tokens = static_cast<int>(std::min<int64_t>(a.tokens, most));
        const dim3 grid(static_cast<unsigned>((a.tokens * units + 256 / g - 1) / (256 / g)));
        if (g == 8) {
            hipLaunchKernelGGL((heads_kernel<IN, 8, C>), grid, dim3(256), 0, stream, a);
        } else if (g == 16) {
            hipLaunchKernelGGL((heads_kernel<IN, 16, C>), grid, dim3(256), 0, stream, a);
        } else if constexpr (std::is_same_v<C, void>) {
            hipLaunchKernelGGL((heads_kernel<IN, 32, C>), grid, dim3(256), 0, stream, a);
        }
    }
}

// ---- reading back -------------------------------------------------------------

// Sixteen codes of k and of v of one row and head a lane; RR rows a workgroup, whose
// sequences its first wave finds once. Bound by memory: 55255 keys of 4 heads of 128 from
// e4m3 to bf16, 170 MB, 40 us (4.2 TB/s); of few keys by the search's loads, 7 us.
constexpr int RR = 32;

template <class C, int OUT>
__device__ __forceinline__ void read16(const uint8_t* codes, uint32_t exp, void* out, int64_t at) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(codes);
    const float scale = exp_scale(exp);
    if constexpr (OUT == QIMG_FP32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<v4f*>(static_cast<float*>(out) + at + 4 * i) = C::decode4(w[i], scale);
    } else {
        u32x4 r[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint2 p = decode_pairs<C, OUT == QIMG_BF16>(w[i], scale);
            r[i / 2][i % 2 * 2] = p.x;
            r[i / 2][i % 2 * 2 + 1] = p.y;
        }
        u32x4* o = reinterpret_cast<u32x4*>(static_cast<uint16_t*>(out) + at);
        o[0] = r[0];
        o[1] = r[1];
    }
}

template <class C, int OUT>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheReadArgs a, int first) {
    __shared__ int64_t src[RR];  // first slot's row of head 0, -1: nothing to read
    const int row0 = first + blockIdx.x * RR;
    if (threadIdx.x < RR) {
        const int row = row0 + threadIdx.x;
        // the last sequence that starts at or before the row, among those of a rising list
        int lo = 0, hi = a.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (a.cu[mid] <= row) lo = mid; else hi = mid;
        }
        int64_t at = -1;
        const int64_t key = static_cast<int64_t>(row) - a.cu[lo];
        if (row < a.total && key >= 0 && row < a.cu[lo + 1] && key < a.k_lens[lo] &&
            (key >> a.c.page_shift) < a.max_blocks) {
            const int page = a.table[static_cast<int64_t>(lo) * a.max_blocks + (key >> a.c.page_shift)];
            if (page >= 0 && page < a.c.n_pages)
                at = ((static_cast<int64_t>(page) * a.c.hk) << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1));
        }
        src[threadIdx.x] = at;
    }
    __syncthreads();
    const int per = a.d / 16, lanes = a.c.hk * per;
    for (int i = threadIdx.x; i < RR * lanes; i += 256) {
        const int r = i / lanes, head = (i % lanes) / per, c = i % per;
        if (src[r] < 0) continue;
        const int64_t row = src[r] + (static_cast<int64_t>(head) << a.c.page_shift);
        read16<C, OUT>(a.c.k + row * a.d + 16 * c, a.c.ke[row], a.k, (row0 + r) * a.k_t + head * a.k_h + 16 * c);
        read16<C, OUT>(a.c.v + row * a.d + 16 * c, a.c.ve[row], a.v, (row0 + r) * a.v_t + head * a.v_h + 16 * c);
    }
}

}  // namespace

template <class C>
struct Tag {
    using type = C;
};

hipError_t launch_heads(const HeadsArgs& a, int x_dtype, int codes, hipStream_t stream) {
    const auto go = [&](auto c) {
        using C = typename decltype(c)::type;
        switch (x_dtype) {
        case QIMG_FP32: launch_heads_in<QIMG_FP32, C>(a, stream); break;
        case QIMG_BF16: launch_heads_in<QIMG_BF16, C>(a, stream); break;
        default: launch_heads_in<QIMG_FP16, C>(a, stream); break;
        }
    };
    if (codes == QIMG_INT8) go(Tag<Int8Codes>{});
    else if (codes == QIMG_FP8_E4M3) go(Tag<E4m3Codes>{});
    else go(Tag<void>{});
    return hipGetLastError();
}

template <class C>
static void launch_read(const CacheReadArgs& a, int out_dtype, hipStream_t stream) {
    const int blocks = (a.total + RR - 1) / RR;
    for (int b = 0; b < blocks; b += kMostBlocks) {
        const dim3 grid(std::min(blocks - b, kMostBlocks));
        const int first = b * RR;
        switch (out_dtype) {
        case QIMG_FP32: hipLaunchKernelGGL((cache_read_kernel<C, QIMG_FP32>), grid, dim3(256), 0, stream, a, first); break;
        case QIMG_BF16: hipLaunchKernelGGL((cache_read_kernel<C, QIMG_BF16>), grid, dim3(256), 0, stream, a, first); break;
        default: hipLaunchKernelGGL((cache_read_kernel<C, QIMG_FP16>), grid, dim3(256), 0, stream, a, first); break;
        }
    }
}

hipError_t launch_cache_read(const CacheReadArgs& a, int codes, int out_dtype, hipStream_t stream) {
    if (codes == QIMG_INT8) launch_read<Int8Codes>(a, out_dtype, stream);
    else launch_read<E4m3Codes>(a, out_dtype, stream);
    return hipGetLastError();
}

}  // namespace qimg
