// rope_packed.hip — rotary positions of packed heads: of each token's h heads
// of d values the first h_rot are turned in their first r values,
//   (a, b) -> (a cos - b sin, b cos + a sin)
// with a, b the values (i, i + r / 2), or (2 i, 2 i + 1) interleaved, and
// (cos, sin) entry i of the table's row `position of the token`; all other
// values are copied. In fp32, one rounding to out's type.
//
// Bound by memory: each value is read and written once, eight (or twice four)
// neighbouring values a thread. A thread holds both values of each of its
// pairs before it writes, so out may be x. Angles come from the table (made
// by the caller in 64 bits once): fp32 angles of far positions are off by
// position * 2^-24 radians.
#include "qimg_device.h"
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
template <int DT>
__device__ __forceinline__ void store4(void* p, int64_t i, v4f f) {
    if constexpr (DT == QIMG_FP32) {
        *reinterpret_cast<v4f*>(static_cast<float*>(p) + i) = f;
    } else {
        uint2 u;
        if constexpr (DT == QIMG_BF16) {
            u = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
        } else {
            u = make_uint2(f32_to_f16(f[0]) | (static_cast<uint32_t>(f32_to_f16(f[1])) << 16),
                           f32_to_f16(f[2]) | (static_cast<uint32_t>(f32_to_f16(f[3])) << 16));
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = u;
    }
}

// Thread: eight values of one head of one token. The first r / 8 threads of a
// turned head take pairs (halves: values 4 i .. and r / 2 + 4 i ..;
// interleaved: 8 i ..), the rest copy eight values.
template <int IN, int OUT>
__device__ __forceinline__ void rope_eight(const RopeArgs& a, int64_t idx) {
    const int per = a.d / 8;
    const int64_t th = idx / per;
    const int e = static_cast<int>(idx % per);
    const int64_t t = th / a.h;
    const int head = static_cast<int>(th % a.h);
    const int pos = a.positions[t];
    if (pos < 0 || pos >= a.table_rows) return;  // such a token is left alone
    const int64_t x = t * a.x_t + head * a.x_h, o = t * a.o_t + head * a.o_h;
    const bool turn = head < a.h_rot && e < a.r / 8;
    const bool halves = turn && !a.interleaved;
    const int i0 = halves ? 4 * e : 8 * e, i1 = halves ? a.r / 2 + 4 * e : 8 * e + 4;
    v4f p = load4<IN>(a.x, x + i0), q = load4<IN>(a.x, x + i1);
    if (turn) {
        // (cos, sin) of pairs 4 e .. 4 e + 3
        const float* cs = a.table + static_cast<int64_t>(pos) * a.r + 8 * e;
        const v4f lo = *reinterpret_cast<const v4f*>(cs), hi = *reinterpret_cast<const v4f*>(cs + 4);
        const float co[4] = {lo[0], lo[2], hi[0], hi[2]}, si[4] = {lo[1], lo[3], hi[1], hi[3]};
        if (halves) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float u = p[c], v = q[c];
                p[c] = __builtin_fmaf(u, co[c], -(v * si[c]));
                q[c] = __builtin_fmaf(v, co[c], u * si[c]);
            }
        } else {
            const v4f u = p, v = q;
            p[0] = __builtin_fmaf(u[0], co[0], -(u[1] * si[0]));
            p[1] = __builtin_fmaf(u[1], co[0], u[0] * si[0]);
            p[2] = __builtin_fmaf(u[2], co[1], -(u[3] * si[1]));
            p[3] = __builtin_fmaf(u[3], co[1], u[2] * si[1]);
            q[0] = __builtin_fmaf(v[0], co[2], -(v[1] * si[2]));
            q[1] = __builtin_fmaf(v[1], co[2], v[0] * si[2]);
            q[2] = __builtin_fmaf(v[2], co[3], -(v[3] * si[3]));
            q[3] = __builtin_fmaf(v[3], co[3], v[2] * si[3]);
        }
    }
    store4<OUT>(a.out, o + i0, p);
    store4<OUT>(a.out, o + i1, q);
}

constexpr int64_t kMaxBlocks = 1 << 22;  // (a grid has less than 2^32 threads)

template <int IN, int OUT>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    const int64_t total = static_cast<int64_t>(a.tokens) * a.h * (a.d / 8);
    for (int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; idx < total;
         idx += static_cast<int64_t>(gridDim.x) * 256)
        rope_eight<IN, OUT>(a, idx);
}

template <int IN>
hipError_t launch_in(const RopeArgs& a, int out_dtype, hipStream_t stream) {
    const int64_t total = static_cast<int64_t>(a.tokens) * a.h * (a.d / 8);
    const int64_t blocks = (total + 255) / 256;
    const dim3 grid(static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks));
    switch (out_dtype) {
    case QIMG_FP32: hipLaunchKernelGGL((rope_kernel<IN, QIMG_FP32>), grid, dim3(256), 0, stream, a); break;
    case QIMG_BF16: hipLaunchKernelGGL((rope_kernel<IN, QIMG_BF16>), grid, dim3(256), 0, stream, a); break;
    default: hipLaunchKernelGGL((rope_kernel<IN, QIMG_FP16>), grid, dim3(256), 0, stream, a); break;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rope_packed(const RopeArgs& a, int x_dtype, int out_dtype, hipStream_t stream) {
    if (a.tokens == 0 || a.h == 0) return hipSuccess;
    switch (x_dtype) {
    case QIMG_FP32: return launch_in<QIMG_FP32>(a, out_dtype, stream);
    case QIMG_BF16: return launch_in<QIMG_BF16>(a, out_dtype, stream);
    default: return launch_in<QIMG_FP16>(a, out_dtype, stream);
    }
}

}  // namespace qimg
