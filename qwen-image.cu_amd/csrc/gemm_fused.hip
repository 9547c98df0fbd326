// gemm_fused.hip — the bf16 linear with its epilogue:
//   z[m,n] = sum_k bf16(x[m,k]) w[n,k] + bias[n]
//   y[m,n] = act(z[m,n]) * (sum_k bf16(x[m,k]) w_up[n,k] + bias_up[n])   (the second factor with w_up only)
//   out[m,n] = residual[m,n] + gate[n] * y[m,n]                          (each where given)
// x fp32 (rounded to bf16, nearest even) or bf16, weights bf16 [N, K], fp32
// accumulation; bias, activation, product, gate and residual in fp32 on the
// accumulators, one rounding to out's type.
//
// linear_gemv_kernel (one or two rows) and linear_rows_kernel (up to 16) are bound
// by reading the weights; linear_small_kernel takes products of few tiles (a
// prompt of some hundred tokens), linear_tile_kernel the rest, both also with the
// sum over k split over workgroups; linear_join_kernel then adds the parts in
// order and applies the epilogue. x in fp32 for the tiles, and operands whose
// rows are not whole 16-byte pieces, first go through pack_rows_kernel into
// scratch. linear_fused_plan chooses.
#include <algorithm>
#include <type_traits>

#include "qimg_device.h"
#include "qimg_internal.h"

namespace qimg {

namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr int kRsrcWord3 = 0x00020000;  // raw unswizzled buffer (gfx9 family)
constexpr uint32_t kOob = 0x80000000u;  // offset >= num_records: reads zero

// v / (1 + 2^-t): the sigmoid form of both activations keeps the relative
// error of small results (no 1 - 1), also far in the negative tail: with e = 2^(-|t|/2)
// it is v / (1 + e^2), for t < 0 times e twice, so that nothing but the result leaves
// the range of normal numbers (1 / (1 + 2^-t) did from v = -87 on)
__device__ __forceinline__ float activate(float v, int act) {
    if (act == QIMG_ACT_NONE) return v;
    float h;  // t / 2: log2(e) / 2 times the sigmoid's argument
    if (act == QIMG_ACT_SILU)
        h = v * 0.72134752044448170f;
    else
        h = v * __builtin_fmaf(0.05147162f, v * v, 1.1511041f);  // sqrt(2/pi) log2(e) (v + 0.044715 v^3)
    const float e = __builtin_amdgcn_exp2f(-fabsf(h)), f = h < 0.0f ? e : 1.0f;
    return v * f * __builtin_amdgcn_rcpf(__builtin_fmaf(e, e, 1.0f)) * f;
}

// The epilogue of four neighbouring outputs of row m, columns n ..; their
// bias, bias_up and gate are loaded once per column.
struct Columns {
    float b[4], bu[4], g[4];
};
__device__ __forceinline__ Columns load_columns(const LinearFusedArgs& a, int n) {
    Columns c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = min(n + i, a.N - 1);
        c.b[i] = a.bias != nullptr ? bf16_to_f32(a.bias[k]) : 0.0f;
        c.bu[i] = a.bias_up != nullptr ? bf16_to_f32(a.bias_up[k]) : 0.0f;
        c.g[i] = a.gate != nullptr ? a.gate[k] : 1.0f;
    }
    return c;
}
// gate * act(z + bias) [* (u + bias_up)]
template <bool GATED, class V>
__device__ __forceinline__ void finish_values(const LinearFusedArgs& a, const Columns& c, const V& z, const V& u,
                                              float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = activate(z[i] + c.b[i], a.act);
        if (GATED) v[i] *= u[i] + c.bu[i];
        v[i] *= c.g[i];
    }
}
template <bool GATED>
__device__ __forceinline__ void finish4(const LinearFusedArgs& a, const Columns& c, int m, int n, const float (&z)[4],
                                        const float (&u)[4]) {
    float v[4];
    finish_values<GATED>(a, c, z, u, v);
    const int64_t o = m * a.ldo + n, r = m * a.ldr + n;
    const bool bf = a.out_dtype == QIMG_BF16;
    if (a.vec4 && n + 3 < a.N) {
        if (a.residual != nullptr) {
            if (a.res_dtype == QIMG_BF16) {
                const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.residual) + r);
                v[0] += __uint_as_float(q.x << 16);
                v[1] += __uint_as_float(q.x & 0xffff0000u);
                v[2] += __uint_as_float(q.y << 16);
                v[3] += __uint_as_float(q.y & 0xffff0000u);
            } else {
                const v4f q = *reinterpret_cast<const v4f*>(static_cast<const float*>(a.residual) + r);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += q[i];
            }
        }
        if (bf)
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + o) =
                make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        else
            *reinterpret_cast<v4f*>(static_cast<float*>(a.out) + o) = (v4f){v[0], v[1], v[2], v[3]};
        return;
    }
    for (int i = 0; i < 4 && n + i < a.N; ++i) {
        if (a.residual != nullptr)
            v[i] += a.res_dtype == QIMG_BF16 ? bf16_to_f32(static_cast<const uint16_t*>(a.residual)[r + i])
                                             : static_cast<const float*>(a.residual)[r + i];
        if (bf)
            static_cast<uint16_t*>(a.out)[o + i] = f32_to_bf16(v[i]);
        else
            static_cast<float*>(a.out)[o + i] = v[i];
    }
}

// the epilogue of one output
template <bool GATED>
__device__ __forceinline__ void finish1(const LinearFusedArgs& a, int m, int n, float z, float u) {
    float v = activate(z + (a.bias != nullptr ? bf16_to_f32(a.bias[n]) : 0.0f), a.act);
    if (GATED) v *= u + (a.bias_up != nullptr ? bf16_to_f32(a.bias_up[n]) : 0.0f);
    if (a.gate != nullptr) v *= a.gate[n];
    const int64_t o = m * a.ldo + n, r = m * a.ldr + n;
    if (a.residual != nullptr)
        v += a.res_dtype == QIMG_BF16 ? bf16_to_f32(static_cast<const uint16_t*>(a.residual)[r])
                                      : static_cast<const float*>(a.residual)[r];
    if (a.out_dtype == QIMG_BF16)
        static_cast<uint16_t*>(a.out)[o] = f32_to_bf16(v);
    else
        static_cast<float*>(a.out)[o] = v;
}

// ---- tiles -------------------------------------------------------------------
// A workgroup of eight waves owns TM x TN products (TN weight rows; with GATED
// 16 rows of w and 16 of w_up in turn, so a lane holds both factors of an
// output), wave (wm, wn) of 2 x 4 its TM/2 x TN/4, as 16x16 blocks
// (v_mfma_f32_16x16x32_bf16, w as the A operand: a lane holds four neighbouring
// columns of a row). K advances 64 elements (128-byte rows) a stage through a
// ring of LDS slots filled by buffer loads: whole lines, 8 rows an instruction,
// 16-byte chunk c of row r at c ^ ((r >> 1) & 7), so a fragment's 16 rows fall on
// different banks; rows past M or N and k past K arrive as zeros.
//
// A stage is four phases, one quadrant (half of the wave's rows x half of its
// columns) each: first fragments are read, then its MFMAs run. Phases 0 and 2 read
// the rows' halves, 1 the second half of the columns, and 3 the first half of the
// next stage's, into the registers of this stage's second: every other stage takes
// the halves in the other order, and no phase reads more than its MFMAs take (LDS
// gives a CU 128 bytes a cycle: 8 fragments of four waves 256 cycles). Waves 4-7
// are one barrier behind waves 0-3, so on every SIMD one wave's MFMAs run beside
// the other's LDS reads and DMA issue. A quarter of a slot (A rows or B rows of one
// half) is refilled two barriers after its last reader, with the stage NS later.
//
// Measured: 4352x3584x12288 with gate and residual 283 us (1.35 PFLOP/s, the matrix
// units busy 78% of the time at the clock that power allows), 8192^3 873 us; all
// waves in step 15% more, the reads not evened out 1%.
template <int TM_, int TN_>
struct Tile {
    static constexpr int TM = TM_, TN = TN_;
    static constexpr int MB = TM / 32, NB = TN / 64;               // 16-blocks of a wave
    static constexpr int MB0 = (MB + 1) / 2, MB1 = MB - MB0;       // rows of phases 0, 1 and of 2, 3
    static constexpr int NB0 = NB / 2, NB1 = NB - NB0;
    static constexpr int AB = TM * 128, BB = TN * 128, STAGE = AB + BB;
    static constexpr int NS = 152 * 1024 / STAGE < 4 ? 152 * 1024 / STAGE : 4;
    // DMA instructions a wave issues per quarter
    static constexpr int IA0 = (4 * MB0 + 7) / 8, IA1 = (4 * MB1 + 7) / 8, IB0 = NB0, IB1 = NB1;
    static constexpr int ALL = IA0 + IB0 + IB1 + IA1;
    static constexpr int LDS = NS * STAGE + 1024;  // the last KB takes the DMA of waves without a share
    static_assert(NS >= 2 && LDS <= 160 * 1024 && NB % 2 == 0, "ring");
    static constexpr int PITCH = TN / 4 + 4;  // floats per row of a wave's output staging
    static_assert(8 * 16 * PITCH * 4 <= NS * STAGE, "staging takes the ring's place");
};

template <class T, bool GATED>
__global__ __launch_bounds__(512) void linear_tile_kernel(LinearFusedArgs a) {
    constexpr int NS = T::NS, MB = T::MB, NB = T::NB, MB0 = T::MB0, NB0 = T::NB0, MB1 = T::MB1;
    constexpr int TNO = GATED ? T::TN / 2 : T::TN;  // output columns of the tile
    __shared__ __attribute__((aligned(1024))) uint8_t lds[T::LDS];

    const int tiles_m = (a.M + T::TM - 1) / T::TM, tiles_n = (a.N + TNO - 1) / TNO;
    // An XCD's workgroups take neighbouring tiles, eight tile rows by n: the 32 in
    // flight read about 8 + 4 tiles' operands through its L2.
    const int logical = xcd_remap(blockIdx.x, tiles_m * tiles_n * a.splits);
    const int split = logical / (tiles_m * tiles_n);
    const int in_split = logical - split * (tiles_m * tiles_n);
    const int band = in_split / (8 * tiles_n);
    const int high = min(tiles_m - 8 * band, 8);
    const int in_band = in_split - band * 8 * tiles_n;
    const int m0 = (8 * band + in_band % high) * T::TM;
    const int n0 = in_band / high * TNO;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    const int st0 = split * a.split_stages;
    const int nst = min((a.K + 63) / 64 - st0, a.split_stages);

    // DMA: a wave's instructions of quarter A0, A1 (rows wm * 16 MB + 16 MB0 ..),
    // B0, B1; instruction q = wave + 8 i of a quarter brings 8 rows
    const int rows_m = min(a.M - m0, T::TM), rows_n = min(a.N - n0, TNO);
    uint32_t offa[T::IA0 + T::IA1], offb[T::IB0 + T::IB1];
    int dsta[T::IA0 + T::IA1], dstb[T::IB0 + T::IB1];  // LDS offset in a slot (A rows, then B rows)
    int ka[T::IA0 + T::IA1], kb[T::IB0 + T::IB1];      // first k of a lane's chunk
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int cnt = h == 0 ? 4 * MB0 : 4 * MB1, per = cnt / 2;  // instructions, of one wm
#pragma unroll
        for (int i = 0; i < (h == 0 ? T::IA0 : T::IA1); ++i) {
            const int q = wave + 8 * i, j = h == 0 ? i : T::IA0 + i;
            const int r0 = q / per * (16 * MB) + (h == 0 ? 0 : 16 * MB0) + q % per * 8;
            const int row = r0 + (lane >> 3);
            const int c = (lane & 7) ^ ((row >> 1) & 7);
            dsta[j] = q < cnt ? r0 * 128 : -1;
            ka[j] = c * 8;
            offa[j] = q < cnt && row < rows_m ? static_cast<uint32_t>(row) * static_cast<uint32_t>(a.ldx) * 2u + c * 16
                                              : kOob;
        }
#pragma unroll
        for (int i = 0; i < (h == 0 ? T::IB0 : T::IB1); ++i) {
            const int q = wave + 8 * i, j = h == 0 ? i : T::IB0 + i;
            const int r0 = q / (2 * NB0) * (16 * NB) + h * 16 * NB0 + q % (2 * NB0) * 8;
            const int row = r0 + (lane >> 3);
            const int c = (lane & 7) ^ ((row >> 1) & 7);
            const int n = GATED ? (row >> 5) * 16 + (row & 15) : row;
            dstb[j] = T::AB + r0 * 128;
            kb[j] = c * 8;
            offb[j] = n < rows_n ? static_cast<uint32_t>(n) * static_cast<uint32_t>(a.ldw) * 2u + c * 16 : kOob;
        }
    }
    // (16-row blocks of w and w_up in turn: with four blocks a wave's columns
    // instruction q is of block q / 2 % 2 of a half, with two a half is one block)
    const bool up0 = GATED && NB0 == 2 && ((wave >> 1) & 1);
    const int64_t woff = static_cast<int64_t>(n0) * a.ldw + st0 * 64;
    const int kleft = a.K - st0 * 64;
    // An operand's rows from the next stage to issue on: first byte, and bytes to
    // the end of the last row (nothing past it is read). 3 scalar operations move it
    // a stage on.
    struct Rows {
        const uint16_t* p;
        int bytes;
    };
    Rows xr = {a.x16 + static_cast<int64_t>(m0) * a.ldx + st0 * 64,
               static_cast<int>((static_cast<int64_t>(rows_m - 1) * a.ldx + kleft) * 2)};
    const int wbytes = static_cast<int>((static_cast<int64_t>(rows_n - 1) * a.ldw + kleft) * 2);
    Rows wr[2] = {{(up0 ? a.w_up : a.w) + woff, wbytes}, {(GATED && (NB0 == 1 || up0) ? a.w_up : a.w) + woff, wbytes}};
    const int tail = kleft / 64, tail_k = kleft % 64;  // the stage that K ends inside, and where
    int fill = 0, fill_at = 0;                         // stage to issue next, its slot's offset

    auto issue = [&](const Rows& w, uint32_t off, int k, int dst) {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(w.p), 0, fill < nst ? w.bytes : 0, kRsrcWord3);  // past the range: zeros, unread
        const uint32_t o = k >= (fill == tail ? tail_k : 64) ? kOob : off;
        uint8_t* to = lds + (dst >= 0 ? fill_at + dst : NS * T::STAGE);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)to, 16, o, 0, 0, 0);
    };
    auto issue_a = [&](int h) {
#pragma unroll
        for (int i = 0; i < T::IA0 + T::IA1; ++i)
            if ((i >= T::IA0) == (h == 1)) issue(xr, offa[i], ka[i], dsta[i]);
    };
    auto issue_b = [&](int h) {
#pragma unroll
        for (int i = 0; i < T::IB0 + T::IB1; ++i)
            if ((i >= T::IB0) == (h == 1)) issue(wr[h], offb[i], kb[i], dstb[i]);
    };
    auto next_fill = [&]() {
        xr = {xr.p + 64, xr.bytes - 128};
        wr[0] = {wr[0].p + 64, wr[0].bytes - 128};
        wr[1] = {wr[1].p + 64, wr[1].bytes - 128};
        ++fill;
        fill_at = fill_at + T::STAGE == NS * T::STAGE ? 0 : fill_at + T::STAGE;
    };

    v4f acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    const int r = lane & 15, kq = lane >> 4;
    // fragment of 16-row block `row0`, k-step ks: lane (r, kq) has k 32 ks + 8 kq ..
    const int lane0 = r * 128 + ((kq ^ (r >> 1)) << 4), lane1 = r * 128 + (((kq + 4) ^ (r >> 1)) << 4);
    auto frag = [&](const uint8_t* slot, int row0, int ks) {
        return *reinterpret_cast<const v8bf*>(slot + row0 * 128 + (ks ? lane1 : lane0));
    };
    v8bf fa[MB0][2], fb[2][NB0][2];
    auto mma = [&](auto hm, auto hn) {
        constexpr int HM = decltype(hm)::value, HN = decltype(hn)::value;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < (HM ? MB1 : MB0); ++i)
#pragma unroll
                for (int j = 0; j < NB0; ++j)
                    acc[HM * MB0 + i][HN * NB0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        fb[HN][j][ks], fa[i][ks], acc[HM * MB0 + i][HN * NB0 + j], 0, 0, 0);
        __builtin_amdgcn_s_setprio(0);
    };
    auto barrier = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    using H0 = std::integral_constant<int, 0>;
    using H1 = std::integral_constant<int, 1>;

    // A wave issues a stage's four quarters in the order in which its slot's are
    // free: A0, a B half, the other, A1. Behind its wait before a barrier its share
    // of what the next phases read has landed.
    constexpr int kAhead = (NS - 2) * T::ALL;
    const uint8_t *as, *bs;  // the wave's rows in the slot that is read, which is the one filled behind the reads
    const auto enter = [&]() {
        as = lds + fill_at + wm * (16 * MB) * 128;
        bs = lds + fill_at + T::AB + wn * (16 * NB) * 128;
    };
    const auto read_b = [&](int h) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < NB0; ++j) fb[h][j][ks] = frag(bs, 16 * (h * NB0 + j), ks);
    };
#pragma unroll
    for (int st = 0; st < NS; ++st) {
        issue_a(0);
        issue_b(0);
        issue_b(1);
        issue_a(1);
        next_fill();
    }
    wait_vmcnt<T::IA1 + T::ALL + kAhead>();  // A0, B0, B1 of stage 0
    barrier();
    const bool lag = wave >= 4;
    if (lag) barrier();
    enter();
    read_b(0);
    // One stage, column half F first: its fragments are there already
    const auto stage = [&](auto first, auto second) __attribute__((always_inline)) {
        constexpr int F = decltype(first)::value, S = decltype(second)::value;
        // phase 0: rows 0, columns F
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < MB0; ++i) fa[i][ks] = frag(as, 16 * i, ks);
        wait_lgkmcnt0();
        barrier();
        mma(H0{}, first);
        barrier();
        // phase 1: rows 0, columns S
        read_b(S);
        __builtin_amdgcn_sched_barrier(0);
        issue_a(0);
        issue_b(F);
        wait_vmcnt<T::ALL + T::IA0 + T::IB0 + kAhead>();  // A1
        wait_lgkmcnt0();
        barrier();
        mma(H0{}, second);
        barrier();
        // phase 2: rows 1, columns S
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < MB1; ++i) fa[i][ks] = frag(as, 16 * (MB0 + i), ks);
        __builtin_amdgcn_sched_barrier(0);
        issue_b(S);
        wait_vmcnt<T::ALL + kAhead>();  // A0, B0, B1 of the next stage
        wait_lgkmcnt0();
        barrier();
        mma(H1{}, second);
        barrier();
        // phase 3: rows 1, columns F; the fragments of columns S of the next stage
        issue_a(1);
        next_fill();
        enter();
        read_b(S);
        barrier();
        mma(H1{}, first);
        barrier();
    };
    for (int st = 0; st < nst; st += 2) {
        stage(H0{}, H1{});
        if (st + 1 < nst) stage(H1{}, H0{});
    }
    if (!lag) barrier();
    wait_vmcnt<0>();
    __syncthreads();

    // 16 rows of the wave at a time through LDS, so that a store covers whole
    // lines of a row: lane 4 columns, OL lanes a row
    constexpr int WN = T::TN / 4, WO = GATED ? WN / 2 : WN, OL = WO / 4, RP = 64 / OL;
    float* sh = reinterpret_cast<float*>(lds) + wave * 16 * T::PITCH;
    const int oc = (lane % OL) * 4;  // output column of the wave
    const int n = n0 + wn * WO + oc;
    // staged column of it: GATED: block oc / 16 of w at 32 (oc / 16), of w_up 16 further
    const int sc = GATED ? (oc >> 4) * 32 + (oc & 15) : oc;
    Columns col;
    if (a.splits == 1 && n < a.N) col = load_columns(a, n);
    // Whole groups with a residual: its values are loaded 16 rows ahead. (Loaded
    // beside its use, each waits for the stores before it as well.)
    const auto residual = [&](auto res_bf, auto out_bf) __attribute__((always_inline)) {
        constexpr bool RB = decltype(res_bf)::value, OB = decltype(out_bf)::value;
        using res_t = std::conditional_t<RB, uint2, v4f>;
        using out_t = std::conditional_t<OB, uint2, v4f>;
        const int row0 = m0 + wm * (16 * MB) + lane / OL, at = min(n, a.N - 4);
        const auto load = [&](int i, res_t(&d)[16 / RP]) {
#pragma unroll
            for (int q = 0; q < 16 / RP; ++q) {
                const int64_t m = min(row0 + 16 * i + q * RP, a.M - 1);
                d[q] = *reinterpret_cast<const res_t*>(static_cast<const uint8_t*>(a.residual) +
                                                       (m * a.ldr + at) * (RB ? 2 : 4));
            }
        };
        res_t res[2][16 / RP];
        load(0, res[0]);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            if (i + 1 < MB) load(i + 1, res[(i + 1) & 1]);
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int j = 0; j < NB; ++j) *reinterpret_cast<v4f*>(sh + r * T::PITCH + 16 * j + 4 * kq) = acc[i][j];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < 16 / RP; ++q) {
                const int m = row0 + 16 * i + q * RP;
                const v4f z = *reinterpret_cast<const v4f*>(sh + (q * RP + lane / OL) * T::PITCH + sc);
                v4f u = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (GATED) u = *reinterpret_cast<const v4f*>(sh + (q * RP + lane / OL) * T::PITCH + sc + 16);
                float v[4];
                finish_values<GATED>(a, col, z, u, v);
                if constexpr (RB) {
                    const uint2 t = res[i & 1][q];
                    v[0] += __uint_as_float(t.x << 16);
                    v[1] += __uint_as_float(t.x & 0xffff0000u);
                    v[2] += __uint_as_float(t.y << 16);
                    v[3] += __uint_as_float(t.y & 0xffff0000u);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += res[i & 1][q][e];
                }
                if (m < a.M && n < a.N) {
                    out_t* o = reinterpret_cast<out_t*>(static_cast<uint8_t*>(a.out) + (m * a.ldo + n) * (OB ? 2 : 4));
                    if constexpr (OB)
                        *o = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
                    else
                        *o = (v4f){v[0], v[1], v[2], v[3]};
                }
            }
        }
    };
    if (a.splits == 1 && a.residual != nullptr && a.vec4 && a.N % 4 == 0) {
        const bool rb = a.res_dtype == QIMG_BF16, ob = a.out_dtype == QIMG_BF16;
        if (rb && ob)
            residual(H1{}, H1{});
        else if (rb)
            residual(H1{}, H0{});
        else if (ob)
            residual(H0{}, H1{});
        else
            residual(H0{}, H0{});
        return;
    }
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < NB; ++j) *reinterpret_cast<v4f*>(sh + r * T::PITCH + 16 * j + 4 * kq) = acc[i][j];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < 16 / RP; ++q) {
            const int row = q * RP + lane / OL;
            const int m = m0 + wm * (16 * MB) + 16 * i + row;
            const v4f z = *reinterpret_cast<const v4f*>(sh + row * T::PITCH + sc);
            v4f u = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (GATED) u = *reinterpret_cast<const v4f*>(sh + row * T::PITCH + sc + 16);
            if (m >= a.M || n >= a.N) continue;
            if (a.splits == 1) {
                const float zz[4] = {z[0], z[1], z[2], z[3]}, uu[4] = {u[0], u[1], u[2], u[3]};
                finish4<GATED>(a, col, m, n, zz, uu);
            } else {  // part rows hold the columns padded to four, then w_up's
                float* p = a.part + (static_cast<int64_t>(split) * a.M + m) * a.part_ld + n;
                *reinterpret_cast<v4f*>(p) = z;
                if constexpr (GATED) *reinterpret_cast<v4f*>(p + a.part_ld / 2) = u;
            }
        }
    }
}

// ---- small tiles -----------------------------------------------------------------
// For products of few tiles the eight barriers of a stage above cost more than its
// MFMAs. Here a stage is 128 elements of K (256-byte rows, 4 rows a DMA
// instruction, chunk c of row r at c ^ (r & 15)) with one barrier, and the eight
// waves are two halves of the tile's rows times four quarters of the stage's K, so a
// wave reads each operand byte of its quarter once; the four partial tiles are
// added through LDS in order. A workgroup's time is its operand bytes through
// the CU's port to L2, with NS - 1 stages in flight.
template <int TM_, int TN_>
struct Small {
    static constexpr int TM = TM_, TN = TN_;
    static constexpr int AB = TM * 256, STAGE = AB + TN * 256;
    static constexpr int NS = 152 * 1024 / STAGE < 4 ? 152 * 1024 / STAGE : 4;
    static constexpr int IA = TM / 32, IB = TN / 32, PER = IA + IB;  // DMA instructions per wave and stage
    static constexpr int PITCH = TN + 4;
    static_assert(NS >= 2 && TM % 32 == 0 && TN % 32 == 0, "DMA shares");
    static_assert(4 * TM * PITCH * 4 <= NS * STAGE, "the partial tiles take the ring's place");
};

template <class T, bool GATED>
__global__ __launch_bounds__(512) void linear_small_kernel(LinearFusedArgs a) {
    constexpr int NS = T::NS, TM = T::TM, TN = T::TN, WB = TM / 32, NB = TN / 16;
    constexpr int TNO = GATED ? TN / 2 : TN;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[NS * T::STAGE];
    const int tiles_m = (a.M + TM - 1) / TM, tiles_n = (a.N + TNO - 1) / TNO;
    const int logical = xcd_remap(blockIdx.x, tiles_m * tiles_n * a.splits);
    const int m0 = logical % tiles_m * TM;
    const int n0 = logical / tiles_m % tiles_n * TNO;
    const int split = logical / (tiles_m * tiles_n);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ks = wave & 3, mw = (wave >> 2) * (TM / 2);
    // (split_stages counts stages of 64)
    const int st0 = split * a.split_stages / 2;
    const int nst = min((a.K + 127) / 128 - st0, a.split_stages / 2);

    const int rows_m = min(a.M - m0, TM), rows_n = min(a.N - n0, TNO);
    uint32_t off[T::PER];
    int kc[T::PER];
#pragma unroll
    for (int i = 0; i < T::PER; ++i) {
        const int row = 4 * (wave + 8 * (i < T::IA ? i : i - T::IA)) + (lane >> 4);
        const int c = (lane & 15) ^ (row & 15);
        const int n = GATED ? (row >> 5) * 16 + (row & 15) : row;  // of a weight row: w and w_up, 16 in turn
        kc[i] = 8 * c;
        if (i < T::IA)
            off[i] = row < rows_m ? static_cast<uint32_t>(row) * static_cast<uint32_t>(a.ldx) * 2u + c * 16 : kOob;
        else
            off[i] = n < rows_n ? static_cast<uint32_t>(n) * static_cast<uint32_t>(a.ldw) * 2u + c * 16 : kOob;
    }
    const int kleft = a.K - st0 * 128;
    const uint16_t* xp = a.x16 + static_cast<int64_t>(m0) * a.ldx + st0 * 128;
    const uint16_t* wp = (GATED && wave >= 4 ? a.w_up : a.w) + static_cast<int64_t>(n0) * a.ldw + st0 * 128;
    int xbytes = static_cast<int>((static_cast<int64_t>(rows_m - 1) * a.ldx + kleft) * 2);
    int wbytes = static_cast<int>((static_cast<int64_t>(rows_n - 1) * a.ldw + kleft) * 2);
    const int tail = kleft / 128, tail_k = kleft % 128;
    int fill = 0, fill_at = 0;
    auto issue = [&]() {
        const bool in = fill < nst;  // past the range: zeros, unread
        const __amdgpu_buffer_rsrc_t rx =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(xp), 0, in ? xbytes : 0, kRsrcWord3);
        const __amdgpu_buffer_rsrc_t rw =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(wp), 0, in ? wbytes : 0, kRsrcWord3);
        const int klim = fill == tail ? tail_k : 128;
#pragma unroll
        for (int i = 0; i < T::PER; ++i) {
            const uint32_t o = kc[i] >= klim ? kOob : off[i];
            const int q = wave + 8 * (i < T::IA ? i : i - T::IA);
            uint8_t* to = lds + fill_at + (i < T::IA ? 0 : T::AB) + q * 1024;
            if (i < T::IA)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr_t)to, 16, o, 0, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr_t)to, 16, o, 0, 0, 0);
        }
        xp += 128;
        wp += 128;
        xbytes -= 256;
        wbytes -= 256;
        ++fill;
        fill_at = fill_at + T::STAGE == NS * T::STAGE ? 0 : fill_at + T::STAGE;
    };

    v4f acc[WB][NB];
#pragma unroll
    for (int i = 0; i < WB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    const int r = lane & 15, kq = lane >> 4;
    const int lane_at = r * 256 + (((4 * ks + kq) ^ r) << 4);
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) issue();
    int at = 0;
    for (int st = 0; st < nst; ++st) {
        // this stage has landed in every wave, and every wave is done with the one before, whose
        // slot is filled next
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<(NS - 2) * T::PER>();
        wait_lgkmcnt0();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        issue();
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t* as = lds + at + mw * 256 + lane_at;
        const uint8_t* bs = lds + at + T::AB + lane_at;
        v8bf fa[WB], fb[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) fb[j] = *reinterpret_cast<const v8bf*>(bs + j * 16 * 256);
#pragma unroll
        for (int i = 0; i < WB; ++i) fa[i] = *reinterpret_cast<const v8bf*>(as + i * 16 * 256);
#pragma unroll
        for (int i = 0; i < WB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], acc[i][j], 0, 0, 0);
        at = at + T::STAGE == NS * T::STAGE ? 0 : at + T::STAGE;
    }
    wait_vmcnt<0>();
    __syncthreads();
    float* red = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int i = 0; i < WB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
            *reinterpret_cast<v4f*>(red + (ks * TM + mw + 16 * i + r) * T::PITCH + 16 * j + 4 * kq) = acc[i][j];
    __syncthreads();
    constexpr int GR = TNO / 4;  // groups of four columns a row
    const int oc = static_cast<int>(threadIdx.x) % GR * 4;
    const int n = n0 + oc;
    const int sc = GATED ? (oc >> 4) * 32 + (oc & 15) : oc;
    if (n >= a.N) return;
    Columns col;
    if (a.splits == 1) col = load_columns(a, n);
#pragma unroll
    for (int q = 0; q < (TM * GR + 511) / 512; ++q) {
        const int row = (static_cast<int>(threadIdx.x) + 512 * q) / GR;
        const int m = m0 + row;
        if (row >= TM || m >= a.M) continue;
        float z[4], u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = u[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float* p = red + (w * TM + row) * T::PITCH + sc;
            const v4f t = *reinterpret_cast<const v4f*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] += t[i];
            if constexpr (GATED) {
                const v4f t2 = *reinterpret_cast<const v4f*>(p + 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] += t2[i];
            }
        }
        if (a.splits == 1) {
            finish4<GATED>(a, col, m, n, z, u);
        } else {
            float* p = a.part + (static_cast<int64_t>(split) * a.M + m) * a.part_ld + n;
            *reinterpret_cast<v4f*>(p) = (v4f){z[0], z[1], z[2], z[3]};
            if constexpr (GATED) *reinterpret_cast<v4f*>(p + a.part_ld / 2) = (v4f){u[0], u[1], u[2], u[3]};
        }
    }
}

template <bool GATED>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearFusedArgs a) {
    const int groups = (a.N + 3) / 4;
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (idx >= static_cast<int64_t>(groups) * a.M) return;
    const int m = static_cast<int>(idx / groups), n = static_cast<int>(idx % groups) * 4;
    const Columns col = load_columns(a, n);
    float z[4] = {0.0f, 0.0f, 0.0f, 0.0f}, u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const float* p = a.part + (static_cast<int64_t>(s) * a.M + m) * a.part_ld + n;
        const v4f q = *reinterpret_cast<const v4f*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] += q[i];
        if constexpr (GATED) {
            const v4f t = *reinterpret_cast<const v4f*>(p + a.part_ld / 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] += t[i];
        }
    }
    finish4<GATED>(a, col, m, n, z, u);
}

// ---- up to 16 rows -------------------------------------------------------------
// One workgroup of four waves per 16 output columns; the waves take the 32-k
// steps of K in turn, RD at a time, and read their weights straight into
// fragments (64 bytes of each of 16 rows an instruction, the next ones following
// in the same lines), the next RD steps' loads in flight while these are
// multiplied. The partial tiles are added through LDS in wave order. Bound by
// the weights' bytes: what counts is how many of them are in flight.
constexpr int RW = 4;

template <bool XF32, bool GATED>
__global__ __launch_bounds__(RW * 64, 4) void linear_rows_kernel(LinearFusedArgs a) {
    constexpr int NP = GATED ? 2 : 1, XV = XF32 ? 2 : 1;
    constexpr int RD = NP + XV == 4 ? 2 : 4;  // 128 registers: four workgroups a CU
    __shared__ v4f red[NP][RW][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16;
    const int r = lane & 15, kq = lane >> 4;
    const int rows_n = min(a.N - n0, 16);
    const int64_t wbytes = (static_cast<int64_t>(rows_n - 1) * a.ldw + a.K) * 2;
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(a.w + static_cast<int64_t>(n0) * a.ldw), 0, static_cast<int>(wbytes), kRsrcWord3);
    const __amdgpu_buffer_rsrc_t ru = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(GATED ? a.w_up + static_cast<int64_t>(n0) * a.ldw : a.w), 0,
        GATED ? static_cast<int>(wbytes) : 0, kRsrcWord3);
    constexpr int XE = XF32 ? 4 : 2;
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<void*>(XF32 ? a.x : static_cast<const void*>(a.x16)), 0,
        static_cast<int>((static_cast<int64_t>(a.M - 1) * a.ldx + a.K) * XE), kRsrcWord3);
    // rows past N or M and k past K read as zeros
    const uint32_t ow = r < rows_n ? static_cast<uint32_t>(r) * static_cast<uint32_t>(a.ldw) * 2u + kq * 16 : kOob;
    const uint32_t ox = r < a.M ? static_cast<uint32_t>(r) * static_cast<uint32_t>(a.ldx) * XE + kq * 8 * XE : kOob;

    v4f acc[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) acc[p] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    const int steps = (a.K + 31) / 32;
    v4i fw[2][NP][RD], fx[2][XV][RD];
    auto load = [&](int b, int s0) {
#pragma unroll
        for (int d = 0; d < RD; ++d) {
            const uint32_t bad = (s0 + d) * 32 + 8 * kq < a.K ? 0u : kOob;
            const uint32_t o = (ow + static_cast<uint32_t>(s0 + d) * 64) | (ow & kOob) | bad;
            const uint32_t x = (ox + static_cast<uint32_t>(s0 + d) * (32 * XE)) | (ox & kOob) | bad;
#pragma unroll
            for (int v = 0; v < XV; ++v)
                fx[b][v][d] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rx, x + 16 * v, 0, 0));
            fw[b][0][d] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw, o, 0, 0));
            if constexpr (GATED)
                fw[b][NP - 1][d] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(ru, o, 0, 0));
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](int b) {
#pragma unroll
        for (int d = 0; d < RD; ++d) {
            v8bf x = __builtin_bit_cast(v8bf, fx[b][0][d]);
            if constexpr (XF32) {
                const v4f lo = __builtin_bit_cast(v4f, fx[b][0][d]), hi = __builtin_bit_cast(v4f, fx[b][XV - 1][d]);
                x = __builtin_bit_cast(v8bf, (v4i){static_cast<int>(pack_bf16x2(lo[0], lo[1])),
                                                   static_cast<int>(pack_bf16x2(lo[2], lo[3])),
                                                   static_cast<int>(pack_bf16x2(hi[0], hi[1])),
                                                   static_cast<int>(pack_bf16x2(hi[2], hi[3]))});
            }
#pragma unroll
            for (int p = 0; p < NP; ++p)
                acc[p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, fw[b][p][d]), x, acc[p], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    load(0, wave * RD);
    for (int s0 = wave * RD; s0 < steps; s0 += 2 * RW * RD) {
        load(1, s0 + RW * RD);
        multiply(0);
        load(0, s0 + 2 * RW * RD);
        multiply(1);
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) red[p][wave][lane] = acc[p];
    __syncthreads();
    if (wave != 0) return;
    // lane: row lane % 16, columns 4 (lane / 16) ..
    v4f z = red[0][0][lane], u = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 1; w < RW; ++w) z += red[0][w][lane];
    if constexpr (GATED) {
        u = red[NP - 1][0][lane];
#pragma unroll
        for (int w = 1; w < RW; ++w) u += red[NP - 1][w][lane];
    }
    const int n = n0 + 4 * kq;
    if (r >= a.M || n >= a.N) return;
    const float zz[4] = {z[0], z[1], z[2], z[3]}, uu[4] = {u[0], u[1], u[2], u[3]};
    finish4<GATED>(a, load_columns(a, n), r, n, zz, uu);
}

// ---- one or two rows -------------------------------------------------------------
// A wave takes two weight rows (GATED: one of w and one of w_up) and all of K, 512
// elements an instruction: whole KB reads of one row, eight of them in flight
// for each, products on the vector unit (x rounded to bf16, fp32 sums per lane,
// then over the lanes).
template <bool XF32, bool GATED, int MM>
__global__ __launch_bounds__(256, 2) void linear_gemv_kernel(LinearFusedArgs a) {
    constexpr int U = 8, XE = XF32 ? 4 : 2, XV = XF32 ? 2 : 1;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = (blockIdx.x * 4 + wave) * (GATED ? 1 : 2);
    if (n0 >= a.N) return;
    const int n1 = min(n0 + 1, a.N - 1);
    const int64_t row = static_cast<int64_t>(n0) * a.ldw;
    const __amdgpu_buffer_rsrc_t rw[2] = {
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.w + row), 0, a.K * 2, kRsrcWord3),
        __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(GATED ? a.w_up + row : a.w + static_cast<int64_t>(n1) * a.ldw), 0, a.K * 2, kRsrcWord3)};
    const uint8_t* xb = static_cast<const uint8_t*>(XF32 ? a.x : static_cast<const void*>(a.x16));
    float s[2][MM];
#pragma unroll
    for (int m = 0; m < MM; ++m) s[0][m] = s[1][m] = 0.0f;
    for (int k0 = 0; k0 < a.K; k0 += 512 * U) {
        v4i w[2][U], x[MM][XV][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + 512 * u + 8 * lane;  // past K: out of the row's range, zeros
#pragma unroll
            for (int m = 0; m < MM; ++m) {
                const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
                    const_cast<uint8_t*>(xb + static_cast<int64_t>(m) * a.ldx * XE), 0, a.K * XE, kRsrcWord3);
#pragma unroll
                for (int v = 0; v < XV; ++v)
                    x[m][v][u] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rx, k * XE + 16 * v, 0, 0));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
                w[i][u] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw[i], k * 2, 0, 0));
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int m = 0; m < MM; ++m) {
                uint32_t xp[4];  // eight bf16
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if constexpr (XF32) {
                        const v4f f = __builtin_bit_cast(v4f, x[m][c >> 1][u]);
                        xp[c] = pack_bf16x2(f[2 * (c & 1)], f[2 * (c & 1) + 1]);
                    } else {
                        xp[c] = static_cast<uint32_t>(x[m][0][u][c]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t wp = static_cast<uint32_t>(w[i][u][c]);
                        s[i][m] = __builtin_fmaf(__uint_as_float(xp[c] << 16), __uint_as_float(wp << 16), s[i][m]);
                        s[i][m] = __builtin_fmaf(__uint_as_float(xp[c] & 0xffff0000u), __uint_as_float(wp & 0xffff0000u),
                                                 s[i][m]);
                    }
            }
    }
#pragma unroll
    for (int m = 0; m < MM; ++m) {
        s[0][m] = wave_sum_dpp(s[0][m]);
        s[1][m] = wave_sum_dpp(s[1][m]);
    }
    // lane: row lane / 2, column lane % 2 of the wave's
    const int m = lane >> 1, c = GATED ? 0 : lane & 1;
    if (m >= MM || n0 + c >= a.N || (GATED && (lane & 1))) return;
    float z = s[0][0], u = s[1][0];
    if constexpr (MM == 2) {
        z = m ? s[0][1] : z;
        u = m ? s[1][1] : u;
    }
    if (!GATED && c) z = u;
    finish1<GATED>(a, m, n0 + c, z, u);
}

// rows of K values, fp32 or bf16, to bf16 rows of Kp >= K (a multiple of 8),
// zeros behind K: eight values a thread
template <bool F32>
__global__ __launch_bounds__(256) void pack_rows_kernel(const void* __restrict__ in, int64_t ld, int64_t rows, int K,
                                                        int Kp, uint16_t* __restrict__ out) {
    const int per = Kp / 8;
    for (int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; idx < rows * per;
         idx += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = idx / per;
        const int k = static_cast<int>(idx % per) * 8;
        const float* f = static_cast<const float*>(in) + row * ld + k;
        const uint16_t* h = static_cast<const uint16_t*>(in) + row * ld + k;
        uint32_t w[4];
        if (F32 && k + 8 <= K && (reinterpret_cast<uintptr_t>(f) & 15) == 0) {
            const v4f lo = *reinterpret_cast<const v4f*>(f), hi = *reinterpret_cast<const v4f*>(f + 4);
            w[0] = pack_bf16x2(lo[0], lo[1]);
            w[1] = pack_bf16x2(lo[2], lo[3]);
            w[2] = pack_bf16x2(hi[0], hi[1]);
            w[3] = pack_bf16x2(hi[2], hi[3]);
        } else {
            uint16_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k + i < K ? (F32 ? f32_to_bf16(f[i]) : h[i]) : static_cast<uint16_t>(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = v[2 * i] | (static_cast<uint32_t>(v[2 * i + 1]) << 16);
        }
        *reinterpret_cast<u32x4*>(out + row * Kp + k) = (u32x4){w[0], w[1], w[2], w[3]};
    }
}

hipError_t launch_pack(const void* in, bool f32, int64_t ld, int64_t rows, int K, int Kp, uint16_t* out,
                       hipStream_t stream) {
    const int64_t want = (rows * (Kp / 8) + 255) / 256, most = 1 << 22;  // (a grid has less than 2^32 threads)
    const dim3 grid(static_cast<unsigned>(want < most ? want : most));
    if (f32)
        hipLaunchKernelGGL(pack_rows_kernel<true>, grid, dim3(256), 0, stream, in, ld, rows, K, Kp, out);
    else
        hipLaunchKernelGGL(pack_rows_kernel<false>, grid, dim3(256), 0, stream, in, ld, rows, K, Kp, out);
    return hipGetLastError();
}

template <int TM, int TN, bool GATED>
hipError_t launch_tile(const LinearFusedArgs& a, hipStream_t stream) {
    constexpr int TNO = GATED ? TN / 2 : TN;
    const int tiles = ((a.M + TM - 1) / TM) * ((a.N + TNO - 1) / TNO);
    hipLaunchKernelGGL((linear_tile_kernel<Tile<TM, TN>, GATED>), dim3(tiles * a.splits), dim3(512), 0, stream, a);
    return hipGetLastError();
}

template <int TM, int TN, bool GATED>
hipError_t launch_small(const LinearFusedArgs& a, hipStream_t stream) {
    constexpr int TNO = GATED ? TN / 2 : TN;
    const int tiles = ((a.M + TM - 1) / TM) * ((a.N + TNO - 1) / TNO);
    hipLaunchKernelGGL((linear_small_kernel<Small<TM, TN>, GATED>), dim3(tiles * a.splits), dim3(512), 0, stream, a);
    return hipGetLastError();
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace

// Kernel, tile and number of K splits: the least estimated time of the launch
// (us). A stage of linear_tile_kernel takes 0.4 us and 1.2 us for each 256x256 of
// the tile (measured: 256x256 1.6, 224x256 1.5, 160x256 1.2, 128x128 0.7), one of
// linear_small_kernel its bytes at 75 KB a us; the weights come at 4.8 TB/s at
// best, the parts of a split sum are written and read once, mostly in the caches.
// linear_rows_kernel takes about 4 us and the weights' bytes at 2.5 TB/s; fp32 rows
// spare it a packing launch of 3 us. Measured (us, bf16 x, weights not resident):
// 16x3584x3584 rows 10.8, 32x64 tiles 13; 16x4608x3584 17.5 / 11.7; 21x3584x14336
// 32x64 split in 4 25, 32x128 in 9 26; 269x4608x3584 96x64 tiles 20.5, 160x256 split
// in 4 28; 269x3584x14336 160x256 split in 9 45-49, 96x64 split in 4 72;
// 281x3584x12288 160x256 split in 9 45, 96x64 split in 3 56; 500x4608x3584 128x256
// split in 3 36, 96x64 38; 930x4608x3584 160x256 split in 2 49, 96x64 56;
// 1672x3584x3584 192x256 split in 2 58, 128x256 65; 781x14336x3584 gated 224x256 158,
// 256x256 162; 64x14336x3584 gated 64x128 43. Not always the best: 2605x3584x12288
// 224x256 split in 3 218, 160x256 215.
LinearFusedPlan linear_fused_plan(int x_dtype, int M, int K, int N, bool gated) {
    LinearFusedPlan best{};  // tm = 0: linear_gemv_kernel or linear_rows_kernel
    if (M <= kLinearGemvRows) return best;
    const double bytes = 2.0 * N * K * (gated ? 2 : 1);  // of weights
    double best_t = M <= kLinearRows ? 4.0 + bytes / 2.5e6 - (x_dtype == QIMG_FP32 ? 3.0 : 0.0) : 1e30;
    static const struct {
        int tm, tn, k;  // k: elements of K a stage
    } shapes[] = {{256, 256, 64}, {224, 256, 64}, {192, 256, 64}, {160, 256, 64}, {128, 256, 64}, {128, 128, 64},
                  {128, 64, 128}, {96, 64, 128},  {64, 128, 128}, {64, 64, 128},  {32, 128, 128}, {32, 64, 128}};
    for (const auto& c : shapes) {
        const int tno = gated ? c.tn / 2 : c.tn;
        const int64_t tiles = static_cast<int64_t>((M + c.tm - 1) / c.tm) * ((N + tno - 1) / tno);
        const int stages = (K + c.k - 1) / c.k;
        const double stage =
            c.k == 64 ? 0.4 + 1.2 * c.tm * c.tn / 65536.0 : (c.tm + c.tn) * 256 / 75e3;
        for (int s = 1; s <= 16 && s <= stages && tiles * (s - 1) < 512; ++s) {  // (past two rounds no split gains)
            const int per = (stages + s - 1) / s;
            if (per * (s - 1) >= stages) continue;  // the last range would be empty
            const double rounds = static_cast<double>((tiles * s + 255) / 256);
            const double work = rounds * (per * stage + (c.k == 64 ? 3.0 : 1.5)), read = bytes / 4.8e6 + 3.0;
            double t = 3.0 + std::max(work, read) + 0.2 * std::min(work, read);
            if (s > 1) t += 4.0 + 0.3 * s + 2.0 * s * M * N * (gated ? 8.0 : 4.0) / 10e6;
            if (t < best_t) {
                best_t = t;
                best.tm = c.tm;
                best.tn = c.tn;
                best.small = c.k == 128;
                best.splits = s;
                best.split_stages = per * (c.k / 64);
            }
        }
    }
    return best;
}

// Scratch: packed x, packed w and w_up, the parts of a split sum.
LinearFusedScratch linear_fused_scratch(const LinearFusedPlan& p, int x_dtype, int M, int K, int N, bool gated) {
    LinearFusedScratch s{};
    if (M <= 0 || K <= 0 || N <= 0) return s;
    const int Kp = (K + 7) / 8 * 8;
    const bool odd = Kp != K;
    if (odd || (x_dtype == QIMG_FP32 && p.tm != 0)) s.x = align256(static_cast<int64_t>(M) * Kp * 2);
    if (odd) s.w = align256(static_cast<int64_t>(N) * Kp * 2);
    if (odd && gated) s.w_up = s.w;
    if (p.splits > 1) s.part = align256(static_cast<int64_t>(p.splits) * M * ((N + 3) / 4 * 4) * (gated ? 8 : 4));
    return s;
}

hipError_t launch_linear_fused(LinearFusedArgs a, const LinearFusedPlan& plan, int x_dtype, void* scratch,
                               hipStream_t stream) {
    const bool gated = a.w_up != nullptr;
    const LinearFusedScratch s = linear_fused_scratch(plan, x_dtype, a.M, a.K, a.N, gated);
    uint8_t* p = static_cast<uint8_t*>(scratch);
    const int Kp = (a.K + 7) / 8 * 8;
    bool f32 = x_dtype == QIMG_FP32;
    hipError_t e = hipSuccess;
    a.x16 = static_cast<const uint16_t*>(a.x);
    a.ldw = a.K;
    if (s.x) {
        uint16_t* xp = reinterpret_cast<uint16_t*>(p);
        e = launch_pack(a.x, f32, a.ldx, a.M, a.K, Kp, xp, stream);
        if (e != hipSuccess) return e;
        a.x = a.x16 = xp;
        a.ldx = Kp;
        f32 = false;
        p += s.x;
    }
    for (int i = 0; i < 2; ++i) {
        if (!(i ? s.w_up : s.w)) continue;
        uint16_t* wp = reinterpret_cast<uint16_t*>(p);
        e = launch_pack(i ? a.w_up : a.w, false, a.K, a.N, a.K, Kp, wp, stream);
        if (e != hipSuccess) return e;
        (i ? a.w_up : a.w) = wp;
        p += i ? s.w_up : s.w;
    }
    if (s.w) a.ldw = a.K = Kp;
    a.part = reinterpret_cast<float*>(p);
    a.part_ld = static_cast<int64_t>((a.N + 3) / 4 * 4) * (gated ? 2 : 1);
    if (plan.tm == 0) {
        a.splits = 1;
        if (a.M <= kLinearGemvRows) {
            const dim3 grid(gated ? (a.N + 3) / 4 : (a.N + 7) / 8), block(256);
#define QIMG_GEMV(F32, GATED)                                                                        \
    if (f32 == F32 && gated == GATED) {                                                              \
        if (a.M == 1)                                                                                \
            hipLaunchKernelGGL((linear_gemv_kernel<F32, GATED, 1>), grid, block, 0, stream, a);      \
        else                                                                                         \
            hipLaunchKernelGGL((linear_gemv_kernel<F32, GATED, 2>), grid, block, 0, stream, a);      \
    }
            QIMG_GEMV(true, true)
            QIMG_GEMV(true, false)
            QIMG_GEMV(false, true)
            QIMG_GEMV(false, false)
#undef QIMG_GEMV
            return hipGetLastError();
        }
        const dim3 grid((a.N + 15) / 16), block(RW * 64);
        if (f32 && gated)
            hipLaunchKernelGGL((linear_rows_kernel<true, true>), grid, block, 0, stream, a);
        else if (f32)
            hipLaunchKernelGGL((linear_rows_kernel<true, false>), grid, block, 0, stream, a);
        else if (gated)
            hipLaunchKernelGGL((linear_rows_kernel<false, true>), grid, block, 0, stream, a);
        else
            hipLaunchKernelGGL((linear_rows_kernel<false, false>), grid, block, 0, stream, a);
        return hipGetLastError();
    }
    a.splits = plan.splits;
    a.split_stages = plan.split_stages;
#define QIMG_TILE(TM, TN)                                                                       \
    if (!plan.small && plan.tm == TM && plan.tn == TN)                                          \
    e = gated ? launch_tile<TM, TN, true>(a, stream) : launch_tile<TM, TN, false>(a, stream)
    QIMG_TILE(256, 256);
    QIMG_TILE(224, 256);
    QIMG_TILE(192, 256);
    QIMG_TILE(160, 256);
    QIMG_TILE(128, 256);
    QIMG_TILE(128, 128);
#undef QIMG_TILE
#define QIMG_TILE(TM, TN)                                                                       \
    if (plan.small && plan.tm == TM && plan.tn == TN)                                           \
    e = gated ? launch_small<TM, TN, true>(a, stream) : launch_small<TM, TN, false>(a, stream)
    QIMG_TILE(128, 64);
    QIMG_TILE(96, 64);
    QIMG_TILE(64, 128);
    QIMG_TILE(64, 64);
    QIMG_TILE(32, 128);
    QIMG_TILE(32, 64);
#undef QIMG_TILE
    if (e != hipSuccess || plan.splits == 1) return e;
    const int64_t groups = static_cast<int64_t>((a.N + 3) / 4) * a.M;
    const dim3 grid(static_cast<unsigned>((groups + 255) / 256));
    if (gated)
        hipLaunchKernelGGL(linear_join_kernel<true>, grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(linear_join_kernel<false>, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace qimg
