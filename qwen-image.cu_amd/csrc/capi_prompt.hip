// capi_prompt.hip — C entry points of the operators around a prompt: argument
// checks on the host, then the launches.
#include <cmath>

#include "capi_checks.h"

extern "C" {

int64_t qimg_attention_varlen_scratch_bytes(int total_q, int total_k, int batch, int n_heads, int n_kv_heads,
                                            int head_dim, int causal) {
    if (total_q <= 0 || total_k <= 0 || batch <= 0 || n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 ||
        n_heads % n_kv_heads != 0)
        return 0;
    const int64_t rows =
        qimg::attn_varlen_plan(total_q, total_k, batch, n_heads, n_kv_heads, head_dim, causal != 0).part_rows;
    return align256(rows * head_dim * 4) + align256(rows * 8);
}

int qimg_attention_varlen(const qimg_attn_varlen* args, void* scratch, int64_t scratch_bytes, void* stream) {
    const char* fn = "qimg_attention_varlen";
    QIMG_REQUIRE(args, "%s: args is null", fn);
    const qimg_attn_varlen& p = *args;
    QIMG_REQUIRE(p.dtype == QIMG_BF16 || p.dtype == QIMG_FP16, "%s: dtype %d must be BF16 or FP16", fn, p.dtype);
    QIMG_REQUIRE(p.batch >= 0 && p.total_q >= 0 && p.total_k >= 0, "%s: bad sizes batch=%d total_q=%d total_k=%d", fn,
                 p.batch, p.total_q, p.total_k);
    QIMG_REQUIRE(p.n_heads > 0 && p.n_kv_heads > 0 && p.n_heads % p.n_kv_heads == 0,
                 "%s: n_heads %d must be a multiple of n_kv_heads %d", fn, p.n_heads, p.n_kv_heads);
    if (p.head_dim != 64 && p.head_dim != 128)
        return qimg::api_fail(QIMG_ERR_UNSUPPORTED, "%s: head_dim %d not supported (64 or 128)", fn, p.head_dim);
    const float scale_log2 = p.sm_scale * 1.4426950408889634f;
    QIMG_REQUIRE(std::isfinite(scale_log2) && scale_log2 > 0.0f, "%s: sm_scale must be positive and finite", fn);
    QIMG_REQUIRE(static_cast<int64_t>(p.total_q) * p.n_heads < (int64_t{1} << 30) && p.total_k < (1 << 30) &&
                     p.batch < (1 << 30),
                 "%s: total_q * n_heads, total_k and batch must be < 2^30", fn);
    QIMG_REQUIRE(good_strides(p.q_stride_t, p.q_stride_h) && good_strides(p.k_stride_t, p.k_stride_h) &&
                     good_strides(p.v_stride_t, p.v_stride_h) && good_strides(p.out_stride_t, p.out_stride_h),
                 "%s: strides must be non-negative multiples of 8, token strides at most 2^24", fn);
    if (p.batch == 0 || p.total_q == 0) return QIMG_OK;
    QIMG_REQUIRE(p.q && p.out && p.cu_seqlens_q && p.cu_seqlens_k, "%s: null pointer", fn);
    QIMG_REQUIRE(p.total_k == 0 || (p.k && p.v), "%s: null pointer", fn);
    QIMG_REQUIRE(aligned16(p.q) && aligned16(p.k) && aligned16(p.v) && aligned16(p.out),
                 "%s: q, k, v and out must be 16-byte aligned", fn);
    QIMG_REQUIRE(p.out != p.q && p.out != p.k && p.out != p.v, "%s: out must not be q, k or v", fn);
    QIMG_REQUIRE(p.total_k <= 1 || (p.k_stride_t >= p.head_dim && p.v_stride_t >= p.head_dim),
                 "%s: k and v token strides must be at least head_dim", fn);
    QIMG_REQUIRE(apart(p.total_q, p.out_stride_t, p.n_heads, p.out_stride_h, p.head_dim),
                 "%s: out strides must keep its tokens and heads apart", fn);
    qimg::AttnVarlenArgs a{};
    a.q = static_cast<const uint16_t*>(p.q);
    a.k = static_cast<const uint16_t*>(p.k);
    a.v = static_cast<const uint16_t*>(p.v);
    a.out = static_cast<uint16_t*>(p.out);
    a.q_t = p.q_stride_t, a.q_h = p.q_stride_h, a.k_t = p.k_stride_t, a.k_h = p.k_stride_h;
    a.v_t = p.v_stride_t, a.v_h = p.v_stride_h, a.o_t = p.out_stride_t, a.o_h = p.out_stride_h;
    a.cu_q = p.cu_seqlens_q, a.cu_k = p.cu_seqlens_k, a.k_lens = p.k_lens;
    a.batch = p.batch, a.total_q = p.total_q, a.total_k = p.total_k;
    a.hq = p.n_heads, a.hk = p.n_kv_heads, a.group = p.n_heads / p.n_kv_heads;
    a.causal = p.causal != 0;
    a.scale_log2 = scale_log2;
    const qimg::AttnVarlenPlan plan =
        qimg::attn_varlen_plan(p.total_q, p.total_k, p.batch, p.n_heads, p.n_kv_heads, p.head_dim, a.causal);
    a.many = plan.many, a.groups = plan.groups, a.splits = plan.splits;
    a.tail = plan.tail, a.tail_tiles = plan.tail_tiles;
    if (a.splits > 1) {
        const int64_t bytes_o = align256(plan.part_rows * p.head_dim * 4);
        const int64_t need = bytes_o + align256(plan.part_rows * 8);
        if (!scratch || scratch_bytes < need)
            return qimg::api_fail(QIMG_ERR_SCRATCH, "%s: scratch %lld bytes < required %lld", fn,
                                  static_cast<long long>(scratch_bytes), static_cast<long long>(need));
        QIMG_REQUIRE(aligned16(scratch), "%s: scratch must be 16-byte aligned", fn);
        a.part_o = static_cast<float*>(scratch);
        a.part_ml = a.part_o + bytes_o / 4;
    }
    return qimg::api_hip_status(
        qimg::launch_attention_varlen(a, p.dtype, p.head_dim, static_cast<hipStream_t>(stream)), fn);
}

int64_t qimg_linear_bf16_fused_scratch_bytes(int x_dtype, int M, int K, int N, int gated) {
    if (M <= 0 || K <= 0 || N <= 0) return 0;
    const qimg::LinearFusedPlan plan = qimg::linear_fused_plan(x_dtype, M, K, N, gated != 0);
    const qimg::LinearFusedScratch s = qimg::linear_fused_scratch(plan, x_dtype, M, K, N, gated != 0);
    return s.x + s.w + s.w_up + s.part;
}

int qimg_linear_bf16_fused(const qimg_linear_fused* args, void* scratch, int64_t scratch_bytes, void* stream) {
    const char* fn = "qimg_linear_bf16_fused";
    QIMG_REQUIRE(args, "%s: args is null", fn);
    const qimg_linear_fused& p = *args;
    const auto float_type = [](int t) { return t == QIMG_FP32 || t == QIMG_BF16; };
    QIMG_REQUIRE(float_type(p.x_dtype), "%s: x_dtype %d must be FP32 or BF16", fn, p.x_dtype);
    QIMG_REQUIRE(float_type(p.out_dtype), "%s: out_dtype %d must be FP32 or BF16", fn, p.out_dtype);
    QIMG_REQUIRE(!p.residual || float_type(p.residual_dtype), "%s: residual_dtype %d must be FP32 or BF16", fn,
                 p.residual_dtype);
    QIMG_REQUIRE(p.act >= QIMG_ACT_NONE && p.act <= QIMG_ACT_SILU, "%s: unknown activation %d", fn, p.act);
    QIMG_REQUIRE(p.M >= 0 && p.N >= 0 && p.K > 0, "%s: bad sizes M=%d N=%d K=%d", fn, p.M, p.N, p.K);
    if (p.M == 0 || p.N == 0) return QIMG_OK;
    QIMG_REQUIRE(p.x && p.w && p.out, "%s: null pointer", fn);
    QIMG_REQUIRE(!p.bias_up || p.w_up, "%s: bias_up without w_up", fn);
    QIMG_REQUIRE(aligned16(p.x) && aligned16(p.w) && aligned16(p.w_up) && aligned16(p.out) && aligned16(p.residual),
                 "%s: x, w, w_up, residual and out must be 16-byte aligned", fn);
    const int64_t most = int64_t{1} << 22;
    QIMG_REQUIRE(p.K < most && p.N < most && p.M < (1 << 24), "%s: sizes M=%d N=%d K=%d too large", fn, p.M, p.N, p.K);
    QIMG_REQUIRE(static_cast<int64_t>(p.M / 64 + 1) * (p.N / 64 + 1) < (int64_t{1} << 26), "%s: M=%d N=%d too large", fn,
                 p.M, p.N);
    QIMG_REQUIRE(p.ldx >= p.K && p.ldx < most, "%s: ldx %lld must be at least K and below 2^22", fn,
                 static_cast<long long>(p.ldx));
    QIMG_REQUIRE(p.ldo >= p.N && p.ldo < most, "%s: ldo %lld must be at least N and below 2^22", fn,
                 static_cast<long long>(p.ldo));
    QIMG_REQUIRE(!p.residual || (p.ld_residual >= p.N && p.ld_residual < most),
                 "%s: ld_residual %lld must be at least N and below 2^22", fn, static_cast<long long>(p.ld_residual));
    if (p.K % 8 == 0)
        QIMG_REQUIRE(p.ldx % (p.x_dtype == QIMG_FP32 ? 4 : 8) == 0, "%s: rows of x must be 16-byte aligned (ldx %lld)",
                     fn, static_cast<long long>(p.ldx));
    QIMG_REQUIRE(p.out != p.residual || (p.ldo == p.ld_residual && p.out_dtype == p.residual_dtype),
                 "%s: out in residual's place must have its type and rows", fn);
    QIMG_REQUIRE(p.out != p.x && p.out != static_cast<const void*>(p.w) && p.out != static_cast<const void*>(p.w_up),
                 "%s: out must not be x or a weight", fn);
    const qimg::LinearFusedPlan plan = qimg::linear_fused_plan(p.x_dtype, p.M, p.K, p.N, p.w_up != nullptr);
    const qimg::LinearFusedScratch parts =
        qimg::linear_fused_scratch(plan, p.x_dtype, p.M, p.K, p.N, p.w_up != nullptr);
    const int64_t need = parts.x + parts.w + parts.w_up + parts.part;
    if (need > 0) {
        if (!scratch || scratch_bytes < need)
            return qimg::api_fail(QIMG_ERR_SCRATCH, "%s: scratch %lld bytes < required %lld", fn,
                                  static_cast<long long>(scratch_bytes), static_cast<long long>(need));
        QIMG_REQUIRE(aligned16(scratch), "%s: scratch must be 16-byte aligned", fn);
    }
    qimg::LinearFusedArgs a{};
    a.x = p.x, a.ldx = p.ldx, a.w = p.w, a.w_up = p.w_up;
    a.M = p.M, a.N = p.N, a.K = p.K;
    a.bias = p.bias, a.bias_up = p.bias_up, a.gate = p.gate;
    a.residual = p.residual, a.ldr = p.ld_residual, a.res_dtype = p.residual_dtype;
    a.out = p.out, a.ldo = p.ldo, a.out_dtype = p.out_dtype;
    a.act = p.act;
    a.vec4 = p.ldo % 4 == 0 && (!p.residual || p.ld_residual % 4 == 0);
    return qimg::api_hip_status(qimg::launch_linear_fused(a, plan, p.x_dtype, scratch, static_cast<hipStream_t>(stream)),
                                fn);
}

int qimg_rope_packed(const qimg_rope* args, void* stream) {
    const char* fn = "qimg_rope_packed";
    QIMG_REQUIRE(args, "%s: args is null", fn);
    const qimg_rope& p = *args;
    const auto float_type = [](int t) { return t == QIMG_FP32 || t == QIMG_BF16 || t == QIMG_FP16; };
    QIMG_REQUIRE(float_type(p.x_dtype) && float_type(p.out_dtype), "%s: dtypes %d and %d must be FP32, BF16 or FP16", fn,
                 p.x_dtype, p.out_dtype);
    QIMG_REQUIRE(p.tokens >= 0 && p.n_heads >= 0 && p.n_rotated >= 0 && p.n_rotated <= p.n_heads && p.table_rows >= 0,
                 "%s: bad sizes tokens=%d n_heads=%d n_rotated=%d table_rows=%d", fn, p.tokens, p.n_heads, p.n_rotated,
                 p.table_rows);
    QIMG_REQUIRE(p.head_dim > 0 && p.rotary_dim > 0 && p.rotary_dim <= p.head_dim,
                 "%s: need 0 < rotary_dim <= head_dim (rotary_dim=%d head_dim=%d)", fn, p.rotary_dim, p.head_dim);
    if (p.head_dim % 8 != 0 || p.rotary_dim % 8 != 0)
        return qimg::api_fail(QIMG_ERR_UNSUPPORTED, "%s: head_dim %d and rotary_dim %d must be multiples of 8", fn,
                              p.head_dim, p.rotary_dim);
    QIMG_REQUIRE(good_strides(p.x_stride_t, p.x_stride_h) && good_strides(p.out_stride_t, p.out_stride_h),
                 "%s: strides must be non-negative multiples of 8, token strides at most 2^24", fn);
    if (p.tokens == 0 || p.n_heads == 0) return QIMG_OK;
    QIMG_REQUIRE(p.x && p.out && p.positions && (p.cos_sin || p.table_rows == 0), "%s: null pointer", fn);
    QIMG_REQUIRE(aligned16(p.x) && aligned16(p.out) && aligned16(p.cos_sin),
                 "%s: x, out and cos_sin must be 16-byte aligned", fn);
    QIMG_REQUIRE(apart(p.tokens, p.out_stride_t, p.n_heads, p.out_stride_h, p.head_dim),
                 "%s: out strides must keep its tokens and heads apart", fn);
    QIMG_REQUIRE(p.out != p.x || (p.out_dtype == p.x_dtype && p.out_stride_t == p.x_stride_t &&
                                  p.out_stride_h == p.x_stride_h),
                 "%s: out in x's place must have its type and strides", fn);
    qimg::RopeArgs a{};
    a.x = p.x, a.out = p.out;
    a.x_t = p.x_stride_t, a.x_h = p.x_stride_h, a.o_t = p.out_stride_t, a.o_h = p.out_stride_h;
    a.tokens = p.tokens, a.h = p.n_heads, a.h_rot = p.n_rotated, a.d = p.head_dim, a.r = p.rotary_dim;
    a.interleaved = p.interleaved != 0;
    a.table = p.cos_sin, a.table_rows = p.table_rows, a.positions = p.positions;
    return qimg::api_hip_status(
        qimg::launch_rope_packed(a, p.x_dtype, p.out_dtype, static_cast<hipStream_t>(stream)), fn);
}

}  // extern "C"
