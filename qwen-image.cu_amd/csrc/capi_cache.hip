// capi_cache.hip — C entry points of the operators around a quantized key/value
// cache: argument checks on the host, then the launches.
#include <cmath>

#include "capi_checks.h"

namespace {

// what a cache may have
bool page_sizes(int n) { return n >= 16 && n <= 256 && (n & (n - 1)) == 0; }
bool head_dims(int d) { return d == 64 || d == 128; }
bool kv_heads(int n) { return n > 0 && n < (1 << 16); }

int check_cache(const char* fn, const qimg_kv_cache* c, bool data) {
    QIMG_REQUIRE(c, "%s: cache is null", fn);
    QIMG_REQUIRE(c->dtype == QIMG_INT8 || c->dtype == QIMG_FP8_E4M3, "%s: cache dtype %d must be INT8 or FP8_E4M3", fn,
                 c->dtype);
    QIMG_REQUIRE(c->n_pages >= 0 && c->n_kv_heads > 0, "%s: bad cache sizes n_pages=%d n_kv_heads=%d", fn, c->n_pages,
                 c->n_kv_heads);
    if (!page_sizes(c->page_size))
        return qimg::api_fail(QIMG_ERR_UNSUPPORTED, "%s: page_size %d not supported (16, 32, 64, 128 or 256)", fn,
                              c->page_size);
    if (!head_dims(c->head_dim))
        return qimg::api_fail(QIMG_ERR_UNSUPPORTED, "%s: head_dim %d of a cache not supported (64 or 128)", fn,
                              c->head_dim);
    QIMG_REQUIRE(static_cast<int64_t>(c->n_pages) * c->page_size < (int64_t{1} << 31) && kv_heads(c->n_kv_heads),
                 "%s: n_pages * page_size must be < 2^31, n_kv_heads < 2^16", fn);
    if (!data || c->n_pages == 0) return QIMG_OK;
    QIMG_REQUIRE(c->k && c->v && c->k_exp && c->v_exp, "%s: null pointer in the cache", fn);
    QIMG_REQUIRE(aligned16(c->k) && aligned16(c->v) && aligned16(c->k_exp) && aligned16(c->v_exp),
                 "%s: the cache's codes and exponents must be 16-byte aligned", fn);
    return QIMG_OK;
}

int page_shift(const qimg_kv_cache& c) { return __builtin_ctz(static_cast<unsigned>(c.page_size)); }

bool float_type(int t) { return t == QIMG_FP32 || t == QIMG_BF16 || t == QIMG_FP16; }

// What qimg_norm_rope_packed and qimg_norm_rope_cache share; `heads` of x, `out_heads` of out.
int check_heads(const char* fn, const qimg_norm_rope& p, int64_t heads, int out_heads) {
    QIMG_REQUIRE(float_type(p.x_dtype) && float_type(p.out_dtype), "%s: dtypes %d and %d must be FP32, BF16 or FP16", fn,
                 p.x_dtype, p.out_dtype);
    QIMG_REQUIRE(p.tokens >= 0 && p.n_q_heads >= 0 && p.n_kv_heads >= 0, "%s: bad sizes tokens=%d n_q_heads=%d n_kv_heads=%d",
                 fn, p.tokens, p.n_q_heads, p.n_kv_heads);
    QIMG_REQUIRE(static_cast<int64_t>(p.tokens) * heads < (int64_t{1} << 30) && heads < (1 << 24),
                 "%s: tokens * heads must be < 2^30", fn);
    if (p.head_dim <= 0 || p.head_dim > 256 || p.head_dim % 8 != 0)
        return qimg::api_fail(QIMG_ERR_UNSUPPORTED, "%s: head_dim %d not supported (a multiple of 8 up to 256)", fn,
                              p.head_dim);
    QIMG_REQUIRE(!p.q_norm && !p.k_norm ? true : std::isfinite(p.eps) && p.eps >= 0.0f,
                 "%s: eps must be finite and not negative", fn);
    QIMG_REQUIRE(p.table_rows >= 0, "%s: bad sizes table_rows=%d", fn, p.table_rows);
    if (p.cos_sin) {
        QIMG_REQUIRE(p.rotary_dim > 0 && p.rotary_dim <= p.head_dim,
                     "%s: need 0 < rotary_dim <= head_dim (rotary_dim=%d head_dim=%d)", fn, p.rotary_dim, p.head_dim);
        if (p.rotary_dim % 8 != 0)
            return qimg::api_fail(QIMG_ERR_UNSUPPORTED, "%s: rotary_dim %d must be a multiple of 8", fn, p.rotary_dim);
    }
    QIMG_REQUIRE(good_strides(p.x_stride_t, p.x_stride_h) && good_strides(p.out_stride_t, p.out_stride_h),
                 "%s: strides must be non-negative multiples of 8, token strides at most 2^24", fn);
    if (p.tokens == 0 || heads == 0) return QIMG_OK;
    QIMG_REQUIRE(p.x && (p.out || out_heads == 0) && (!p.cos_sin || p.positions), "%s: null pointer", fn);
    QIMG_REQUIRE(aligned16(p.x) && aligned16(p.out) && aligned16(p.cos_sin) && aligned16(p.q_norm) && aligned16(p.k_norm),
                 "%s: x, out, cos_sin, q_norm and k_norm must be 16-byte aligned", fn);
    if (out_heads > 0) {
        QIMG_REQUIRE(apart(p.tokens, p.out_stride_t, out_heads, p.out_stride_h, p.head_dim),
                     "%s: out strides must keep its tokens and heads apart", fn);
        QIMG_REQUIRE(p.out != p.x || (p.out_dtype == p.x_dtype && p.out_stride_t == p.x_stride_t &&
                                      p.out_stride_h == p.x_stride_h),
                     "%s: out in x's place must have its type and strides", fn);
    }
    return QIMG_OK;
}

qimg::HeadsArgs heads_args(const qimg_norm_rope& p) {
    qimg::HeadsArgs a{};
    a.x = p.x, a.out = p.out, a.out_dtype = p.out_dtype;
    a.x_t = p.x_stride_t, a.x_h = p.x_stride_h, a.o_t = p.out_stride_t, a.o_h = p.out_stride_h;
    a.tokens = p.tokens, a.nq = p.n_q_heads, a.nk = p.n_kv_heads, a.d = p.head_dim;
    a.r = p.cos_sin ? p.rotary_dim : 0, a.interleaved = p.interleaved != 0;
    a.wq = p.q_norm, a.wk = p.k_norm, a.eps = p.eps;
    a.table = p.cos_sin, a.table_rows = p.table_rows, a.positions = p.positions;
    return a;
}

void put_cache(qimg::HeadsArgs& a, const qimg_kv_cache& c, const int32_t* slots) {
    a.ck = c.k, a.cv = c.v, a.cke = c.k_exp, a.cve = c.v_exp;
    a.page_shift = page_shift(c), a.n_slots = c.n_pages * c.page_size;
    a.slots = slots;
}

qimg::CachePages pages_of(const qimg_kv_cache& c) {
    return {c.k, c.v, c.k_exp, c.v_exp, c.n_pages, page_shift(c), c.n_kv_heads};
}

// Sizes of attention over a cache: queries, and tokens of a table's pages.
bool attn_sizes(int64_t total_q, int n_heads, int batch, int max_blocks, int prefix_blocks, int page_size) {
    const int64_t most = int64_t{1} << 30;
    return total_q * n_heads < most && batch < most && static_cast<int64_t>(max_blocks) * page_size < most &&
           static_cast<int64_t>(prefix_blocks) * page_size < most;
}

int64_t bytes_of(int elem_dtype) { return elem_dtype == QIMG_FP32 ? 4 : 2; }

}  // namespace

extern "C" {

int qimg_norm_rope_packed(const qimg_norm_rope* args, void* stream) {
    const char* fn = "qimg_norm_rope_packed";
    QIMG_REQUIRE(args, "%s: args is null", fn);
    const qimg_norm_rope& p = *args;
    const int64_t heads = static_cast<int64_t>(p.n_q_heads) + 2 * static_cast<int64_t>(p.n_kv_heads);
    if (const int e = check_heads(fn, p, heads, static_cast<int>(heads < (1 << 24) ? heads : 0)); e != QIMG_OK) return e;
    if (p.tokens == 0 || heads == 0) return QIMG_OK;
    return qimg::api_hip_status(
        qimg::launch_heads(heads_args(p), p.x_dtype, -1, static_cast<hipStream_t>(stream)), fn);
}

int qimg_norm_rope_cache(const qimg_norm_rope* args, const qimg_kv_cache* cache, const int32_t* slots, void* stream) {
    const char* fn = "qimg_norm_rope_cache";
    QIMG_REQUIRE(args, "%s: args is null", fn);
    const qimg_norm_rope& p = *args;
    if (const int e = check_cache(fn, cache, true); e != QIMG_OK) return e;
    const int64_t heads = static_cast<int64_t>(p.n_q_heads) + 2 * static_cast<int64_t>(p.n_kv_heads);
    if (const int e = check_heads(fn, p, heads, p.n_q_heads); e != QIMG_OK) return e;
    QIMG_REQUIRE(p.n_kv_heads == cache->n_kv_heads && p.head_dim == cache->head_dim,
                 "%s: the cache has %d kv heads of %d, x %d of %d", fn, cache->n_kv_heads, cache->head_dim, p.n_kv_heads,
                 p.head_dim);
    if (p.tokens == 0) return QIMG_OK;
    QIMG_REQUIRE(slots, "%s: null pointer", fn);
    qimg::HeadsArgs a = heads_args(p);
    const char* x = static_cast<const char*>(p.x);
    a.k = x + bytes_of(p.x_dtype) * p.n_q_heads * p.x_stride_h;
    a.v = x + bytes_of(p.x_dtype) * (p.n_q_heads + static_cast<int64_t>(p.n_kv_heads)) * p.x_stride_h;
    a.k_t = a.v_t = p.x_stride_t, a.k_h = a.v_h = p.x_stride_h;
    put_cache(a, *cache, slots);
    return qimg::api_hip_status(
        qimg::launch_heads(a, p.x_dtype, cache->dtype, static_cast<hipStream_t>(stream)), fn);
}

int qimg_kv_cache_write(const void* k, const void* v, int dtype, int64_t k_stride_t, int64_t k_stride_h,
                        int64_t v_stride_t, int64_t v_stride_h, int tokens, const qimg_kv_cache* cache,
                        const int32_t* slots, void* stream) {
    const char* fn = "qimg_kv_cache_write";
    if (const int e = check_cache(fn, cache, true); e != QIMG_OK) return e;
    QIMG_REQUIRE(float_type(dtype), "%s: dtype %d must be FP32, BF16 or FP16", fn, dtype);
    QIMG_REQUIRE(tokens >= 0 && static_cast<int64_t>(tokens) * cache->n_kv_heads < (int64_t{1} << 30),
                 "%s: tokens %d times heads must be at least 0 and < 2^30", fn, tokens);
    QIMG_REQUIRE(good_strides(k_stride_t, k_stride_h) && good_strides(v_stride_t, v_stride_h),
                 "%s: strides must be non-negative multiples of 8, token strides at most 2^24", fn);
    if (tokens == 0) return QIMG_OK;
    QIMG_REQUIRE(k && v && slots, "%s: null pointer", fn);
    QIMG_REQUIRE(aligned16(k) && aligned16(v), "%s: k and v must be 16-byte aligned", fn);
    qimg::HeadsArgs a{};
    a.tokens = tokens, a.nk = cache->n_kv_heads, a.d = cache->head_dim;
    a.k = k, a.v = v, a.k_t = k_stride_t, a.k_h = k_stride_h, a.v_t = v_stride_t, a.v_h = v_stride_h;
    put_cache(a, *cache, slots);
    return qimg::api_hip_status(qimg::launch_heads(a, dtype, cache->dtype, static_cast<hipStream_t>(stream)), fn);
}

int qimg_kv_cache_read(const qimg_kv_cache* cache, const int32_t* block_table, int max_blocks, const int32_t* k_lens,
                       const int32_t* cu_seqlens_k, int batch, void* k, void* v, int dtype, int64_t k_stride_t,
                       int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h, int total_k, void* stream) {
    const char* fn = "qimg_kv_cache_read";
    if (const int e = check_cache(fn, cache, true); e != QIMG_OK) return e;
    QIMG_REQUIRE(float_type(dtype), "%s: dtype %d must be FP32, BF16 or FP16", fn, dtype);
    QIMG_REQUIRE(batch >= 0 && total_k >= 0 && max_blocks >= 0 && batch < (1 << 30) && total_k < (1 << 30),
                 "%s: batch %d, total_k %d and max_blocks %d must be at least 0, the first two < 2^30", fn, batch, total_k,
                 max_blocks);
    QIMG_REQUIRE(good_strides(k_stride_t, k_stride_h) && good_strides(v_stride_t, v_stride_h),
                 "%s: strides must be non-negative multiples of 8, token strides at most 2^24", fn);
    if (batch == 0 || total_k == 0 || max_blocks == 0 || cache->n_pages == 0) return QIMG_OK;
    QIMG_REQUIRE(k && v && block_table && k_lens && cu_seqlens_k, "%s: null pointer", fn);
    QIMG_REQUIRE(aligned16(k) && aligned16(v), "%s: k and v must be 16-byte aligned", fn);
    QIMG_REQUIRE(k != v, "%s: k and v must not be the same", fn);
    QIMG_REQUIRE(apart(total_k, k_stride_t, cache->n_kv_heads, k_stride_h, cache->head_dim) &&
                     apart(total_k, v_stride_t, cache->n_kv_heads, v_stride_h, cache->head_dim),
                 "%s: the outputs' strides must keep their tokens and heads apart", fn);
    qimg::CacheReadArgs a{};
    a.c = pages_of(*cache), a.d = cache->head_dim;
    a.batch = batch, a.total = total_k, a.max_blocks = max_blocks;
    a.table = block_table, a.k_lens = k_lens, a.cu = cu_seqlens_k;
    a.k = k, a.v = v, a.k_t = k_stride_t, a.k_h = k_stride_h, a.v_t = v_stride_t, a.v_h = v_stride_h;
    return qimg::api_hip_status(qimg::launch_cache_read(a, cache->dtype, dtype, static_cast<hipStream_t>(stream)), fn);
}

int64_t qimg_attention_cache_scratch_bytes(int total_q, int batch, int n_heads, int n_kv_heads, int head_dim,
                                           int page_size, int max_blocks, int prefix_blocks) {
    if (total_q <= 0 || batch <= 0 || n_heads <= 0 || !kv_heads(n_kv_heads) || n_heads % n_kv_heads != 0 ||
        !head_dims(head_dim) || !page_sizes(page_size) || max_blocks < 0 || prefix_blocks < 0 ||
        !attn_sizes(total_q, n_heads, batch, max_blocks, prefix_blocks, page_size))
        return 0;
    const qimg::AttnCacheScratch s = qimg::attn_cache_scratch(
        qimg::attn_cache_plan(total_q, batch, n_heads, n_kv_heads, head_dim, static_cast<int64_t>(max_blocks) * page_size,
                              static_cast<int64_t>(prefix_blocks) * page_size),
        head_dim);
    return s.part_o + s.part_ml + 2 * s.dense;
}

int qimg_attention_cache(const qimg_attn_cache* args, const qimg_kv_cache* cache, void* scratch, int64_t scratch_bytes,
                         void* stream) {
    const char* fn = "qimg_attention_cache";
    QIMG_REQUIRE(args, "%s: args is null", fn);
    const qimg_attn_cache& p = *args;
    if (const int e = check_cache(fn, cache, true); e != QIMG_OK) return e;
    QIMG_REQUIRE(p.dtype == QIMG_BF16 || p.dtype == QIMG_FP16, "%s: dtype %d must be BF16 or FP16", fn, p.dtype);
    QIMG_REQUIRE(p.batch >= 0 && p.total_q >= 0 && p.max_blocks >= 0 && p.prefix_blocks >= 0,
                 "%s: bad sizes batch=%d total_q=%d max_blocks=%d prefix_blocks=%d", fn, p.batch, p.total_q, p.max_blocks,
                 p.prefix_blocks);
    QIMG_REQUIRE(p.n_heads > 0 && p.n_heads % cache->n_kv_heads == 0,
                 "%s: n_heads %d must be a multiple of the cache's n_kv_heads %d", fn, p.n_heads, cache->n_kv_heads);
    const float scale_log2 = p.sm_scale * 1.4426950408889634f;
    QIMG_REQUIRE(std::isfinite(scale_log2) && scale_log2 > 0.0f, "%s: sm_scale must be positive and finite", fn);
    QIMG_REQUIRE(attn_sizes(p.total_q, p.n_heads, p.batch, p.max_blocks, p.prefix_blocks, cache->page_size),
                 "%s: total_q * n_heads, batch and a table's pages times page_size must be < 2^30", fn);
    QIMG_REQUIRE(good_strides(p.q_stride_t, p.q_stride_h) && good_strides(p.out_stride_t, p.out_stride_h),
                 "%s: strides must be non-negative multiples of 8, token strides at most 2^24", fn);
    if (p.batch == 0 || p.total_q == 0) return QIMG_OK;
    QIMG_REQUIRE(p.q && p.out && p.cu_seqlens_q && p.k_lens, "%s: null pointer", fn);
    QIMG_REQUIRE((p.block_table || p.max_blocks == 0) && ((p.prefix_table && p.prefix_len) || p.prefix_blocks == 0),
                 "%s: null pointer", fn);
    QIMG_REQUIRE(aligned16(p.q) && aligned16(p.out), "%s: q and out must be 16-byte aligned", fn);
    QIMG_REQUIRE(p.out != p.q, "%s: out must not be q", fn);
    QIMG_REQUIRE(apart(p.total_q, p.out_stride_t, p.n_heads, p.out_stride_h, cache->head_dim),
                 "%s: out strides must keep its tokens and heads apart", fn);
    qimg::AttnCacheArgs a{};
    a.q = static_cast<const uint16_t*>(p.q);
    a.out = static_cast<uint16_t*>(p.out);
    a.q_t = p.q_stride_t, a.q_h = p.q_stride_h, a.o_t = p.out_stride_t, a.o_h = p.out_stride_h;
    a.c = pages_of(*cache);
    a.cu_q = p.cu_seqlens_q, a.table = p.block_table, a.k_lens = p.k_lens;
    a.prefix_table = p.prefix_table, a.prefix_len = p.prefix_len;
    // (a cache without pages holds no keys)
    a.max_blocks = cache->n_pages ? p.max_blocks : 0, a.prefix_blocks = cache->n_pages ? p.prefix_blocks : 0;
    a.batch = p.batch, a.total_q = p.total_q, a.hq = p.n_heads, a.group = p.n_heads / cache->n_kv_heads;
    a.causal = p.causal != 0;
    a.scale_log2 = scale_log2;
    const qimg::AttnCachePlan plan = qimg::attn_cache_plan(
        p.total_q, p.batch, p.n_heads, cache->n_kv_heads, cache->head_dim,
        static_cast<int64_t>(p.max_blocks) * cache->page_size, static_cast<int64_t>(p.prefix_blocks) * cache->page_size);
    a.own_splits = plan.own_splits, a.prefix_splits = plan.prefix_splits;
    const qimg::AttnCacheScratch parts = qimg::attn_cache_scratch(plan, cache->head_dim);
    const int64_t need = parts.part_o + parts.part_ml + 2 * parts.dense;
    if (need > 0) {
        if (!scratch || scratch_bytes < need)
            return qimg::api_fail(QIMG_ERR_SCRATCH, "%s: scratch %lld bytes < required %lld", fn,
                                  static_cast<long long>(scratch_bytes), static_cast<long long>(need));
        QIMG_REQUIRE(aligned16(scratch), "%s: scratch must be 16-byte aligned", fn);
        a.part_o = static_cast<float*>(scratch);
        a.part_ml = a.part_o + parts.part_o / 4;
        a.dense_k = reinterpret_cast<uint16_t*>(a.part_ml + parts.part_ml / 4);
        a.dense_v = a.dense_k + parts.dense / 2;
    }
    return qimg::api_hip_status(
        qimg::launch_attention_cache(a, plan, p.dtype, cache->dtype, cache->head_dim, static_cast<hipStream_t>(stream)),
        fn);
}

}  // extern "C"
