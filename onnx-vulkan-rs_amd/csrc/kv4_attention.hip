// Attention of the newest tokens of many sequences over the paged 4-bit cache (hipc_kv4_attention).
#include "kv4.h"
#include "lanes.h"

namespace hipc {

namespace {

struct Kv4Attend {
    hipc_kv4_cache cache;
    const void *q;
    void *y;
    int64_t q_stride, y_stride;
    int tokens, n_q_heads, window;
    float scale;
};

// One wavefront per query row: one key after the other, the running maximum and sum of the softmax beside the sums.
template <typename T>
__global__ void __launch_bounds__(64) kv4_attend_kernel(const Kv4Attend a) {
    const int lane = threadIdx.x, dim = a.cache.head_dim;
    const int64_t row = blockIdx.x;
    const int seq = (int)(row / a.tokens), h = blockIdx.y, kvh = h / (a.n_q_heads / a.cache.n_kv_heads);
    const int pos = kv4_length(a.cache, seq) - a.tokens + (int)(row - (int64_t)seq * a.tokens);
    const T *q = static_cast<const T *>(a.q) + row * a.q_stride + (int64_t)h * dim;
    T *y = static_cast<T *>(a.y) + row * a.y_stride + (int64_t)h * dim;
    constexpr int C = kKv4MaxHead / 64;
    float qv[C], acc[C] = {};
#pragma unroll
    for (int i = 0; i < C; i++) qv[i] = lane + 64 * i < dim ? (float)q[lane + 64 * i] * a.scale : 0.f;
    float m = -INFINITY, l = 0.f;
    for (int t = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0; t <= pos; t++) {
        const Kv4Place place = kv4_place(a.cache, seq, t);
        if (!place.there) continue;
        const int64_t r = place.slot + (int64_t)kvh * a.cache.page_size;
        auto value = [&](const void *codes, const void *params, int c) -> float {
            const int n = (static_cast<const uint8_t *>(codes)[r * (dim / 2) + c / 2] >> (4 * (c & 1))) & 15;
            const kvh2 p = static_cast<const kvh2 *>(params)[r * (dim / kKv4Group) + c / kKv4Group];
            return (float)__builtin_fmaf16((_Float16)n, p.x, p.y);
        };
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < C; i++)
            if (lane + 64 * i < dim) s = __builtin_fmaf(qv[i], value(a.cache.k_codes, a.cache.k_params, lane + 64 * i), s);
        s = lean_wave_sum(s);
        const float grown = fmaxf(m, s), keep = m == -INFINITY ? 0.f : expf(m - grown), p = expf(s - grown);
        m = grown, l = l * keep + p;
#pragma unroll
        for (int i = 0; i < C; i++)
            if (lane + 64 * i < dim) acc[i] = acc[i] * keep + p * value(a.cache.v_codes, a.cache.v_params, lane + 64 * i);
    }
#pragma unroll
    for (int i = 0; i < C; i++)
        if (lane + 64 * i < dim) y[lane + 64 * i] = (T)(l > 0.f ? acc[i] / l : l);
}

}  // namespace

int attention_check(hipc_ctx *ctx, const char *who, const hipc_attention_heads *h, int dtype, float *scale) {
    HIPC_REQUIRE(ctx, h, "%s: null heads", who);
    HIPC_REFUSE(ctx, dtype != HIPC_F16 && dtype != HIPC_F32, "%s: element type %d (f16 and f32 are taken)", who, dtype);
    HIPC_REQUIRE(ctx, h->n_kv_heads > 0 && h->n_q_heads > 0 && h->n_q_heads % h->n_kv_heads == 0 && h->n_q_heads <= 65535,
                 "%s: %d query heads over %d kv heads", who, h->n_q_heads, h->n_kv_heads);
    HIPC_REQUIRE(ctx, h->head_dim > 0, "%s: head_dim %d", who, h->head_dim);
    HIPC_REQUIRE(ctx, h->window >= 0 && (h->causal || h->window == 0), "%s: a window of %d (0 or more; causal calls only)", who, h->window);
    HIPC_REQUIRE(ctx, h->scale == h->scale && h->scale - h->scale == 0.f, "%s: the scale is no finite number", who);
    *scale = h->scale != 0.f ? h->scale : 1.f / sqrtf((float)h->head_dim);
    return HIPC_OK;
}

}  // namespace hipc

using namespace hipc;

extern "C" {

int hipc_kv4_attention(hipc_ctx *ctx, const hipc_kv4_cache *cache, const hipc_attention_heads *heads, int dtype, int64_t tokens,
                       const void *Q, int64_t q_stride, void *Y, int64_t y_stride) {
    return entry(ctx, [&]() -> int {
        const char *who = "hipc_kv4_attention";
        Kv4Attend a{};
        if (int rc = kv4_check(ctx, who, cache)) return rc;
        if (int rc = attention_check(ctx, who, heads, dtype, &a.scale)) return rc;
        HIPC_REQUIRE(ctx, heads->causal, "%s: a cache is attended to causally", who);
        HIPC_REQUIRE(ctx, heads->n_kv_heads == cache->n_kv_heads && heads->head_dim == cache->head_dim, "%s: %d kv heads of %d channels, the cache has %d of %d", who,
                     heads->n_kv_heads, heads->head_dim, cache->n_kv_heads, cache->head_dim);
        const int64_t group = heads->n_q_heads / heads->n_kv_heads;
        HIPC_REQUIRE(ctx, tokens > 0, "%s: %lld tokens a sequence", who, (long long)tokens);
        HIPC_REFUSE(ctx, tokens > 1024 || tokens * group > 1024, "%s: %lld tokens of %lld heads to a kv head: more than 1024 query rows", who, (long long)tokens, (long long)group);
        if (cache->n_seqs == 0) return HIPC_OK;
        const size_t size = dtype == HIPC_F16 ? 2 : 4;
        const int64_t width = (int64_t)heads->n_q_heads * heads->head_dim;
        HIPC_REQUIRE(ctx, Q && Y && aligned(Q, size) && aligned(Y, size), "%s: Q and Y", who);
        HIPC_REQUIRE(ctx, q_stride >= width && y_stride >= width && q_stride <= (int64_t)1 << 40 && y_stride <= (int64_t)1 << 40,
                     "%s: rows %lld and %lld apart, of %lld values", who, (long long)q_stride, (long long)y_stride, (long long)width);
        a.cache = *cache, a.q = Q, a.y = Y, a.q_stride = q_stride, a.y_stride = y_stride;
        a.tokens = (int)tokens, a.n_q_heads = heads->n_q_heads, a.window = heads->window;
        const dim3 grid((unsigned)(cache->n_seqs * tokens), heads->n_q_heads);
        if (dtype == HIPC_F16) hipLaunchKernelGGL((kv4_attend_kernel<_Float16>), grid, 64, 0, ctx->stream, a);
        else hipLaunchKernelGGL((kv4_attend_kernel<float>), grid, 64, 0, ctx->stream, a);
        HIPC_LAUNCHED(ctx);
        return HIPC_OK;
    });
}

}  // extern "C"
