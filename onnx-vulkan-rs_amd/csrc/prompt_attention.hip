// Attention over packed prompts (hipc_prompt_attention).
#include "kv4.h"
#include "lanes.h"

namespace hipc {

namespace {

constexpr int kPromptMaxHead = 512;

struct PromptArgs {
    const void *q, *k, *v;
    void *y;
    const int *q_starts, *k_starts;
    int64_t q_stride, k_stride, v_stride, y_stride;
    int n_seqs, total_q, total_k, n_q_heads, group, dim, causal, window;
    float scale;
};

// Any head width and alignment: one wavefront per query row and head, one key after the other.
template <typename T>
__global__ void __launch_bounds__(64) prompt_rows_kernel(const PromptArgs a) {
    const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, kvh = h / a.group;
    int seq, first, end;
    if (!packed_sequence(a.q_starts, a.n_seqs, a.total_q, row, &seq, &first, &end)) return;
    const int k0 = max(a.k_starts[seq], 0), k1 = min(a.k_starts[seq + 1], a.total_k);
    const int keys = max(k1 - k0, 0);
    const int pos = keys - (end - first) + (row - first);
    const T *q = static_cast<const T *>(a.q) + a.q_stride * row + (int64_t)h * a.dim;
    T *y = static_cast<T *>(a.y) + a.y_stride * row + (int64_t)h * a.dim;
    constexpr int C = kPromptMaxHead / 64;
    float qv[C], acc[C] = {};
#pragma unroll
    for (int i = 0; i < C; i++) qv[i] = lane + 64 * i < a.dim ? (float)q[lane + 64 * i] * a.scale : 0.f;
    float m = -INFINITY, l = 0.f;
    const int from = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0, to = a.causal ? pos + 1 : keys;
    for (int t = from; t < to; t++) {
        const T *k = static_cast<const T *>(a.k) + a.k_stride * (k0 + t) + (int64_t)kvh * a.dim;
        const T *v = static_cast<const T *>(a.v) + a.v_stride * (k0 + t) + (int64_t)kvh * a.dim;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < C; i++)
            if (lane + 64 * i < a.dim) s = __builtin_fmaf(qv[i], (float)k[lane + 64 * i], s);
        s = lean_wave_sum(s);
        const float grown = fmaxf(m, s), keep = m == -INFINITY ? 0.f : expf(m - grown), p = expf(s - grown);
        m = grown, l = l * keep + p;
#pragma unroll
        for (int i = 0; i < C; i++)
            if (lane + 64 * i < a.dim) acc[i] = acc[i] * keep + p * (float)v[lane + 64 * i];
    }
#pragma unroll
    for (int i = 0; i < C; i++)
        if (lane + 64 * i < a.dim) y[lane + 64 * i] = (T)(l > 0.f ? acc[i] / l : l);
}

}  // namespace

}  // namespace hipc

using namespace hipc;

extern "C" {

int hipc_prompt_attention(hipc_ctx *ctx, const hipc_attention_heads *heads, int dtype, const void *Q, int64_t q_stride, const void *K,
                          int64_t k_stride, const void *V, int64_t v_stride, const void *q_starts, const void *k_starts, int64_t n_seqs,
                          int64_t total_q, int64_t total_k, void *Y, int64_t y_stride) {
    return entry(ctx, [&]() -> int {
        const char *who = "hipc_prompt_attention";
        PromptArgs a{};
        if (int rc = attention_check(ctx, who, heads, dtype, &a.scale)) return rc;
        HIPC_REFUSE(ctx, heads->head_dim > kPromptMaxHead, "%s: head_dim %d (up to %d is taken)", who, heads->head_dim, kPromptMaxHead);
        HIPC_REQUIRE(ctx, n_seqs >= 0 && n_seqs <= 1 << 20 && total_q >= 0 && total_q <= 0x7fffffff && total_k >= 0 && total_k <= 0x7fffffff,
                     "%s: %lld sequences, %lld query rows, %lld keys", who, (long long)n_seqs, (long long)total_q, (long long)total_k);
        if (n_seqs == 0 || total_q == 0) return HIPC_OK;
        const size_t size = dtype == HIPC_F16 ? 2 : 4;
        const int64_t qw = (int64_t)heads->n_q_heads * heads->head_dim, kw = (int64_t)heads->n_kv_heads * heads->head_dim, far = (int64_t)1 << 40;
        HIPC_REQUIRE(ctx, Q && Y && q_starts && k_starts && (total_k == 0 || (K && V)), "%s: null pointer", who);
        HIPC_REQUIRE(ctx, q_stride >= qw && y_stride >= qw && k_stride >= kw && v_stride >= kw, "%s: rows of Q, K, V and Y that overlap", who);
        HIPC_REQUIRE(ctx, q_stride <= far && y_stride <= far && k_stride <= far && v_stride <= far, "%s: rows too far apart", who);
        HIPC_REQUIRE(ctx, aligned(Q, size) && aligned(K, size) && aligned(V, size) && aligned(Y, size) && aligned(q_starts, 4) && aligned(k_starts, 4), "%s: a pointer off its elements", who);
        a.q = Q, a.k = K, a.v = V, a.y = Y, a.q_starts = static_cast<const int *>(q_starts), a.k_starts = static_cast<const int *>(k_starts);
        a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride, a.y_stride = y_stride;
        a.n_seqs = (int)n_seqs, a.total_q = (int)total_q, a.total_k = (int)total_k, a.n_q_heads = heads->n_q_heads, a.group = heads->n_q_heads / heads->n_kv_heads;
        a.dim = heads->head_dim, a.causal = heads->causal != 0, a.window = heads->window;
        const dim3 grid((unsigned)total_q, heads->n_q_heads);
        if (dtype == HIPC_F16) hipLaunchKernelGGL((prompt_rows_kernel<_Float16>), grid, 64, 0, ctx->stream, a);
        else hipLaunchKernelGGL((prompt_rows_kernel<float>), grid, 64, 0, ctx->stream, a);
        HIPC_LAUNCHED(ctx);
        return HIPC_OK;
    });
}

}  // extern "C"
