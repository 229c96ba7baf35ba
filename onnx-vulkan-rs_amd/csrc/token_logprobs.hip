// Log probabilities, entropy and the best alternatives of rows of logits (hipc_token_logprobs).
#include <hip/hip_fp16.h>

#include "internal.h"
#include "lanes.h"

namespace hipc {

namespace {

struct LogprobArgs {
    const void *x;
    int64_t row_stride;
    int vocab, top;
    const int *tokens;
    float *logprob, *entropy, *top_logprobs;
    int *top_ids;
};

struct Best {
    float x;
    int id;
};
__device__ __forceinline__ bool better(float x, int id, float than_x, int than_id) { return x > than_x || (x == than_x && id < than_id); }

// One workgroup per row, a pass over it for the largest value, one for the sums and one for each alternative.
template <typename T>
__global__ void __launch_bounds__(256) logprob_rows_kernel(const LogprobArgs a) {
    __shared__ float part[256], part2[256];
    __shared__ int part_id[256];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.row_stride;
    auto joined = [&](float v, auto op, float *buf) {
        buf[tid] = v;
        __syncthreads();
        for (int n = 128; n > 0; n >>= 1) {
            if (tid < n) buf[tid] = op(buf[tid], buf[tid + n]);
            __syncthreads();
        }
        const float r = buf[0];
        __syncthreads();
        return r;
    };
    auto plus = [](float p, float q) { return p + q; };
    float m = -INFINITY;
    for (int i = tid; i < a.vocab; i += 256) m = fmaxf(m, (float)x[i]);
    m = joined(m, [](float p, float q) { return fmaxf(p, q); }, part);
    float l = 0.f, w = 0.f;
    for (int i = tid; i < a.vocab; i += 256) {
        const float v = (float)x[i], e = expf(v - m);
        l += e;
        if (e != 0.f) w += e * (v - m);
    }
    l = joined(l, plus, part), w = joined(w, plus, part2);
    const float lse = m + logf(l);   // NaN where the row has no finite largest value
    if (tid == 0) {
        if (a.logprob) {
            const int t = a.tokens[row];
            a.logprob[row] = t == -1 ? 0.f : t < 0 || t >= a.vocab ? NAN : (float)x[t] - lse;
        }
        if (a.entropy) a.entropy[row] = logf(l) - w / l;
    }
    Best last{INFINITY, -1};
    for (int k = 0; k < a.top; k++) {
        Best b{-INFINITY, -1};
        for (int i = tid; i < a.vocab; i += 256) {
            const float v = (float)x[i];
            if (v == v && better(last.x, last.id, v, i) && (b.id < 0 || better(v, i, b.x, b.id))) b = {v, i};
        }
        part[tid] = b.x, part_id[tid] = b.id;
        __syncthreads();
        for (int n = 128; n > 0; n >>= 1) {
            if (tid < n && part_id[tid + n] >= 0 && (part_id[tid] < 0 || better(part[tid + n], part_id[tid + n], part[tid], part_id[tid])))
                part[tid] = part[tid + n], part_id[tid] = part_id[tid + n];
            __syncthreads();
        }
        last = {part[0], part_id[0]};
        __syncthreads();
        if (tid == 0) a.top_ids[row * a.top + k] = last.id, a.top_logprobs[row * a.top + k] = last.id < 0 ? NAN : last.x - lse;
        if (last.id < 0) {
            for (int j = k + 1 + tid; j < a.top; j += 256) a.top_ids[row * a.top + j] = -1, a.top_logprobs[row * a.top + j] = NAN;
            break;
        }
    }
}

}  // namespace

}  // namespace hipc

using namespace hipc;

extern "C" {

int hipc_token_logprobs(hipc_ctx *ctx, int dtype, const void *logits, int64_t row_stride, int64_t rows, int64_t vocab, const void *tokens,
                        void *logprob, void *entropy, int top, void *top_ids, void *top_logprobs) {
    return entry(ctx, [&]() -> int {
        const char *who = "hipc_token_logprobs";
        HIPC_REFUSE(ctx, dtype != HIPC_F16 && dtype != HIPC_F32, "%s: element type %d (f16 and f32 are taken)", who, dtype);
        HIPC_REQUIRE(ctx, rows >= 0 && rows <= 0x7fffffff && vocab > 0 && vocab <= 1 << 30, "%s: %lld rows of %lld logits", who, (long long)rows, (long long)vocab);
        HIPC_REQUIRE(ctx, row_stride >= vocab && row_stride <= (int64_t)1 << 40, "%s: rows %lld apart, of %lld logits", who, (long long)row_stride, (long long)vocab);
        HIPC_REQUIRE(ctx, top >= 0 && top <= HIPC_TOP_MAX, "%s: %d alternatives (0 to %d are taken)", who, top, HIPC_TOP_MAX);
        if (rows == 0) return HIPC_OK;
        HIPC_REQUIRE(ctx, !tokens == !logprob, "%s: tokens and logprob are given together", who);
        HIPC_REQUIRE(ctx, (top > 0) == (top_ids != nullptr) && (top > 0) == (top_logprobs != nullptr), "%s: top_ids and top_logprobs are given where top is not 0, and only there", who);
        HIPC_REQUIRE(ctx, logits && aligned(logits, dtype == HIPC_F16 ? 2 : 4), "%s: logits", who);
        HIPC_REQUIRE(ctx, aligned(tokens, 4) && aligned(logprob, 4) && aligned(entropy, 4) && aligned(top_ids, 4) && aligned(top_logprobs, 4), "%s: a pointer off its elements", who);
        LogprobArgs a{logits, row_stride, (int)vocab, top, static_cast<const int *>(tokens), static_cast<float *>(logprob), static_cast<float *>(entropy),
                      static_cast<float *>(top_logprobs), static_cast<int *>(top_ids)};
        if (dtype == HIPC_F16) hipLaunchKernelGGL((logprob_rows_kernel<_Float16>), (unsigned)rows, 256, 0, ctx->stream, a);
        else hipLaunchKernelGGL((logprob_rows_kernel<float>), (unsigned)rows, 256, 0, ctx->stream, a);
        HIPC_LAUNCHED(ctx);
        return HIPC_OK;
    });
}

}  // extern "C"
