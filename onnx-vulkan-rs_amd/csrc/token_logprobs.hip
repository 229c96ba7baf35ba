// Log probabilities, entropy and the best alternatives of rows of logits (hipc_token_logprobs).
#include <hip/hip_fp16.h>

#include <algorithm>

#include "internal.h"

namespace hipc {

namespace {

constexpr int kScratchLogprobs = 7;   // scratch slot of this operator alone
constexpr int kLogWaves = 4;
constexpr int kLogChunk = 2048;       // logits a wavefront holds at a time: 32 a lane
constexpr int kLogWorkgroups = 2048;  // at most that many share rows
constexpr int kLogBuffer = 256;       // candidates a wavefront ranks at a time
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LogprobArgs {
    const void *x;
    int64_t row_stride;
    int vocab, top, parts;   // workgroups of a row
    const int *tokens;
    float *logprob, *entropy, *top_logprobs;
    int *top_ids;
    struct LogPart *part;    // [row][parts]
    uint32_t *arrived;       // [row], zero between calls
};

// What a stretch of a row amounts to: its largest value m, sum of e = exp(x - m), and sum of e log2(e).
struct LogSum {
    float m, l, w;
};
struct LogPart {
    LogSum sum;
    uint32_t pad;
    uint64_t best[HIPC_TOP_MAX];   // keys, largest first; 0 where there are fewer
};

// A logit and its place as one whole number that orders as the alternatives do: by value, the lower id first among equals.
// Never 0 for a value that compares.
__device__ __forceinline__ uint64_t log_key(float x, int id) {
    const uint32_t b = __float_as_uint(x + 0.f);   // (-0 is 0)
    return (uint64_t)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b >> 31 ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ int key_id(uint64_t k) { return (int)~(uint32_t)k; }

__device__ __forceinline__ uint64_t lane_key(uint64_t v, int l) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const uint64_t o = (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), d) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)v, d);
        v = o > v ? o : v;
    }
    return v;
}

// A wavefront's `top` largest keys so far, the j-th in lane j (0: none), and N more of each lane to take in.
// Those that can count are written side by side into the wavefront's LDS, with the list, and ranked by counting the larger ones. Where
// too many pass the list's last -- a list that is not full yet, or ascending logits -- the top-th largest of the lanes' own largest is the bar:
// at least `top` keys are at or above it. If equal values still leave too many, one key after the other is picked.
template <int N, typename Key>
__device__ __forceinline__ void log_take(uint64_t &list, int top, uint64_t *buffer, Key key) {
    const int lane = threadIdx.x & 63;
    uint64_t bar = lane_key(list, top - 1);   // (keys at or below it cannot count)
    int count = 0;
    for (int round = 0;; round++) {
        count = 0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint64_t k = key(i);
            const uint64_t in = __ballot(k > bar);
            const int at = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
            if (k > bar && at < kLogBuffer - HIPC_TOP_MAX) buffer[at] = k;
            count += __popcll(in);
        }
        if (count <= kLogBuffer - HIPC_TOP_MAX) break;
        if (round == 1) {
            count = -1;
            break;
        }
        // the value of the top-th largest of the lanes' largest keys, bit by bit
        uint64_t own = 0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint64_t k = key(i);
            own = k > own ? k : own;
        }
        const uint32_t v = (uint32_t)(own >> 32);
        uint32_t reach = 0;
        for (int b = 31; b >= 0; b--) {
            const uint32_t next = reach | 1u << b;
            if (__popcll(__ballot(v >= next)) >= top) reach = next;
        }
        const uint64_t higher = reach ? ((uint64_t)reach << 32) - 1 : 0;
        bar = higher > bar ? higher : bar;
    }
    if (count == 0) return;
    if (count < 0) {
        uint64_t last = ~(uint64_t)0, mine = 0;
        for (int j = 0; j < top; j++) {
            uint64_t own = list < last ? list : 0;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const uint64_t k = key(i);
                own = k < last && k > own ? k : own;
            }
            last = wave_max(own);
            if (lane == j) mine = last;
            if (last == 0) break;
        }
        list = mine;
        return;
    }
    if (lane < top) buffer[count + lane] = list;
    const int all = count + top;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    uint64_t sorted = 0;
    for (int base = 0; base < all; base += 64) {
        const bool have = base + lane < all;
        const uint64_t k = have ? buffer[base + lane] : 0;
        int rank = 0;
        for (int j = 0; j < all; j++) rank += buffer[j] > k;
        // the lane of that rank takes it (empty places of the list, key 0, are taken by nobody)
        for (uint64_t left = __ballot(k != 0 && rank < top); left; left &= left - 1) {
            const int b = __builtin_ctzll(left);
            const uint64_t moved = lane_key(k, b);
            if (lane == __builtin_amdgcn_readlane(rank, b)) sorted = moved;
        }
    }
    list = sorted;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (read before the next call writes)
}

__device__ __forceinline__ LogSum log_join(const LogSum &a, const LogSum &b) {
    const float m = fmaxf(a.m, b.m);
    // a side without a value above -inf adds nothing (its difference to m may be no number)
    const float da = a.m == m ? 0.f : (a.m - m) * kLog2e, db = b.m == m ? 0.f : (b.m - m) * kLog2e;
    const float fa = a.l == 0.f ? 0.f : __builtin_amdgcn_exp2f(da), fb = b.l == 0.f ? 0.f : __builtin_amdgcn_exp2f(db);
    const float wa = a.l == 0.f || fa == 0.f ? 0.f : fa * __builtin_fmaf(a.l, da, a.w), wb = b.l == 0.f || fb == 0.f ? 0.f : fb * __builtin_fmaf(b.l, db, b.w);
    return {m, (a.l == 0.f ? 0.f : a.l * fa) + (b.l == 0.f ? 0.f : b.l * fb), wa + wb};
}

template <typename T>
__device__ void log_finish(const LogprobArgs &a, int64_t row, const LogSum &s, uint64_t list) {
    const int lane = threadIdx.x & 63;
    // no finite largest value: no distribution (a NaN among the logits has made l one; +inf too, by inf - inf)
    const float log_l = logf(s.l), lse = s.m == -INFINITY ? NAN : s.m + log_l;
    if (lane == 0) {
        if (a.logprob) {
            const int t = a.tokens[row];
            a.logprob[row] = t == -1 ? 0.f : t < 0 || t >= a.vocab ? NAN : (float)static_cast<const T *>(a.x)[row * a.row_stride + t] - lse;
        }
        if (a.entropy) a.entropy[row] = s.m == -INFINITY ? NAN : log_l - kLn2 * (s.w / s.l);
    }
    if (lane < a.top) {
        a.top_ids[row * a.top + lane] = list ? key_id(list) : -1;
        a.top_logprobs[row * a.top + lane] = list ? key_value(list) - lse : NAN;
    }
}

// A row is read once, by a.parts workgroups; a wavefront streams 2048 logits at a time, the next ones on their way meanwhile, with a running
// maximum and sums per lane and without a barrier. The alternatives cost a comparison per logit; only where one passes the list's last is there
// more to do, which after the first few thousand logits is rare.
template <typename T>
__global__ void __launch_bounds__(64 * kLogWaves) logprob_kernel(const LogprobArgs a) {
    constexpr int VEC = 16 / sizeof(T), LOADS = kLogChunk / 64 / VEC;
    typedef T TV __attribute__((ext_vector_type(VEC)));
    __shared__ uint64_t buffers[kLogWaves][kLogBuffer];
    __shared__ LogSum sums[kLogWaves];
    __shared__ uint64_t lists[kLogWaves][HIPC_TOP_MAX];
    __shared__ int last_here;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x - row * a.parts);
    uint64_t *buffer = buffers[wave];

    // the row in pieces of 16 aligned bytes: the first and the last may hold less of it
    const T *x = static_cast<const T *>(a.x) + row * a.row_stride;
    const int head = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const int pieces = (int)(((int64_t)a.vocab + head + VEC - 1) / VEC);
    const int chunks = (pieces + 64 * LOADS - 1) / (64 * LOADS);
    const int per = (chunks + a.parts * kLogWaves - 1) / (a.parts * kLogWaves);   // of a wavefront, one behind the other
    const int c0 = (part * kLogWaves + wave) * per, c1 = min(c0 + per, chunks);

    TV now[LOADS], next[LOADS];
    auto load = [&](int chunk, TV (&v)[LOADS]) {
#pragma unroll
        for (int e = 0; e < LOADS; e++) {
            const int64_t at = ((int64_t)(chunk * LOADS + e) * 64 + lane) * VEC - head;   // of the row
            if (at >= 0 && at + VEC <= a.vocab) {
                v[e] = __builtin_nontemporal_load(reinterpret_cast<const TV *>(x + at));
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j++) v[e][j] = at + j >= 0 && at + j < a.vocab ? x[at + j] : (T)-INFINITY;
            }
        }
    };
    float m = -INFINITY, l = 0.f, w = 0.f;
    uint64_t list = 0;
    float bar = -INFINITY;
    bool full = false;
    if (c0 < c1) load(c0, now);
    for (int c = c0; c < c1; c++) {
        if (c + 1 < c1) load(c + 1, next);
        float most = -INFINITY;
#pragma unroll
        for (int e = 0; e < LOADS; e++)
#pragma unroll
            for (int j = 0; j < VEC; j++) most = fmaxf(most, (float)now[e][j]);
        if (most > m) {
            const float f = l == 0.f ? 0.f : __builtin_amdgcn_exp2f((m - most) * kLog2e);
            w = f == 0.f ? 0.f : f * __builtin_fmaf(l, (m - most) * kLog2e, w), l *= f;
            m = most;
        }
        const float shift = m == -INFINITY ? 0.f : m;   // (subtracted before the scaling: a row at its type's lowest value times log2 e would be an infinity)
        float l2 = 0.f, w2 = 0.f;
#pragma unroll
        for (int e = 0; e < LOADS; e++)
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                // (a masked logit: t = -inf, its exponential 0, and 0 times the held t; a NaN stays one through the exponential)
                const float t = ((float)now[e][j] - shift) * kLog2e, y = __builtin_amdgcn_exp2f(t);
                l2 += y, w2 = __builtin_fmaf(y, fmaxf(t, -200.f), w2);
            }
        l += l2, w += w2;
        if (a.top > 0 && (__any(most > bar) || !full)) {
            log_take<LOADS * VEC>(list, a.top, buffer, [&](int i) -> uint64_t {
                const float v = (float)now[i / VEC][i % VEC];
                const int64_t id = ((int64_t)(c * LOADS + i / VEC) * 64 + lane) * VEC - head + i % VEC;
                return v == v && id >= 0 && id < a.vocab ? log_key(v, (int)id) : 0;
            });
            const uint64_t lowest = lane_key(list, a.top - 1);
            full = lowest != 0;
            if (full) bar = key_value(lowest);   // (later logits have higher ids: an equal one does not count)
        }
#pragma unroll
        for (int e = 0; e < LOADS; e++) now[e] = next[e];
    }

    // lanes, then wavefronts
    LogSum s{m, l, w};
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s = log_join(s, LogSum{__shfl_xor(s.m, d), __shfl_xor(s.l, d), __shfl_xor(s.w, d)});
    if (lane == 0) sums[wave] = s;
    if (lane < HIPC_TOP_MAX) lists[wave][lane] = list;
    __syncthreads();
    if (wave == 0) {
        for (int v = 1; v < kLogWaves; v++) s = log_join(s, sums[v]);
        if (a.top > 0) {
            uint64_t more[(kLogWaves - 1) * HIPC_TOP_MAX / 64 + 1] = {};
            constexpr int N = sizeof more / sizeof more[0];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int at = i * 64 + lane;
                if (at < (kLogWaves - 1) * HIPC_TOP_MAX) more[i] = lists[1 + at / HIPC_TOP_MAX][at % HIPC_TOP_MAX];
            }
            log_take<N>(list, a.top, buffer, [&](int i) { return more[i]; });
        }
    }
    if (a.parts == 1) {
        if (wave == 0) log_finish<T>(a, row, s, list);
        return;
    }
    // several workgroups: the one that comes last joins what they found
    LogPart *mine = a.part + row * a.parts;
    if (wave == 0) {
        auto put = [](void *to, uint32_t v) { __hip_atomic_store(static_cast<uint32_t *>(to), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        if (lane == 0) put(&mine[part].sum.m, __float_as_uint(s.m)), put(&mine[part].sum.l, __float_as_uint(s.l)), put(&mine[part].sum.w, __float_as_uint(s.w));
        if (lane < a.top) __hip_atomic_store(&mine[part].best[lane], list, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the stores are where everyone sees them
        if (lane == 0) {
            const uint32_t before = __hip_atomic_fetch_add(a.arrived + row, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
            last_here = before == (uint32_t)a.parts - 1;
            if (last_here) __hip_atomic_store(a.arrived + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next call
        }
    }
    __syncthreads();
    if (!last_here || wave != 0) return;
    auto get = [](const void *at) { return __hip_atomic_load(static_cast<const uint32_t *>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    s = {-INFINITY, 0.f, 0.f};
    for (int q = lane; q < a.parts; q += 64)
        s = log_join(s, LogSum{__uint_as_float(get(&mine[q].sum.m)), __uint_as_float(get(&mine[q].sum.l)), __uint_as_float(get(&mine[q].sum.w))});
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s = log_join(s, LogSum{__shfl_xor(s.m, d), __shfl_xor(s.l, d), __shfl_xor(s.w, d)});
    list = 0;
    if (a.top > 0) {
        constexpr int N = 8;
        for (int from = 0; from < a.parts * a.top; from += 64 * N) {
            uint64_t more[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int at = from + i * 64 + lane, q = at / a.top;
                more[i] = at < a.parts * a.top ? __hip_atomic_load(&mine[q].best[at - q * a.top], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
            }
            log_take<N>(list, a.top, buffer, [&](int i) { return more[i]; });
        }
    }
    log_finish<T>(a, row, s, list);
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
        LogprobArgs a{logits, row_stride, (int)vocab, top, 1, static_cast<const int *>(tokens), static_cast<float *>(logprob), static_cast<float *>(entropy),
                      static_cast<float *>(top_logprobs), static_cast<int *>(top_ids), nullptr, nullptr};
        // few rows are shared by several workgroups, each wavefront of which has 2048 logits at least
        const size_t count_bytes = kLogWorkgroups * sizeof(uint32_t), bytes = count_bytes + kLogWorkgroups * sizeof(LogPart);
        if (scratch_fits(ctx, kScratchLogprobs, bytes))
            a.parts = (int)std::max<int64_t>(1, std::min<int64_t>(kLogWorkgroups / rows, ceil_div(vocab, kLogWaves * kLogChunk)));
        if (a.parts > 1) {
            const void *before = ctx->scratch[kScratchLogprobs].ptr;
            void *block = nullptr;
            if (int rc = scratch_get(ctx, kScratchLogprobs, bytes, &block)) return rc;
            a.arrived = static_cast<uint32_t *>(block), a.part = reinterpret_cast<LogPart *>(static_cast<char *>(block) + count_bytes);
            if (block != before) {   // the words that are counted in are zero between calls
                hipLaunchKernelGGL((fill_words), 1, 256, 0, ctx->stream, a.arrived, count_bytes / 4, 0u);
                HIPC_LAUNCHED(ctx);
            }
        }
        HIPC_REQUIRE(ctx, rows * a.parts <= 0x7fffffff, "%s: too many rows", who);
        const unsigned grid = (unsigned)(rows * a.parts);
        if (dtype == HIPC_F16) hipLaunchKernelGGL((logprob_kernel<_Float16>), grid, 64 * kLogWaves, 0, ctx->stream, a);
        else hipLaunchKernelGGL((logprob_kernel<float>), grid, 64 * kLogWaves, 0, ctx->stream, a);
        HIPC_LAUNCHED(ctx);
        return HIPC_OK;
    });
}

}  // extern "C"
