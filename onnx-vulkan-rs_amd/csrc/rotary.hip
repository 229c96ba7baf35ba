// Norms of query and key heads and their rotation by position (hipc_rotary), and the same on the way into the 4-bit cache
// (hipc_kv4_append_rotary).
//
//   x^ = x / sqrt(mean(x^2) + eps) * w                                (per head, where there is a weight w)
//   y_a = x^_a cos - x^_b sin,  y_b = x^_b cos + x^_a sin              (a, b) = (i, i + n) or (2i, 2i + 1), angle = position * frequency[i]
//
// A position's angles are one row's and all its heads'. They are formed in 64 bits: in 32 an angle of a million is off by a sixteenth. A product of
// 31 and 24 bits, in turns; what is left behind whole turns goes to sine and cosine. Everything else is f32, as in the decode step's norm and rotation,
// every step rounded by itself (this file is compiled without contraction): a cache stores what keys are quantized to, and one that stands next to the border
// between two codes, or is the lowest of its group, is to fall on the side where these steps put it, whatever kernel or layout takes them.
//
// Memory bounds it. A wavefront has a row, or some heads of one where rows are few or long, and takes 64 / L heads at a time, L lanes a head; a lane has
// two vectors of V channels, half a rotation apart (the channels that turn with each other, or pairs that lie in one vector), the same channels of every head it sees, so that its
// cosines and sines stay in registers. Graphs of launches, rows of several such calls in turn (1.2 GB) / of the same call again, which the last cache holds in part: 8192 rows of
// 32 / 8 heads of 128 in f16, 168 MB, 38.1 / 29 us, 4.4 TB/s (a 1 GiB copy: 4.96), in f32 62.6 / 49, 5.4 TB/s; 1500 of 16 / 16 heads of 96 in f32 12.4 / 9.2; 48 rows 3.6. Figures below are of rows in turn.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv4.h"
#include "lanes.h"

namespace hipc {

namespace {

constexpr int kRotaryMaxHead = 512;
constexpr int64_t kRotaryCaches = 32 << 20;   // bytes: the L2 caches

struct RotaryArgs {
    hipc_kv4_cache cache;              // storing
    const int *starts, *positions;     // ... and its rows; or the rows' positions
    const void *q, *k, *v;
    void *q_out, *k_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
    const float *frequencies, *q_norm, *k_norm;
    int rows, n_q, n_kv, dim, half;
    int lg_lanes, lg_turning, chunks, per;   // lanes of a head (a power of two) and of its channels that turn; wavefronts of a row, and what each takes of it
    float eps, amplitude;
};

// The sum of x and y over 2^lanes neighbouring lanes, in all of them: over 2^part of x, over as many of y, these two, and then the others' (both numbers are uniform).
__device__ __forceinline__ float lanes_sum(float x, float y, int part, int lanes) {
    if (part > 0) x += lean_dpp<0xB1>(x), y += lean_dpp<0xB1>(y);      // quad_perm [1,0,3,2]
    if (part > 1) x += lean_dpp<0x4E>(x), y += lean_dpp<0x4E>(y);      // quad_perm [2,3,0,1]
    if (part > 2) x += lean_dpp<0x141>(x), y += lean_dpp<0x141>(y);    // the other four of eight (mirrored)
    if (part > 3) x += lean_dpp<0x140>(x), y += lean_dpp<0x140>(y);    // the other eight of sixteen
    if (part > 4) x += __shfl_xor(x, 16), y += __shfl_xor(y, 16);
    if (part > 5) x += __shfl_xor(x, 32), y += __shfl_xor(y, 32);
    x += y;
    if (part < lanes) {
        if (part < 1) x += lean_dpp<0xB1>(x);
        if (part < 2 && lanes > 1) x += lean_dpp<0x4E>(x);
        if (part < 3 && lanes > 2) x += lean_dpp<0x141>(x);
        if (part < 4 && lanes > 3) x += lean_dpp<0x140>(x);
        if (part < 5 && lanes > 4) x += __shfl_xor(x, 16);
        if (lanes > 5) x += __shfl_xor(x, 32);
    }
    return x;
}

// 1 / sqrt(x) to half a step and a little: the function's step of error goes with one Newton step whose remainder, 1 - x y^2, is formed without rounding x y
__device__ __forceinline__ float reciprocal_root(float x) {
    const float y = rsqrtf(x), root = x * y, low = __builtin_fmaf(x, y, -root), rest = __builtin_fmaf(-low, y, __builtin_fmaf(-root, y, 1.f));
    return x > 0.f && x < INFINITY ? __builtin_fmaf(0.5f * y, rest, y) : y;
}

// V values side by side; rows and strides lie on 16 bytes (V values, where these are less) or V is 1
template <typename T, int V>
struct RotaryVector {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T) * V < 16 ? sizeof(T) * V : 16)));
};
template <typename T>
struct RotaryVector<T, 1> {
    typedef T type;
};
template <typename T, int V>
__device__ __forceinline__ void rotary_load(const T *p, T (&x)[V]) {
    const auto v = *reinterpret_cast<const typename RotaryVector<T, V>::type *>(p);
    __builtin_memcpy(x, &v, sizeof x);
}
template <typename T, int V, bool PAST>
__device__ __forceinline__ void rotary_store(T *p, const T (&x)[V]) {
    typename RotaryVector<T, V>::type v;
    __builtin_memcpy(&v, x, sizeof v);
    auto *to = reinterpret_cast<typename RotaryVector<T, V>::type *>(p);
    if constexpr (PAST) __builtin_nontemporal_store(v, to);
    else *to = v;
}

// what this wavefront has stored to its LDS is there for its other lanes
__device__ __forceinline__ void wave_meets() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// NEAR: interleaved pairs; STORE: into a cache; PAST: results leave past the caches
template <typename T, int V, bool NEAR, bool STORE, bool PAST>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
    constexpr int E = V == 1 ? 4 : 1;            // items of a lane: V channels and the V they turn with, or 2 V behind those that turn
    constexpr int N = 2 * V * E, UNITS = N / 8;   // a lane's values at a time; as units of eight side by side
    __shared__ float2 turns[4][kRotaryMaxHead / 2];
    __shared__ float keys[STORE ? 4 : 1][STORE ? 64 * N : 1];
    const int w = kv4_wave(), lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = w / a.chunks, chunk = w - row * a.chunks;
    if (row >= a.rows) return;
    int position;
    Kv4Place place = {0, false};
    if (STORE) {
        int seq, first, end;
        if (!packed_sequence(a.starts, a.cache.n_seqs, a.rows, row, &seq, &first, &end)) return;
        position = kv4_length(a.cache, seq) - end + row;
        place = kv4_place(a.cache, seq, position);
    } else {
        position = a.half > 0 ? a.positions[row] : 0;
    }

    // what this wavefront takes: the query heads, then the key heads, then (storing) units of the values
    const int lanes = 1 << a.lg_lanes, together = 64 >> a.lg_lanes, l = lane & (lanes - 1), head0 = lane >> a.lg_lanes;
    const int q_passes = (a.n_q + together - 1) >> (6 - a.lg_lanes), k_passes = (a.n_kv + together - 1) >> (6 - a.lg_lanes);
    const int v_units = STORE ? a.n_kv * (a.dim >> 3) : 0, v_passes = STORE ? (v_units + 64 * UNITS - 1) / (64 * UNITS) : 0;
    const int passes = STORE && !place.there ? q_passes : q_passes + k_passes + v_passes;
    const int pass0 = chunk * a.per, pass1 = min(pass0 + a.per, passes);
    if (pass0 >= pass1) return;

    // The lane's channels of a head: V each from c[e][0] and c[e][1] on, where there[e][.] (else the head's first stand in), half a rotation apart, so that lanes side by
    // side have vectors side by side; and whether they turn. (NEAR single channels: neighbours.)
    constexpr bool BESIDE = NEAR && V == 1;
    int c[E][2];
    bool turns_here[E];
    bool there[E][2];
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int item = l + (e << a.lg_lanes), turning = a.half / V;
        turns_here[e] = item < turning;
        c[e][0] = turns_here[e] && !BESIDE ? item * V : 2 * item * V;   // (behind the pairs, 2 V an item as well)
        c[e][1] = turns_here[e] && !BESIDE ? a.half + item * V : 2 * item * V + V;
#pragma unroll
        for (int h = 0; h < 2; h++) there[e][h] = c[e][h] < a.dim, c[e][h] = there[e][h] ? c[e][h] : 0;
    }
    auto load = [&](int pass, T (&x)[N]) {
        if (STORE && pass >= q_passes + k_passes) {
#pragma unroll
            for (int i = 0; i < N; i += V) {
                const int u = ((pass - q_passes - k_passes) * UNITS + i / 8) * 64 + lane;
                rotary_load<T, V>(static_cast<const T *>(a.v) + a.v_stride * row + (int64_t)min(u, v_units - 1) * 8 + i % 8, *reinterpret_cast<T(*)[V]>(x + i));
            }
            return;
        }
        const bool key = pass >= q_passes;
        const int head = min((key ? pass - q_passes : pass) * together + head0, (key ? a.n_kv : a.n_q) - 1);
        const T *from = static_cast<const T *>(key ? a.k : a.q) + (key ? a.k_stride : a.q_stride) * row + (int64_t)head * a.dim;
#pragma unroll
        for (int i = 0; i < 2 * E; i++) rotary_load<T, V>(from + c[i / 2][i % 2], *reinterpret_cast<T(*)[V]>(x + i * V));
    };
    T next[N];
    load(pass0, next);

    // norm weights of the lane's channels: the queries', then the keys'
    float weight[N];
    auto load_weights = [&](const float *w) {
        if (!w) return;
#pragma unroll
        for (int i = 0; i < 2 * E; i++) __builtin_memcpy(weight + i * V, w + c[i / 2][i % 2], V * sizeof(float));
    };
    load_weights(pass0 < q_passes ? a.q_norm : a.k_norm);

    // the angles, a pair a lane, while the first heads are on their way
    for (int p = lane; p < a.half; p += 64) {
        const double turn = (double)position * (double)a.frequencies[p] * 0.15915494309189533577;   // 1 / (2 pi)
        double s, co;
        sincospi(2.0 * (turn - __builtin_rint(turn)), &s, &co);
        turns[wave][p] = make_float2((float)co * a.amplitude, (float)s * a.amplitude);
    }
    wave_meets();
    float cosine[E][V], sine[E][V];
#pragma unroll
    for (int e = 0; e < E; e++)
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int pair = !NEAR ? c[e][0] + j : V == 1 ? c[e][0] / 2 : j < V / 2 ? c[e][0] / 2 + j : c[e][1] / 2 + j - V / 2;
            const float2 t = turns_here[e] ? turns[wave][pair] : make_float2(1.f, 0.f);
            cosine[e][j] = t.x, sine[e][j] = t.y;
        }

    // the lane's values of a head, normed and turned
    auto turned = [&](const T (&x)[N], bool norm, T (&y)[N]) {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = (float)x[i];
        if (norm) {
            // squares four side by side, then neighbours by twos: an error that grows with the logarithm, and (V > 1, powers of two) the same order whatever the vectors'
            // width and however many channels turn; a plain form in PyTorch has the same sums to the bit at 128 and 256 channels, so that it and a cache filled here agree in their codes
            float part[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < E; e++) {
                float p[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float quads[(V + 3) / 4];
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float x = v[(2 * e + h) * V + i], square = x * x;
                        quads[i / 4] = i % 4 ? quads[i / 4] + square : square;
                    }
                    p[h] = there[e][h] ? (V == 8 ? quads[0] + quads[V / 8] : quads[0]) : 0.f;
                }
                part[0] += turns_here[e] ? p[0] : p[0] + p[1], part[1] += turns_here[e] ? p[1] : 0.f;
            }
            const float sum = lanes_sum(part[0], part[1], a.lg_turning, a.lg_lanes);
            const float by = reciprocal_root(sum / (float)a.dim + a.eps);
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = v[i] * by * weight[i];
        }
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (int j = 0; j < V; j++) {
                const int ia = 2 * e * V + (NEAR ? 2 * j : j), ib = NEAR ? ia + 1 : ia + V;
                const float first = v[ia] * cosine[e][j] - v[ib] * sine[e][j], second = v[ib] * cosine[e][j] + v[ia] * sine[e][j];
                y[ia] = (T)(turns_here[e] ? first : v[ia]);
                y[ib] = (T)(turns_here[e] ? second : v[ib]);
            }
    };
    auto put = [&](T *to, const T (&y)[N]) {
#pragma unroll
        for (int i = 0; i < 2 * E; i++)
            if (there[i / 2][i % 2]) rotary_store<T, V, PAST>(to + c[i / 2][i % 2], *reinterpret_cast<const T(*)[V]>(y + i * V));
    };
    // unit u of the row's heads, of keys or of values, into the cache
    auto quantize = [&](int u, bool mine, float (&x)[8], void *codes, void *params) {
        uint32_t bits;
        const uint32_t param = kv4_quantize(x, &bits);
        if (!mine) return;
        const int per_head = a.dim >> 3, head = u / per_head, channel = (u - head * per_head) * 8;
        const int64_t r = place.slot + (int64_t)head * a.cache.page_size;
        *reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(codes) + r * (a.dim / 2) + channel / 2) = bits;
        if ((lane & 3) == 0) static_cast<uint32_t *>(params)[r * (a.dim / kKv4Group) + channel / kKv4Group] = param;
    };
    for (int pass = pass0; pass < pass1; pass++) {
        T x[N], y[N];
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = next[i];
        if (pass + 1 < pass1) load(pass + 1, next);
        if (pass < q_passes) {
            const int head = pass * together + head0;
            turned(x, a.q_norm != nullptr, y);
            if (head < a.n_q) put(static_cast<T *>(a.q_out) + a.q_out_stride * row + (int64_t)head * a.dim, y);
        } else if (pass < q_passes + k_passes) {
            const int first = (pass - q_passes) * together, head = first + head0;
            if (pass == q_passes && pass > pass0) load_weights(a.k_norm);
            turned(x, a.k_norm != nullptr, y);
            if (!STORE) {
                if (head < a.n_kv) put(static_cast<T *>(a.k_out) + a.k_out_stride * row + (int64_t)head * a.dim, y);
                continue;
            }
            // the heads' channels in their order, through LDS
#pragma unroll
            for (int i = 0; i < N; i++)
                if (there[i / V / 2][i / V % 2]) keys[wave][head0 * a.dim + c[i / V / 2][i / V % 2] + i % V] = (float)y[i];
            wave_meets();
            const int units = min(together, a.n_kv - first) * (a.dim >> 3);
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const int u = i * 64 + lane;
                float unit[8];
#pragma unroll
                for (int j = 0; j < 8; j++) unit[j] = u < units ? keys[wave][u * 8 + j] : 0.f;
                quantize(first * (a.dim >> 3) + u, u < units, unit, a.cache.k_codes, a.cache.k_params);
            }
            wave_meets();   // (the next heads' channels go where these were)
        } else if (STORE) {
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const int u = ((pass - q_passes - k_passes) * UNITS + i) * 64 + lane;
                float unit[8];
#pragma unroll
                for (int j = 0; j < 8; j++) unit[j] = (float)x[i * 8 + j];
                quantize(u, u < v_units, unit, a.cache.v_codes, a.cache.v_params);
            }
        }
    }
}

int rotary_check(hipc_ctx *ctx, const char *who, const hipc_rotary_heads *h, int dtype, int64_t rows, RotaryArgs *a) {
    HIPC_REQUIRE(ctx, h, "%s: null heads", who);
    HIPC_REFUSE(ctx, dtype != HIPC_F16 && dtype != HIPC_F32, "%s: element type %d (f16 and f32 are taken)", who, dtype);
    HIPC_REQUIRE(ctx, h->n_q_heads >= 0 && h->n_q_heads <= 65535 && h->n_kv_heads >= 0 && h->n_kv_heads <= 65535, "%s: %d query heads, %d key heads", who, h->n_q_heads, h->n_kv_heads);
    HIPC_REQUIRE(ctx, h->head_dim > 0, "%s: head_dim %d", who, h->head_dim);
    HIPC_REFUSE(ctx, h->head_dim > kRotaryMaxHead, "%s: head_dim %d (up to %d is taken)", who, h->head_dim, kRotaryMaxHead);
    HIPC_REQUIRE(ctx, h->rotary_dim >= 0 && h->rotary_dim <= h->head_dim && h->rotary_dim % 2 == 0, "%s: %d channels of %d turn in pairs", who, h->rotary_dim, h->head_dim);
    HIPC_REQUIRE(ctx, h->norm_eps >= 0.f && h->norm_eps - h->norm_eps == 0.f && h->amplitude - h->amplitude == 0.f, "%s: norm_eps and amplitude are finite numbers", who);
    HIPC_REQUIRE(ctx, (h->rotary_dim == 0 || h->frequencies) && aligned(h->frequencies, 4) && aligned(h->q_norm, 4) && aligned(h->k_norm, 4), "%s: frequencies and norm weights", who);
    HIPC_REQUIRE(ctx, rows >= 0 && rows <= 0x7fffffff, "%s: %lld rows", who, (long long)rows);
    a->frequencies = static_cast<const float *>(h->frequencies), a->q_norm = static_cast<const float *>(h->q_norm), a->k_norm = static_cast<const float *>(h->k_norm);
    a->rows = (int)rows, a->n_q = h->n_q_heads, a->n_kv = h->n_kv_heads, a->dim = h->head_dim, a->half = h->rotary_dim / 2;
    a->eps = h->norm_eps, a->amplitude = h->amplitude != 0.f ? h->amplitude : 1.f;
    return HIPC_OK;
}
// rows of `heads` heads, `stride` apart
int rotary_rows(hipc_ctx *ctx, const char *who, const char *what, const RotaryArgs &a, int heads, size_t size, const void *p, int64_t stride) {
    if (heads == 0) return HIPC_OK;
    HIPC_REQUIRE(ctx, p && aligned(p, size), "%s: %s", who, what);
    HIPC_REQUIRE(ctx, stride >= (int64_t)heads * a.dim && stride <= (int64_t)1 << 40, "%s: rows of %s %lld apart, of %lld values", who, what, (long long)stride, (long long)heads * a.dim);
    return HIPC_OK;
}

// rows that are turned where they lie stay there
int rotary_in_place(hipc_ctx *ctx, const char *who, const char *what, const RotaryArgs &a, int heads, const void *p, int64_t stride, const void *out, int64_t out_stride) {
    HIPC_REQUIRE(ctx, heads == 0 || p != out || stride == out_stride || a.rows <= 1, "%s: %s where it lies, rows %lld apart and then %lld", who, what, (long long)stride, (long long)out_stride);
    return HIPC_OK;
}

template <typename T, bool STORE>
int rotary_launch(hipc_ctx *ctx, const char *who, RotaryArgs a, bool near) {
    const int64_t strides[5] = {a.q_stride, a.k_stride, a.v_stride, a.q_out_stride, a.k_out_stride};
    const void *rows[5] = {a.q, a.k, a.v, a.q_out, a.k_out};
    const int heads[5] = {a.n_q, a.n_kv, STORE ? a.n_kv : 0, a.n_q, STORE ? 0 : a.n_kv};
    // vectors of 16 bytes where pairs and rows allow (of eight f32, two loads: 8192 rows of 32 / 8 heads of 128 76.9 us, of four 62.6), f16 ones of 8, or single values
    auto fits = [&](int v) {
        const int64_t bytes = std::min<int64_t>(v * sizeof(T), 16);
        bool ok = a.dim % v == 0 && a.half % v == 0;
        for (int i = 0; i < 5; i++)
            if (heads[i]) ok &= aligned(rows[i], bytes) && strides[i] * (int64_t)sizeof(T) % bytes == 0;
        return ok;
    };
    auto launch = [&](auto width) -> int {
        constexpr int V = decltype(width)::value, N = 2 * V * (V == 1 ? 4 : 1);
        const int items = (int)(a.half / V + ceil_div(a.dim - 2 * a.half, 2 * V));
        while (a.lg_lanes < 6 && 1 << a.lg_lanes < items) a.lg_lanes++;
        while (a.lg_turning < a.lg_lanes && 1 << a.lg_turning < a.half / V) a.lg_turning++;
        const int together = 64 >> a.lg_lanes;
        const int64_t passes = ceil_div(a.n_q, together) + ceil_div(a.n_kv, together) + (STORE ? ceil_div((int64_t)a.n_kv * a.dim, 64 * N) : 0);
        if (passes == 0) return HIPC_OK;
        // Rows that do not fill the device are shared by wavefronts, 32 a CU (storing 16): 1500 rows of 16 / 16 heads of 96 in f32, the same again, 9.0 us, by eight a CU 13.2; stored, of
        // 32 / 8 heads of 128 in f16, 13.3, and 15.3. So are long rows of f32, in pairs of passes, however many: 8192 of 32 / 8 heads of 128 62.6 us, a wavefront each 84.9 (f16 37.8 and 38.1).
        a.chunks = (int)std::max<int64_t>(1, std::min(passes, (STORE ? 16 : 32) * (int64_t)ctx->cu_count / a.rows));
        if (sizeof(T) == 4 && passes > 8) a.chunks = std::max(a.chunks, (int)ceil_div(passes, 2));
        a.per = (int)ceil_div(passes, a.chunks), a.chunks = (int)ceil_div(passes, a.per);
        const int64_t groups = ceil_div((int64_t)a.rows * a.chunks, 4);
        HIPC_REFUSE(ctx, !grid_fits(groups, 256), "%s: %d rows: too many for one call", who, a.rows);
        auto run = [&](auto neighbours, auto past) {
            hipLaunchKernelGGL((rotary_kernel<T, V, decltype(neighbours)::value, STORE, decltype(past)::value>), (unsigned)groups, 256, 0, ctx->stream, a);
        };
        // Many rows -- more than the caches near the CUs hold -- leave past these where neighbouring lanes store side by side, whole lines: 8192 rows of 32 / 8 heads of 128 in f16
        // 38.1 us (through the caches 41.5), in f32 62.6 (69.4).
        constexpr bool LINES = sizeof(T) * V == 16;
        const bool past = LINES && a.half * sizeof(T) % 128 == 0 && (int64_t)a.rows * (a.n_q + (STORE ? 0 : a.n_kv)) * a.dim * (int64_t)sizeof(T) >= kRotaryCaches;
        auto kinds = [&](auto neighbours) {
            if (past) run(neighbours, std::integral_constant<bool, LINES>());
            else run(neighbours, std::false_type());
        };
        if (near) kinds(std::true_type());
        else kinds(std::false_type());
        HIPC_LAUNCHED(ctx);
        return HIPC_OK;
    };
    if constexpr (sizeof(T) == 2)
        if (fits(8)) return launch(std::integral_constant<int, 8>());
    if (fits(4)) return launch(std::integral_constant<int, 4>());
    return launch(std::integral_constant<int, 1>());
}

}  // namespace

}  // namespace hipc

using namespace hipc;

extern "C" {

int hipc_rotary_frequencies(double theta, int32_t rotary_dim, const hipc_rotary_scaling *scaling, float *frequencies) {
    const char *who = "hipc_rotary_frequencies";
    if (!(theta > 0.0) || !std::isfinite(theta)) return host_fail(HIPC_ERR_INVALID, "%s: a base of %g", who, theta);
    if (rotary_dim < 0 || rotary_dim % 2 != 0) return host_fail(HIPC_ERR_INVALID, "%s: %d channels", who, rotary_dim);
    if (rotary_dim > 0 && !frequencies) return host_fail(HIPC_ERR_INVALID, "%s: null pointer", who);
    const double d = rotary_dim;
    if (scaling) {
        if (scaling->kind != HIPC_ROTARY_LINEAR && scaling->kind != HIPC_ROTARY_BASE && scaling->kind != HIPC_ROTARY_BY_PARTS)
            return host_fail(HIPC_ERR_UNSUPPORTED, "%s: scaling of kind %d", who, scaling->kind);
        if (!(scaling->factor >= 1.f) || !std::isfinite(scaling->factor)) return host_fail(HIPC_ERR_INVALID, "%s: a factor of %g", who, scaling->factor);
        if (scaling->kind == HIPC_ROTARY_BY_PARTS && (!(scaling->trained > 0.f) || !std::isfinite(scaling->trained) || !(scaling->slow >= 0.f) || !(scaling->fast > scaling->slow) || !std::isfinite(scaling->fast)))
            return host_fail(HIPC_ERR_INVALID, "%s: %g positions, %g to %g turns", who, scaling->trained, scaling->slow, scaling->fast);
        if (scaling->kind == HIPC_ROTARY_BASE && rotary_dim > 2) theta *= std::pow((double)scaling->factor, d / (d - 2.0));
    }
    auto frequency = [&](int i) {
        double f = std::pow(theta, -2.0 * i / d);
        if (scaling && scaling->kind == HIPC_ROTARY_LINEAR) f /= scaling->factor;
        if (scaling && scaling->kind == HIPC_ROTARY_BY_PARTS) {
            const double turns = scaling->trained * f / 6.283185307179586477;
            const double keep = std::min(std::max((turns - scaling->slow) / ((double)scaling->fast - scaling->slow), 0.0), 1.0);
            f = f / scaling->factor * (1.0 - keep) + f * keep;
        }
        return (float)f;
    };
    for (int i = 0; i < rotary_dim / 2; i++)
        if (!std::isfinite(frequency(i))) return host_fail(HIPC_ERR_INVALID, "%s: a base of %g makes frequency %d infinite", who, theta, i);
    for (int i = 0; i < rotary_dim / 2; i++) frequencies[i] = frequency(i);
    return HIPC_OK;
}

int hipc_rotary(hipc_ctx *ctx, const hipc_rotary_heads *heads, int dtype, const void *positions, int64_t rows, const void *Q, int64_t q_stride,
                const void *K, int64_t k_stride, void *Q_out, int64_t q_out_stride, void *K_out, int64_t k_out_stride) {
    return entry(ctx, [&]() -> int {
        const char *who = "hipc_rotary";
        RotaryArgs a{};
        if (int rc = rotary_check(ctx, who, heads, dtype, rows, &a)) return rc;
        if (rows == 0) return HIPC_OK;
        HIPC_REQUIRE(ctx, (a.half == 0 || positions) && aligned(positions, 4), "%s: positions", who);
        const size_t size = dtype == HIPC_F16 ? 2 : 4;
        if (int rc = rotary_rows(ctx, who, "Q", a, a.n_q, size, Q, q_stride)) return rc;
        if (int rc = rotary_rows(ctx, who, "K", a, a.n_kv, size, K, k_stride)) return rc;
        if (int rc = rotary_rows(ctx, who, "Q_out", a, a.n_q, size, Q_out, q_out_stride)) return rc;
        if (int rc = rotary_rows(ctx, who, "K_out", a, a.n_kv, size, K_out, k_out_stride)) return rc;
        if (int rc = rotary_in_place(ctx, who, "Q", a, a.n_q, Q, q_stride, Q_out, q_out_stride)) return rc;
        if (int rc = rotary_in_place(ctx, who, "K", a, a.n_kv, K, k_stride, K_out, k_out_stride)) return rc;
        a.positions = static_cast<const int *>(positions);
        a.q = Q, a.k = K, a.q_out = Q_out, a.k_out = K_out, a.q_stride = q_stride, a.k_stride = k_stride, a.q_out_stride = q_out_stride, a.k_out_stride = k_out_stride;
        return dtype == HIPC_F16 ? rotary_launch<_Float16, false>(ctx, who, a, heads->interleaved) : rotary_launch<float, false>(ctx, who, a, heads->interleaved);
    });
}

int hipc_kv4_append_rotary(hipc_ctx *ctx, const hipc_kv4_cache *cache, const hipc_rotary_heads *heads, int dtype, const void *starts, int64_t total,
                           const void *Q, int64_t q_stride, const void *K, int64_t k_stride, const void *V, int64_t v_stride, void *Q_out, int64_t q_out_stride) {
    return entry(ctx, [&]() -> int {
        const char *who = "hipc_kv4_append_rotary";
        RotaryArgs a{};
        if (int rc = kv4_check(ctx, who, cache)) return rc;
        if (int rc = rotary_check(ctx, who, heads, dtype, total, &a)) return rc;
        HIPC_REQUIRE(ctx, heads->n_kv_heads == cache->n_kv_heads && heads->head_dim == cache->head_dim, "%s: %d kv heads of %d channels, the cache has %d of %d", who, heads->n_kv_heads,
                     heads->head_dim, cache->n_kv_heads, cache->head_dim);
        if (total == 0 || cache->n_seqs == 0) return HIPC_OK;
        const size_t size = dtype == HIPC_F16 ? 2 : 4;
        HIPC_REQUIRE(ctx, starts && aligned(starts, 4), "%s: starts", who);
        if (int rc = rotary_rows(ctx, who, "Q", a, a.n_q, size, Q, q_stride)) return rc;
        if (int rc = rotary_rows(ctx, who, "K", a, a.n_kv, size, K, k_stride)) return rc;
        if (int rc = rotary_rows(ctx, who, "V", a, a.n_kv, size, V, v_stride)) return rc;
        if (int rc = rotary_rows(ctx, who, "Q_out", a, a.n_q, size, Q_out, q_out_stride)) return rc;
        if (int rc = rotary_in_place(ctx, who, "Q", a, a.n_q, Q, q_stride, Q_out, q_out_stride)) return rc;
        a.cache = *cache, a.starts = static_cast<const int *>(starts);
        a.q = Q, a.k = K, a.v = V, a.q_out = Q_out, a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride, a.q_out_stride = q_out_stride;
        return dtype == HIPC_F16 ? rotary_launch<_Float16, true>(ctx, who, a, heads->interleaved) : rotary_launch<float, true>(ctx, who, a, heads->interleaved);
    });
}

}  // extern "C"
