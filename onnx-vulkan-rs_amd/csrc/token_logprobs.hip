// Log probabilities, entropy and the best alternatives of rows of logits (hipc_token_logprobs).
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "lanes.h"

namespace hipc {

namespace {

constexpr int kScratchLogprobs = 7;   // scratch slot of this operator alone
constexpr int kLogWaves = 4;
constexpr int kLogChunk = 1024;       // logits a wavefront holds at a time: 16 a lane
constexpr int kLogWorkgroups = 512;   // at most that many share rows
constexpr int kLogParts = 64;         // ... a row
constexpr int kLogHeld = 4;           // chunks that a wavefront's registers hold
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

// of a row that begins `head` elements behind 16 aligned bytes
__host__ __device__ inline int log_chunks(int vocab, int head, int vec) { return (int)(((int64_t)vocab + head + vec - 1) / vec + kLogChunk / vec - 1) / (kLogChunk / vec); }

// What a stretch of a row amounts to: its largest value m, sum of e = exp(x - m), and sum of e log2(e).
struct LogSum {
    float m, l, w;
};
struct LogPart {
    LogSum sum[kLogWaves];
    uint64_t best[kLogWaves][HIPC_TOP_MAX];   // of each wavefront: keys, largest first; 0 where there are fewer
};

// A logit and its place as one whole number that orders as the alternatives do: by value, the lower id first among equals.
// Never 0 for a value that compares.
__device__ __forceinline__ uint64_t log_key(float x, int id) {
    const uint32_t b = __float_as_uint(x + 0.f);   // (-0 is 0)
    return (uint64_t)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32 | (uint32_t)~id;
}
constexpr uint32_t kLogLowest = 0x007fffffu;   // of -inf
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

// What a wavefront knows of a row's largest logits: keys in its LDS, `count` of them, and the least value that counts. Keys that pass are
// written side by side; they are ranked, and all but the `top` largest dropped, when there is no room left and at the end. The first bar is the
// top-th largest of the lanes' largest logits: at least `top` reach it, and few more. All of this is short loops with little LDS latency
// in a row: it runs a few times in a launch, one wavefront's time after the other's (bar and
// first chunk 1.7 us, ranking 0.5).
struct LogBuffer {
    float stage[kLogChunk];                          // a chunk's logits: the lane's i-th at 64 i + lane
    uint64_t key[kLogBuffer], ranked[HIPC_TOP_MAX];
};

__device__ __forceinline__ uint32_t wave_least(uint32_t v) {
    auto dpp = [](uint32_t x, auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true); };
    v = min(v, dpp(v, std::integral_constant<int, 0xB1>()));
    v = min(v, dpp(v, std::integral_constant<int, 0x4E>()));
    v = min(v, dpp(v, std::integral_constant<int, 0x124>()));
    v = min(v, dpp(v, std::integral_constant<int, 0x128>()));
    auto lane = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
    return min(min(lane(0), lane(16)), min(lane(32), lane(48)));
}
__device__ __forceinline__ uint32_t wave_most(uint32_t v) { return ~wave_least(~v); }
// The largest whole number that at least `top` of the lanes' are at or above (lanes with 0 have none: 0 where there are fewer). The lanes' numbers are
// gone through from the largest on while that takes fewer steps than to count, for every lane, those above it.
__device__ __forceinline__ uint32_t log_reach(uint32_t v, int top) {
    if (top <= 6) {
        uint32_t most = wave_most(v);
        while (most != 0 && __popcll(__ballot(v >= most)) < top) most = wave_most(v < most ? v : 0u);
        return most;
    }
    int above = 0;
#pragma unroll 16
    for (int j = 0; j < 64; j++) above += (uint32_t)__builtin_amdgcn_readlane((int)v, j) > v;
    return wave_least(above < top ? v : 0xffffffffu);
}
__device__ __forceinline__ int log_before(uint64_t lanes) {   // those in front of this one
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0));
}
// the `top` largest of `count` keys of the buffer, the j-th in lane j (one wavefront's LDS accesses are done in their order)
__device__ __forceinline__ uint64_t log_rank(int top, LogBuffer &buffer, int count) {
    const int lane = threadIdx.x & 63;
    constexpr int STEP = 16;
    if (lane < STEP) buffer.key[count + lane] = 0;
    if (lane < top) buffer.ranked[lane] = 0;
#pragma unroll 1
    for (int base = 0; base < count; base += 64) {
        const uint64_t k = base + lane < count ? buffer.key[base + lane] : 0;
        int rank = 0;
#pragma unroll 1
        for (int j = 0; j < count; j += STEP)
#pragma unroll
            for (int e = 0; e < STEP; e++) rank += buffer.key[j + e] > k;
        if (k != 0 && rank < top) buffer.ranked[rank] = k;
    }
    return lane < top ? buffer.ranked[lane] : 0;
}
constexpr int kLogRoom = kLogBuffer - 16;
// The `top` largest keys of the wavefronts' lists, each sorted and with zeros behind its last: a key's rank is its place in its own list and, by
// halving, the number of larger ones in the others.
__device__ __forceinline__ uint64_t log_lists(int top, LogBuffer &buffer, const uint64_t (&lists)[kLogWaves][HIPC_TOP_MAX]) {
    static_assert(HIPC_TOP_MAX == 32 && kLogWaves == 4, "two lists a wavefront's lanes");
    const int lane = threadIdx.x & 63, place = lane & 31, own = lane >> 5;
    uint64_t k[2];
    int larger[2][3] = {};
#pragma unroll
    for (int r = 0; r < 2; r++) k[r] = lists[2 * r + own][place];
    if (lane < top) buffer.ranked[lane] = 0;
#pragma unroll
    for (int s = 0; s < 6; s++) {
        const int step = s == 5 ? 1 : 16 >> s;
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int o = 0; o < 3; o++)
                if (lists[(2 * r + own + 1 + o) & 3][larger[r][o] + step - 1] > k[r]) larger[r][o] += step;
    }
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const int rank = place + larger[r][0] + larger[r][1] + larger[r][2];
        if (k[r] != 0 && rank < top) buffer.ranked[rank] = k[r];
    }
    return lane < top ? buffer.ranked[lane] : 0;
}

struct LogBest {
    int count = 0;
    uint32_t least = 0;   // as in log_key; 0: not known yet
    float bar = -INFINITY;   // the value of `least`

    __device__ __forceinline__ void raise(uint32_t to) {
        if (to > least) least = to, bar = key_value((uint64_t)to << 32);
    }
    __device__ __forceinline__ void rank(int top, LogBuffer &buffer) {
        keep(top, buffer, log_rank(top, buffer, count));
    }
    __device__ __forceinline__ void keep(int top, LogBuffer &buffer, uint64_t list) {
        const int lane = threadIdx.x & 63;
        if (lane < top) buffer.key[lane] = list;
        count = __popcll(__ballot(list != 0));
        const uint64_t lowest = lane_key(list, top - 1);
        if (lowest) raise((uint32_t)(lowest >> 32) + 1);   // (later logits have higher ids: an equal one does not count)
    }
    // A chunk's logits x, of which the lane's largest is `largest`; id(i) is the place of the lane's i-th, below 0 behind the row's ends.
    template <int N, typename Id>
    __device__ __forceinline__ void scan(int top, LogBuffer &buffer, float largest, const float (&x)[N], Id id) {
        const int lane = threadIdx.x & 63;
        uint32_t reach = 0;   // not 0: what at least `top` of this chunk's logits reach, and the bar is no lower
        auto of_chunk = [&] { raise(reach = log_reach((uint32_t)(log_key(largest, 0) >> 32), top)); };
        if (least == 0) of_chunk();
#pragma unroll
        for (int i = 0; i < N; i++) buffer.stage[64 * i + lane] = x[i];
        for (;;) {
            uint32_t pass = 0;
#pragma unroll
            for (int i = 0; i < N; i++) pass |= x[i] >= bar ? 1u << i : 0u;
            int now = count;
#pragma unroll 1
            while (__any(pass != 0) && now <= kLogRoom) {
                const int i = pass ? __builtin_ctz(pass) : 0, at = id(i);
                const bool counts = pass != 0 && at >= 0;
                pass &= pass - 1;
                const uint64_t in = __ballot(counts);
                const int place = now + log_before(in);
                if (counts && place < kLogRoom) buffer.key[place] = log_key(buffer.stage[64 * i + lane], at);
                now += __popcll(in);
            }
            if (now <= kLogRoom) {
                count = now;
                break;
            }
            // no room: what was there is ranked, then the chunk's own bar is taken, and at last (equal values) one key after the other
            if (count > top) {
                rank(top, buffer);
            } else if (reach == 0) {
                of_chunk();
            } else {
                uint64_t last = ~(uint64_t)0, mine = 0;
                const uint64_t had = lane < count ? buffer.key[lane] : 0;
#pragma unroll 1
                for (int j = 0; j < top; j++) {
                    uint64_t own = had < last ? had : 0;
#pragma unroll 1
                    for (int i = 0; i < N; i++) {
                        const float v = buffer.stage[64 * i + lane];
                        const int at = id(i);
                        const uint64_t k = v == v && at >= 0 ? log_key(v, at) : 0;
                        own = k < last && k > own ? k : own;
                    }
                    last = wave_max(own);
                    if (lane == j) mine = last;
                    if (last == 0) break;
                }
                keep(top, buffer, mine);
                break;
            }
        }
        // For the chunks behind, whose ids are higher: of those `top` one of the same value counts no more. (The reach is passed and not the bar, which the
        // list may have raised past it; and not -inf, with which lanes that have nothing which compares are counted.)
        if (reach > kLogLowest) raise(reach + 1);
        if (count >= 2 * top) rank(top, buffer);
    }
};

// what another workgroup stored is read from where it stored it
__device__ __forceinline__ uint64_t key_of_all(const uint64_t *at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ LogSum sum_of_all(const LogSum *at) {
    auto get = [](const float *v) { return __hip_atomic_load(v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    return {get(&at->m), get(&at->l), get(&at->w)};
}

// The `top` largest keys of up to 64 sorted lists (0: none behind a list's last), one per lane, the lane's at `mine` (any address where `have` is
// false). The top-th largest of the lists' first keys is a bar that at least `top` keys reach.
__device__ __forceinline__ uint64_t log_merge(int top, LogBuffer &buffer, const uint64_t *mine, bool have) {
    uint64_t early[4];   // most lists count with fewer keys than these; they are on their way together
#pragma unroll
    for (int r = 0; r < 4; r++) early[r] = key_of_all(mine + min(r, top - 1));
    const uint32_t reach = log_reach(have ? (uint32_t)(early[0] >> 32) : 0u, top);
    const uint64_t bar = reach ? ((uint64_t)reach << 32) - 1 : 0;
    int count = 0;
#pragma unroll 1
    for (int r = 0; r < top; r++) {
        const uint64_t v = r == 0 ? early[0] : r == 1 ? early[1] : r == 2 ? early[2] : r == 3 ? early[3] : key_of_all(mine + r);
        const uint64_t k = have ? v : 0, in = __ballot(k > bar);
        if (!in) break;
        if (count + __popcll(in) > kLogRoom) {   // (equal values)
            const uint64_t list = log_rank(top, buffer, count);
            if ((int)(threadIdx.x & 63) < top) buffer.key[threadIdx.x & 63] = list;
            count = __popcll(__ballot(list != 0));
        }
        if (k > bar) buffer.key[count + log_before(in)] = k;
        count += __popcll(in);
    }
    return log_rank(top, buffer, count);
}

// the lanes' sums as one: each in units of the largest value of all
__device__ __forceinline__ LogSum log_wave(const LogSum &s) {
    const float m = lean_wave_max(s.m);
    const float d = s.m == m ? 0.f : (s.m - m) * kLog2e, f = s.l == 0.f ? 0.f : __builtin_amdgcn_exp2f(d);
    return {m, lean_wave_sum(s.l == 0.f ? 0.f : s.l * f), lean_wave_sum(s.l == 0.f || f == 0.f ? 0.f : f * __builtin_fmaf(s.l, d, s.w))};
}
__device__ __forceinline__ LogSum log_join(const LogSum &a, const LogSum &b) {
    const float m = fmaxf(a.m, b.m);
    // a side without a value above -inf adds nothing (its difference to m may be no number)
    const float da = a.m == m ? 0.f : (a.m - m) * kLog2e, db = b.m == m ? 0.f : (b.m - m) * kLog2e;
    const float fa = a.l == 0.f ? 0.f : __builtin_amdgcn_exp2f(da), fb = b.l == 0.f ? 0.f : __builtin_amdgcn_exp2f(db);
    const float wa = a.l == 0.f || fa == 0.f ? 0.f : fa * __builtin_fmaf(a.l, da, a.w), wb = b.l == 0.f || fb == 0.f ? 0.f : fb * __builtin_fmaf(b.l, db, b.w);
    return {m, (a.l == 0.f ? 0.f : a.l * fa) + (b.l == 0.f ? 0.f : b.l * fb), wa + wb};
}

// `token` is the row's given one and `given` its logit
__device__ __forceinline__ void log_finish(const LogprobArgs &a, int64_t row, int token, float given, const LogSum &s, uint64_t list) {
    const int lane = threadIdx.x & 63;
    // No finite largest value: no distribution (a NaN among the logits has made l one; +inf too, by inf - inf). The
    // largest logit is taken off first: m + log l would be rounded at the size of m, and what is left could lie above 0.
    const float log_l = logf(s.l);
    auto below = [&](float x) { return (x - s.m) - log_l; };
    if (lane == 0) {
        if (a.logprob) a.logprob[row] = token == -1 ? 0.f : token < 0 || token >= a.vocab || s.m == -INFINITY ? NAN : below(given);
        if (a.entropy) a.entropy[row] = s.m == -INFINITY ? NAN : log_l - kLn2 * (s.w / s.l);
    }
    if (lane < a.top) {
        a.top_ids[row * a.top + lane] = list ? key_id(list) : -1;
        a.top_logprobs[row * a.top + lane] = list && s.m != -INFINITY ? below(key_value(list)) : NAN;
    }
}

// A row is read once, by a.parts workgroups. A wavefront streams 1024 logits at a time, the next ones on their way meanwhile, with a running
// maximum and sums per lane and without a barrier. The alternatives cost a comparison per logit; only where one passes the list's last is there
// more to do, which after the first few thousand logits is rare. HELD: a wavefront's share is kLogHeld chunks at most; they are on their way together
// and stay in registers, so that one bar, of them all, is there before the first is compared (64 rows of 100003 in f16: with the
// five best 15.5 us, 16.4 streamed; with twenty 19.1 and 21.3).
template <typename T, bool HELD>
__global__ void __launch_bounds__(64 * kLogWaves, 4) logprob_kernel(const LogprobArgs a) {
    constexpr int VEC = 16 / sizeof(T), LOADS = kLogChunk / 64 / VEC;
    typedef T TV __attribute__((ext_vector_type(VEC)));
    __shared__ LogBuffer buffers[kLogWaves];
    __shared__ LogSum sums[kLogWaves];
    __shared__ uint64_t lists[kLogWaves][HIPC_TOP_MAX];
    __shared__ int last_here;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x / a.parts;
    const int part = (int)(blockIdx.x - row * a.parts);
    LogBuffer &buffer = buffers[wave];

    // the row in pieces of 16 aligned bytes: the first and the last may hold less of it
    const T *x = static_cast<const T *>(a.x) + row * a.row_stride;
    const int head = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const int chunks = log_chunks(a.vocab, head, VEC);
    const int per = (chunks + a.parts * kLogWaves - 1) / (a.parts * kLogWaves);   // of a wavefront, one behind the other
    const int c0 = (part * kLogWaves + wave) * per, c1 = min(c0 + per, chunks);

    // the given token's logit, which any workgroup may turn out to need at the end, is on its way with the others
    const int token = a.logprob ? a.tokens[row] : -1;
    float given = token >= 0 && token < a.vocab ? (float)x[token] : 0.f;

    float m = -INFINITY, l = 0.f, w = 0.f;
    LogBest best;
    // (below 2^31: the vocabulary is at most 2^30)
    auto first_of = [&](int chunk) { return (chunk * LOADS * 64 + lane) * VEC - head; };
    auto load = [&](int chunk, TV (&v)[LOADS]) {
        const int first = first_of(chunk);
        if (chunk != 0 && chunk != chunks - 1) {
#pragma unroll
            for (int e = 0; e < LOADS; e++) v[e] = __builtin_nontemporal_load(reinterpret_cast<const TV *>(x + first + e * 64 * VEC));
            return;
        }
#pragma unroll
        for (int e = 0; e < LOADS; e++) {
            const int at = first + e * 64 * VEC;
            if (at >= 0 && at + VEC <= a.vocab) {
                v[e] = *reinterpret_cast<const TV *>(x + at);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j++) v[e][j] = at + j >= 0 && at + j < a.vocab ? x[at + j] : (T)-INFINITY;
            }
        }
    };
    auto largest = [&](const TV (&v)[LOADS]) {
        float most = -INFINITY;
#pragma unroll
        for (int e = 0; e < LOADS; e++)
#pragma unroll
            for (int j = 0; j < VEC; j++) most = fmaxf(most, (float)v[e][j]);
        return most;
    };
    auto add = [&](const TV (&v)[LOADS]) {
        const float shift = m == -INFINITY ? 0.f : m;   // (subtracted before the scaling: a row at its type's lowest value times log2 e would be an infinity)
        float l2 = 0.f, w2 = 0.f;
#pragma unroll
        for (int e = 0; e < LOADS; e++)
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                // (a masked logit: t = -inf, its exponential 0, and 0 times the held t; a NaN stays one through the exponential)
                const float t = ((float)v[e][j] - shift) * kLog2e, y = __builtin_amdgcn_exp2f(t);
                l2 += y, w2 = __builtin_fmaf(y, fmaxf(t, -200.f), w2);
            }
        l += l2, w += w2;
    };
    auto look = [&](int chunk, float most, const TV (&v)[LOADS]) {
        if (!__any(most >= best.bar)) return;
        const int first = first_of(chunk);
        float values[LOADS * VEC];
#pragma unroll
        for (int i = 0; i < LOADS * VEC; i++) values[i] = (float)v[i / VEC][i % VEC];
        best.scan(a.top, buffer, most, values, [&](int i) -> int {
            const int at = first + i / VEC * 64 * VEC + i % VEC;
            return at >= 0 && at < a.vocab ? at : -1;
        });
    };
    if constexpr (HELD) {
        TV held[kLogHeld][LOADS];
        float most[kLogHeld];
#pragma unroll
        for (int i = 0; i < kLogHeld; i++)
            if (c0 + i < c1) load(c0 + i, held[i]);
#pragma unroll
        for (int i = 0; i < kLogHeld; i++) {
            most[i] = c0 + i < c1 ? largest(held[i]) : -INFINITY;
            m = fmaxf(m, most[i]);
        }
#pragma unroll
        for (int i = 0; i < kLogHeld; i++)
            if (c0 + i < c1) add(held[i]);
        if (a.top > 0) {
            best.raise(log_reach((uint32_t)(log_key(m, 0) >> 32), a.top));
#pragma unroll
            for (int i = 0; i < kLogHeld; i++)
                if (c0 + i < c1) look(c0 + i, most[i], held[i]);
        }
    } else {
        TV now[LOADS], next[LOADS] = {};
        if (c0 < c1) load(c0, now);
        for (int c = c0; c < c1; c++) {
            if (c + 1 < c1) load(c + 1, next);
            const float most = largest(now);
            if (most > m) {
                const float f = l == 0.f ? 0.f : __builtin_amdgcn_exp2f((m - most) * kLog2e);
                w = f == 0.f ? 0.f : f * __builtin_fmaf(l, (m - most) * kLog2e, w), l *= f;
                m = most;
            }
            add(now);
            if (a.top > 0) look(c, most, now);
#pragma unroll
            for (int e = 0; e < LOADS; e++) now[e] = next[e];
        }
    }

    HIPC_PIN_VGPR(given);

    // lanes, then wavefronts
    LogSum s{m, l, w};
    s = log_wave(s);
    uint64_t list = a.top > 0 && best.count > 0 ? log_rank(a.top, buffer, best.count) : 0;
    if (a.parts == 1) {
        if (lane == 0) sums[wave] = s;
        if (lane < HIPC_TOP_MAX) lists[wave][lane] = list;
        __syncthreads();
        if (wave != 0) return;
#pragma unroll 1
        for (int v = 1; v < kLogWaves; v++) s = log_join(s, sums[v]);
    } else {
        // several workgroups: the one that comes last joins what they found
        LogPart *all = a.part + row * a.parts;
        auto put = [](auto *to, auto v) { __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        LogSum *sum = &all[part].sum[wave];
        if (lane == 0) put(&sum->m, s.m), put(&sum->l, s.l), put(&sum->w, s.w);
        if (lane < a.top) put(&all[part].best[wave][lane], list);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the stores are where everyone sees them
        __syncthreads();
        if (tid == 0) last_here = __hip_atomic_fetch_add(a.arrived + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)a.parts - 1;
        if (wave != 0 && a.top == 0) return;
        if (a.top > 0) __syncthreads();
        if (!last_here) return;
        if (tid == 0) put(a.arrived + row, 0u);   // for the next call
        static_assert(kLogParts * kLogWaves <= 64 * kLogWaves, "a list per thread");
        LogSum found[kLogWaves];
        if (wave == 0) {
#pragma unroll
            for (int v = 0; v < kLogWaves; v++) found[v] = sum_of_all(&all[min(lane, a.parts - 1)].sum[v]);
        }
        if (a.top > 0) {
            const bool have = tid < a.parts * kLogWaves;
            list = log_merge(a.top, buffer, &all[have ? tid / kLogWaves : 0].best[tid % kLogWaves][0], have);
            if (lane < HIPC_TOP_MAX) lists[wave][lane] = list;
        }
        if (wave == 0) {
            s = found[0];
#pragma unroll
            for (int v = 1; v < kLogWaves; v++) s = log_join(s, found[v]);
            if (lane >= a.parts) s = {-INFINITY, 0.f, 0.f};
            s = log_wave(s);
        }
        if (a.top > 0) __syncthreads();
        if (wave != 0) return;
    }
    if (a.top > 0) list = log_lists(a.top, buffer, lists);
    log_finish(a, row, token, given, s, list);
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
        // few rows are shared by several workgroups, each wavefront of which has 1024 logits at least
        const size_t count_bytes = kLogWorkgroups * sizeof(uint32_t), bytes = count_bytes + kLogWorkgroups * sizeof(LogPart);
        if (scratch_fits(ctx, kScratchLogprobs, bytes))
            a.parts = (int)std::max<int64_t>(1, std::min<int64_t>({kLogWorkgroups / rows, ceil_div(vocab, kLogWaves * kLogChunk), kLogParts}));
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
        HIPC_REFUSE(ctx, !grid_fits(rows * a.parts, 64 * kLogWaves), "%s: %lld rows: too many for one call", who, (long long)rows);
        const unsigned grid = (unsigned)(rows * a.parts);
        auto launch = [&](auto held) {
            constexpr bool HELD = decltype(held)::value;
            if (dtype == HIPC_F16) hipLaunchKernelGGL((logprob_kernel<_Float16, HELD>), grid, 64 * kLogWaves, 0, ctx->stream, a);
            else hipLaunchKernelGGL((logprob_kernel<float, HELD>), grid, 64 * kLogWaves, 0, ctx->stream, a);
        };
        // (rows may begin anywhere within 16 bytes)
        const int vec = dtype == HIPC_F16 ? 8 : 4;
        if (log_chunks(a.vocab, vec - 1, vec) <= kLogHeld * kLogWaves * a.parts) launch(std::true_type());
        else launch(std::false_type());
        HIPC_LAUNCHED(ctx);
        return HIPC_OK;
    });
}

}  // extern "C"
