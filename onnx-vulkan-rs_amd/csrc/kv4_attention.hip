// Attention of the newest tokens of many sequences over the paged 4-bit cache (hipc_kv4_attention).
#include <algorithm>
#include <type_traits>

#include "kv4.h"
#include "lanes.h"

namespace hipc {

namespace {

struct Kv4Attend {
    hipc_kv4_cache cache;
    const void *q;
    void *y;
    int64_t q_stride, y_stride;
    int tokens, n_q_heads, group, window, row_blocks, wide;   // wide: rows of Q and Y on 16 bytes
    float scale;
    float *parts;        // [workgroup][2] parts of a unit: rows x channels sums, then (maximum, sum) pairs
    uint32_t *arrived;   // [workgroup]: parts of the unit that began here and went on; all zero between calls
};

typedef _Float16 kvh8 __attribute__((ext_vector_type(8)));
typedef float kvf4 __attribute__((ext_vector_type(4)));
typedef uint32_t kvu2 __attribute__((ext_vector_type(2)));
typedef uint32_t kvu4 __attribute__((ext_vector_type(4)));
typedef int kvi2 __attribute__((ext_vector_type(2)));

constexpr int kScratchKv4 = 6;     // scratch slot of this operator alone
constexpr int kKv4Rows = 16;       // query rows of a unit
constexpr int kKv4Tile = 64;       // keys a wavefront takes at a time
constexpr int kKv4PerCu = 8;       // wavefronts
constexpr float kKv4Log2e = 1.4426950408889634f;
constexpr float kKv4RescaleAt = 8.f;   // the running maximum may fall behind by 2^8 before sums are rescaled ...
constexpr float kKv4Up = 7.f;          // ... and weights are kept 2^7 times as large: up to 2^15, so that two f16 terms hold 22 bits of more of them

// the four groups of 16 lanes, in all lanes
__device__ __forceinline__ float groups_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The key tiles a sequence's newest tokens see: [first, first + count).
struct Kv4Span {
    int length, first, count;
};
__device__ __forceinline__ Kv4Span kv4_span_of(const Kv4Attend &a, int length) {
    const int held = kv4_held(a.cache, length);
    const int begin = a.window > 0 ? max(length - a.tokens - a.window + 1, 0) : 0;
    return {length, begin / kKv4Tile, held > begin ? (held + kKv4Tile - 1) / kKv4Tile - begin / kKv4Tile : 0};
}

__device__ __forceinline__ int kv4_span_length(const Kv4Attend &a, int seq) { return a.cache.n_pages > 0 ? kv4_length(a.cache, min(seq, a.cache.n_seqs - 1)) : 0; }
__device__ __forceinline__ Kv4Span kv4_span(const Kv4Attend &a, int seq) { return kv4_span_of(a, kv4_span_length(a, seq)); }
// body(base, spans) for the sequences in chunks of 64, a lane's is base + lane (the last one's, behind it): the first 64 are there, of
// the others four chunks' lengths are on their way at once. Ends where body is true.
template <typename Body>
__device__ __forceinline__ void kv4_sequences(const Kv4Attend &a, const Kv4Span &early, Body body) {
    if (body(0, early)) return;
    const int lane = threadIdx.x & 63;
    for (int base = 64; base < a.cache.n_seqs; base += 256) {
        int length[4];
#pragma unroll
        for (int e = 0; e < 4; e++) length[e] = kv4_span_length(a, base + 64 * e + lane);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (base + 64 * e < a.cache.n_seqs && body(base + 64 * e, kv4_span_of(a, length[e]))) return;
    }
}

// A unit: (sequence, kv head, block of 16 query rows), counted in this order.
struct Kv4Unit {
    Kv4Span span;
    int seq, inner;       // inner = kv head * row_blocks + block
    int64_t before;       // steps of all units in front of it
};
// a division of whole numbers that are hardly ever beyond 32 bits (one of 64 bits is some 100 instructions)
__device__ __forceinline__ int64_t kv4_div(int64_t x, int64_t y) { return ((uint64_t)(x | y) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y; }
// Steps of a unit: its tiles, or (cut > 0) its parts of up to `cut` tiles. The unit that step number `at` of all units' belongs to.
__device__ __forceinline__ int kv4_steps(int tiles, int cut) { return cut > 0 ? (tiles + cut - 1) / cut : tiles; }
__device__ __forceinline__ bool kv4_find(const Kv4Attend &a, const Kv4Span &early, int per_seq, int64_t at, int cut, Kv4Unit *u) {
    const int lane = threadIdx.x & 63;
    int64_t before = 0;
    bool found = false;
    kv4_sequences(a, early, [&](int base, const Kv4Span &s) {
        const int n = base + lane < a.cache.n_seqs ? kv4_steps(s.count, cut) : 0;
        const int sum = wave_scan(n);
        const uint64_t over = __ballot(before + (int64_t)sum * per_seq > at);
        if (over) {
            const int l = __builtin_ctzll(over), steps = __builtin_amdgcn_readlane(n, l);
            u->span = {__builtin_amdgcn_readlane(s.length, l), __builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.count, l)};
            const int64_t first = before + (int64_t)(__builtin_amdgcn_readlane(sum, l) - steps) * per_seq;
            u->seq = base + l;
            u->inner = (int)kv4_div(at - first, steps);
            u->before = first + (int64_t)u->inner * steps;
            found = true;
        }
        before += (int64_t)__builtin_amdgcn_readlane(sum, 63) * per_seq;
        return over != 0;
    });
    return found;
}
// the unit behind the last one of its sequence, which ended at step `at`
__device__ __forceinline__ bool kv4_next(const Kv4Attend &a, int64_t at, int cut, Kv4Unit *u) {
    const int lane = threadIdx.x & 63;
    for (int base = u->seq + 1; base < a.cache.n_seqs; base += 64) {
        const Kv4Span s = kv4_span(a, base + lane);
        const uint64_t has = __ballot(base + lane < a.cache.n_seqs && kv4_steps(s.count, cut) > 0);
        if (!has) continue;
        const int l = __builtin_ctzll(has);
        u->span = {__builtin_amdgcn_readlane(s.length, l), __builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.count, l)};
        u->seq = base + l, u->inner = 0, u->before = at;
        return true;
    }
    return false;
}
// steps of all units
__device__ __forceinline__ int64_t kv4_total(const Kv4Attend &a, const Kv4Span &early, int per_seq, int cut, float *longest) {
    const int lane = threadIdx.x & 63;
    int64_t total = 0;
    float most = 0.f;
    kv4_sequences(a, early, [&](int base, const Kv4Span &s) {
        const int c = base + lane < a.cache.n_seqs ? s.count : 0;
        total += (int64_t)__builtin_amdgcn_readlane(wave_scan(kv4_steps(c, cut)), 63) * per_seq;
        most = fmaxf(most, lean_wave_max((float)c));
        return false;
    });
    *longest = most;
    return total;
}

// rows that see nothing for want of keys
template <typename T, int HD>
__device__ void kv4_zero_rows(const Kv4Attend &a, const Kv4Span &early) {
    const int lane = threadIdx.x & 63;
    kv4_sequences(a, early, [&](int base, const Kv4Span &span) {
        for (uint64_t none = __ballot(base + lane < a.cache.n_seqs && span.count == 0); none; none &= none - 1) {
            const int64_t s = base + __builtin_ctzll(none);
            for (int r = 0; r < a.tokens; r++)
                for (int i = threadIdx.x; i < a.n_q_heads * HD; i += blockDim.x) static_cast<T *>(a.y)[(s * a.tokens + r) * a.y_stride + i] = (T)0.f;
        }
        return false;
    });
}

// One launch for everything. Where there are fewer units than workgroups, units are cut into parts of at most so many tiles that there is a
// workgroup for each; otherwise all units' tiles are laid end to end and dealt to the workgroups in equal runs. So sequences of any lengths
// keep the whole device busy. A unit that lies in one part is finished there; of one that lies in several the workgroup that comes last joins the
// parts, in their order. (Runs everywhere: a workgroup mostly has the end of one unit and the beginning of another, and starting on a unit and
// leaving it costs some 6 us beside 3 us a tile.)
//
// W: a unit's wavefronts. With four a workgroup each takes every fourth tile and they add up in LDS; where units are many a workgroup is one wavefront, and
// its run of tiles waits for no other's. (us, four / one; 32 / 8 heads of 128 in f16: 20 sequences of up to 8000 27.9 / 32.7, 48 of up to
// 4000 35.7 / 33.2, 64 of up to 3200 47.8 / 33.6, 256 of up to 800 106 / 56, 1024 of up to 200 189 / 76.)
//
// A wavefront takes 64 keys of one kv head at a time, for 16 query rows (tokens times the heads of the group):
//   S^T = K Q^T     16x16x32: of tile t (16 keys) row m is key 16 (m / 4) + 4 t + m % 4, so that a lane ends up with the scores of 16
//                   consecutive keys of one query (query = lane % 16, keys 16 (lane / 16) ..): two steps of the second product
//   O^T = V^T P^T   P as the lanes hold it, V^T by the transposing 4-bit load from the packed rows in LDS (16 keys of a channel per lane)
// The codes become f16 values on their way into the operands (exactly what the cache stands for), weights are two f16 terms, f32 queries
// two terms of the row times a power of two. Keys come straight from memory into operand registers, a tile ahead; values (codes, and
// the parameters of the keys that are seen, zeros for the others) pass through the wavefront's own LDS, without a barrier.
template <int HD, int QT, int W>
__global__ void __launch_bounds__(64 * W, HD <= 128 ? 2 : 1) kv4_attend_kernel(const Kv4Attend a) {
    constexpr int WPL = HD / 32;                              // words of codes of a key per lane; also groups of a row
    constexpr int UNITS = HD <= 32 ? 2 : HD <= 64 ? 4 : HD <= 128 ? 8 : 16;   // 8-byte units of an LDS row of codes
    constexpr int PER = 16 / UNITS;                           // rows of 128 bytes
    constexpr int NP = WPL % 4 == 0 ? WPL / 4 : WPL <= 2 ? 1 : WPL;           // parameters of a key a lane needs for its words
    constexpr int MT = HD / 16;                               // 16-channel tiles
    constexpr int CODES = kKv4Tile * UNITS * 8, PARAMS = WPL * 256;           // LDS of a wavefront
    constexpr int SUMS = W * HD * kKv4Rows * 4;
    constexpr int STAGE = W * (CODES + PARAMS);
    typedef typename std::conditional<QT == 1, _Float16, float>::type T;
    __shared__ __attribute__((aligned(1024))) char smem[STAGE > SUMS ? STAGE : SUMS];
    __shared__ float ml[W][2][kKv4Rows];
    __shared__ int last_here;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, q4 = lane >> 4;
    char *codes = smem + wave * (CODES + PARAMS), *params = codes + CODES;
    const int shift = 31 - __builtin_clz((unsigned)a.cache.page_size), page_mask = a.cache.page_size - 1;
    const int per_seq = a.cache.n_kv_heads * a.row_blocks;
    const Kv4Unpack unpack;

    // at least a tile for each wavefront, and long units in few enough parts that joining them is not the longer half
    const int groups = (int)gridDim.x;
    const Kv4Span early = kv4_span(a, min(lane, a.cache.n_seqs - 1));   // of the first 64 sequences, which mostly are all
    float longest, same;
    const int64_t tiles = kv4_total(a, early, per_seq, 0, &longest);
    if (tiles == 0) {
        if (blockIdx.x == gridDim.x - 1) kv4_zero_rows<T, HD>(a, early);
        return;
    }
    const int64_t even = kv4_div(tiles + groups - 1, groups);
    const int least = max(W, (int)sqrtf(longest * (1.f / 7.f)));
    int64_t share = even > least ? even : least;
    int cut = 0;
    if (kv4_total(a, early, per_seq, 1 << 30, &same) <= groups) {
        cut = (int)share;
        for (;;) {   // (longer parts make fewer of them; with one a unit it ends)
            const int64_t parts = kv4_total(a, early, per_seq, cut, &same);
            if (parts <= groups) break;
            cut = max(cut + 1, (int)min((float)cut * (float)parts / (float)groups, longest));
        }
        share = 1;
    }
    int64_t at = share * blockIdx.x;
    Kv4Unit u;
    if (blockIdx.x == gridDim.x - 1) kv4_zero_rows<T, HD>(a, early);
    if (!kv4_find(a, early, per_seq, at, cut, &u)) return;
    const int64_t run1 = at + share;
    for (;;) {
        const Kv4Span span = u.span;
        const int kvh = u.inner / a.row_blocks, block = u.inner - kvh * a.row_blocks;
        // its tiles of this workgroup
        const int steps = kv4_steps(span.count, cut);
        int from = (int)(at - u.before), to = run1 - u.before < steps ? (int)(run1 - u.before) : steps;
        if (cut > 0) {   // in parts as equal as whole tiles allow
            const int part = from, each = (span.count + steps - 1) / steps;
            from = min(part * each, span.count), to = min(from + each, span.count);
        }

        // the lane's query row
        const int rows = min(a.tokens * a.group - block * kKv4Rows, kKv4Rows);
        const int row = block * kKv4Rows + n, token = min(row, a.tokens * a.group - 1) / a.group, g = row - token * a.group;
        const bool mine = n < rows;
        const int pos = span.length - a.tokens + token;
        const int lane_begin = a.window > 0 ? max(pos - a.window + 1, 0) : 0, lane_end = mine ? pos + 1 : 0;
        const int pos0 = span.length - a.tokens + block * kKv4Rows / a.group;                       // the first row's and the last's
        const int pos1 = span.length - a.tokens + (block * kKv4Rows + rows - 1) / a.group;
        const int any_begin = a.window > 0 ? max(pos0 - a.window + 1, 0) : 0, all_begin = a.window > 0 ? max(pos1 - a.window + 1, 0) : 0;

        float qx[WPL][8];
        {
            const T *q = static_cast<const T *>(a.q) + ((int64_t)u.seq * a.tokens + (mine ? token : 0)) * a.q_stride + (int64_t)(kvh * a.group + (mine ? g : 0)) * HD;
#pragma unroll
            for (int w = 0; w < WPL; w++) kv4_load8(q + 8 * (q4 * WPL + w), a.wide, qx[w]);
        }

        kvf4 o[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) o[i] = kvf4{};
        float m = -INFINITY, l = 0.f;

        // A tile's loads. Blocks of 16 positions lie in one page: block n / 4 for the lane's keys, block q4 for the parameters of its value row.
        // Page numbers are asked for two tiles ahead, values and keys one: the values' registers are free once they are in LDS, the keys' once they
        // are multiplied.
        uint32_t k_codes[4][WPL], k_params[4][NP], v_codes[WPL][4], v_params[WPL];
        const int *table = static_cast<const int *>(a.cache.table) + (int64_t)u.seq * a.cache.table_width;
        auto page_at = [&](int tile, int block) {
            const int entry = ((span.first + tile) * kKv4Tile + 16 * block) >> shift, last = (int)a.cache.table_width - 1, page = table[min(entry, last)];
            return entry <= last ? page : -1;
        };
        auto is_page = [&](int page) { return page >= 0 && page < a.cache.n_pages; };
        auto row_of = [&](int page, int key) -> int64_t {
            return (((int64_t)(is_page(page) ? page : 0) * a.cache.n_kv_heads + kvh) << shift) + (key & page_mask);
        };
        auto load_values = [&](int tile, int page) {   // page: of block q4
            const int key0 = (span.first + tile) * kKv4Tile;
            const int64_t row = row_of(page, key0 + lane);
            const uint32_t *vp = static_cast<const uint32_t *>(a.cache.v_params) + row * WPL;
#pragma unroll
            for (int i = 0; i < WPL; i++) v_params[i] = vp[i];
            // 16-byte chunks of the 64 rows, in their order: chunk 64 e + lane is of row (64 e + lane) / WPL
            auto row_at = [&](int r) -> int64_t {   // uniform r: the lane that has that row
                return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(row >> 32), r) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)row, r));
            };
            const char *vc = static_cast<const char *>(a.cache.v_codes);
#pragma unroll
            for (int e = 0; e < WPL; e++) {
                const char *at;
                if (WPL == 4 || WPL == 8) {   // the rows of a load lie in one block: side by side
                    at = vc + row_at(64 / WPL * e) * (HD / 2) + lane * 16;
                } else if (WPL == 1) {
                    at = vc + row * (HD / 2);
                } else {
                    const int id = 64 * e + lane, r = id / WPL;
                    const uint32_t lo = __shfl((uint32_t)row, r), hi = __shfl((uint32_t)(row >> 32), r);
                    at = vc + (int64_t)((uint64_t)hi << 32 | lo) * (HD / 2) + (id - r * WPL) * 16;
                }
                const kvu4 w = *reinterpret_cast<const kvu4 *>(at);
#pragma unroll
                for (int j = 0; j < 4; j++) v_codes[e][j] = w[j];
            }
        };
        auto load_keys = [&](int tile, int page) {   // page: of block n / 4
            const int64_t row = row_of(page, (span.first + tile) * kKv4Tile + 16 * (n >> 2) + (n & 3));
            const uint32_t *kc = reinterpret_cast<const uint32_t *>(static_cast<const char *>(a.cache.k_codes) + row * (HD / 2)) + q4 * WPL;
            const uint32_t *kp = static_cast<const uint32_t *>(a.cache.k_params) + row * WPL;
#pragma unroll
            for (int t = 0; t < 4; t++) {
#pragma unroll
                for (int w = 0; w < WPL; w++) k_codes[t][w] = kc[t * 4 * (HD / 8) + w];
#pragma unroll
                for (int i = 0; i < NP; i++) k_params[t][i] = kp[t * 4 * WPL + (WPL % 4 == 0 ? q4 * (WPL / 4) + i : (q4 * WPL + i) / 4)];
            }
        };
        int tile = from + wave, v_page = 0, k_page = 0, v_page1 = 0, k_page1 = 0;
        if (tile < to) v_page = page_at(tile, q4), k_page = page_at(tile, n >> 2);
        if (tile + W < to) v_page1 = page_at(tile + W, q4), k_page1 = page_at(tile + W, n >> 2);
        if (tile < to) load_values(tile, v_page), load_keys(tile, k_page);
        // the queries as operands, while the first tile is on its way
        kvh8 qf[WPL][QT];
        float c2 = fabsf(a.scale) * kKv4Log2e;
        {
            const float sign = a.scale < 0.f ? -1.f : 1.f;
            float most = 0.f;
#pragma unroll
            for (int w = 0; w < WPL; w++)
#pragma unroll
                for (int j = 0; j < 8; j++) qx[w][j] *= sign, most = fmaxf(most, fabsf(qx[w][j]));
            if (QT == 2) {
                most = groups_max(most);
                // The row's largest value into [2^14, 2^15); an infinity stays where it is. And no further up than leaves the scores' factor an ordinary
                // number: at 0 it would make NaN of what is hidden (scores of -inf). Rows that this stops have scores of 0 to working precision.
                const int up = most > 0.f && most < INFINITY ? min(14 - ilogbf(most), 126 + ilogbf(fminf(c2, 0x1p126f))) : 0;
                c2 = ldexpf(c2, -up);
#pragma unroll
                for (int w = 0; w < WPL; w++)
#pragma unroll
                    for (int j = 0; j < 8; j++) qx[w][j] = ldexpf(qx[w][j], up);
            }
#pragma unroll
            for (int w = 0; w < WPL; w++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float v = qx[w][(j & 1) * 4 + (j >> 1)];   // the order the codes unpack in: 0 4 1 5 2 6 3 7
                    const _Float16 hi = (_Float16)v;
                    qf[w][0][j] = hi;
                    if (QT == 2) qf[w][QT - 1][j] = (_Float16)(v - (float)hi);
                }
        }
        for (; tile < to; tile += W) {
            const bool more = tile + W < to;
            const int key0 = (span.first + tile) * kKv4Tile;
            const bool v_there = is_page(v_page), masked = key0 + kKv4Tile > pos0 + 1 || key0 < all_begin || !__all(v_there);
            int v_page2 = 0, k_page2 = 0;
            if (tile + 2 * W < to) v_page2 = page_at(tile + 2 * W, q4), k_page2 = page_at(tile + 2 * W, n >> 2);
            // values to LDS: codes in 8-byte units, unit x of row r at x ^ (r / PER), so that the 16 rows of a transposing load lie in different banks
#pragma unroll
            for (int e = 0; e < WPL; e++) {
                const int id = 64 * e + lane, r = id / WPL, c = id - r * WPL, x = (r / PER) & (UNITS - 1);
                const kvu4 w = x & 1 ? kvu4{v_codes[e][2], v_codes[e][3], v_codes[e][0], v_codes[e][1]} : kvu4{v_codes[e][0], v_codes[e][1], v_codes[e][2], v_codes[e][3]};
                *reinterpret_cast<kvu4 *>(codes + r * (UNITS * 8) + (c ^ (x >> 1)) * 16) = w;
            }
            // parameters of eight keys of a group together, in pairs as the codes unpack: scales of keys (i, i + 4), then lowest values
            bool seen = true;
            uint32_t odd_groups = 0;   // (several tokens) groups of the lane's key whose parameters are not finite
            if (masked) {
                const int key = key0 + lane;
                seen = key < span.length && key >= any_begin && v_there;
                if (a.tokens > 1) {
#pragma unroll
                    for (int i = 0; i < WPL; i++)
                        if (((((v_params[i] & 0x7c007c00u) + 0x04000400u) & 0x80008000u) != 0) && seen) odd_groups |= 1u << i;
                }
            }
#pragma unroll
            for (int i = 0; i < WPL; i++) {
                const uint32_t w = seen && !(odd_groups >> i & 1) ? v_params[i] : 0u;
                char *to_lds = params + i * 256 + (lane >> 3) * 32 + (lane & 3) * 4 + ((lane >> 2) & 1) * 2;
                *reinterpret_cast<uint16_t *>(to_lds) = (uint16_t)w;
                *reinterpret_cast<uint16_t *>(to_lds + 16) = (uint16_t)(w >> 16);
            }
            if (more) load_values(tile + W, v_page1);

            kvf4 s[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                s[t] = kvf4{};
#pragma unroll
                for (int w = 0; w < WPL; w++) {
                    const kvh2 p = __builtin_bit_cast(kvh2, k_params[t][WPL % 4 == 0 ? w / 4 : NP == 1 ? 0 : w]);
                    kvh2 v[4];
                    unpack(k_codes[t][w], kvh2{p.x, p.x}, kvh2{p.y, p.y}, v);
                    const kvh8 kf = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
#pragma unroll
                    for (int e = QT - 1; e >= 0; e--) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[w][e], s[t], 0, 0, 0);
                }
            }
            if (more) load_keys(tile + W, k_page1);
            if (masked) {
                const uint64_t there = __ballot(v_there);
                const bool block_there = (there >> (16 * q4)) & 1;   // the lane's 16 keys are one block's
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int k = key0 + 16 * q4 + 4 * t + r;
                        s[t][r] = block_there && k >= lane_begin && k < lane_end ? s[t][r] : -INFINITY;
                    }
            }
            float mx = s[0][0];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) mx = fmaxf(mx, s[t][r]);
            mx = groups_max(mx) * c2;
            if (__any(mx > m + kKv4RescaleAt)) {
                const float grown = mx > m + kKv4RescaleAt ? mx : m, keep = grown == m ? 1.f : __builtin_amdgcn_exp2f(m - grown);   // (a row goes by its own scores)
                m = grown, l *= keep;
#pragma unroll
                for (int i = 0; i < MT; i++) o[i] *= keep;
            }
            const float down = (m == -INFINITY ? 0.f : m) - kKv4Up;
            kvh8 p[2][2];   // [step][term]
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int f = 0; f < 2; f++) {
                        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * h + f][r], c2, -down));
                        const _Float16 hi = (_Float16)w;
                        l += w;
                        p[h][0][2 * r + f] = hi, p[h][1][2 * r + f] = (_Float16)(w - (float)hi);
                    }

#pragma unroll
            for (int i = 0; i < MT; i++) {
                // (row 16 q4 + n of the codes, unit i; the result: this lane's channel 16 i + n, keys 16 q4 .. + 15)
                const int r = 16 * q4 + n;
                const kvi2 w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) kvi2 *)(codes + r * (UNITS * 8) + ((i ^ (r / PER)) & (UNITS - 1)) * 8));
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const char *pp = params + (i / 2) * 256 + (2 * q4 + h) * 32;
                    const kvu4 sc = *reinterpret_cast<const kvu4 *>(pp), lo = *reinterpret_cast<const kvu4 *>(pp + 16);
                    kvh2 v[4];
                    auto pair = [](uint32_t bits) { return __builtin_bit_cast(kvh2, bits); };
                    unpack((uint32_t)w[h], [&](int j) { return pair(sc[j]); }, [&](int j) { return pair(lo[j]); }, v);
                    const kvh8 vf = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, p[h][1], o[i], 0, 0, 0);
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, p[h][0], o[i], 0, 0, 0);
                }
            }
            if (masked && a.tokens > 1) {
                // a key with parameters that are not finite was left out above: what rows that see it get is NaN, the other tokens' rows nothing
                for (uint64_t left = __ballot(odd_groups != 0); left; left &= left - 1) {
                    const int b = __builtin_ctzll(left), k = key0 + b;
                    const uint32_t odd = __builtin_amdgcn_readlane(odd_groups, b);
                    const bool sees = k >= lane_begin && k < lane_end;
#pragma unroll
                    for (int i = 0; i < MT; i++)
                        if ((odd >> (i / 2) & 1) && sees) o[i] += kvf4{NAN, NAN, NAN, NAN};
                }
            }
            v_page = v_page1, k_page = k_page1, v_page1 = v_page2, k_page1 = k_page2;
        }

        // the wavefronts' sums, joined in LDS
        l = groups_sum(l);
        __syncthreads();   // (the codes' LDS becomes the sums')
        if (q4 == 0) ml[wave][0][n] = m, ml[wave][1][n] = l;
        __syncthreads();
        float best = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) best = fmaxf(best, ml[w][0][n]);
#pragma unroll
        for (int w = 0; w < W; w++) sum += ml[w][1][n] == 0.f ? 0.f : ml[w][1][n] * __builtin_amdgcn_exp2f(ml[w][0][n] - best);
        {
            const float keep = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - best);
            float4 *mine_o = reinterpret_cast<float4 *>(smem) + wave * MT * 64 + lane;
#pragma unroll
            for (int i = 0; i < MT; i++) mine_o[i * 64] = l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o[i][0] * keep, o[i][1] * keep, o[i][2] * keep, o[i][3] * keep);
        }
        __syncthreads();
        const bool whole = from == 0 && to == u.span.count;
        auto store_row = [&](int r, int c, const float4 &v, float inv) {
            const int rr = block * kKv4Rows + r, tk = rr / a.group;
            T *y = static_cast<T *>(a.y) + ((int64_t)u.seq * a.tokens + tk) * a.y_stride + (int64_t)(kvh * a.group + rr - tk * a.group) * HD + c;
            typedef T T4 __attribute__((ext_vector_type(4)));
            const T4 out = {(T)(v.x * inv), (T)(v.y * inv), (T)(v.z * inv), (T)(v.w * inv)};
            if (a.wide) {
                *reinterpret_cast<T4 *>(y) = out;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) y[j] = out[j];
            }
        };
        // workgroup w's part of a unit that began in an earlier run (0), or begins here and goes on (1): [row][channel] sums, then maxima and sums
        auto part_of = [&](int64_t w, int which) { return a.parts + (w * 2 + which) * (int64_t)(kKv4Rows * (HD + 2)); };
        float *part = part_of(blockIdx.x, cut == 0 && from == 0 ? 1 : 0);
        // two floats at a time, stored where (and read from where) every workgroup sees them
        auto put = [](float *to_pair, float x, float y) {
            __hip_atomic_store(reinterpret_cast<uint64_t *>(to_pair), (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        auto get = [](const float *pair) {
            const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(pair), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
        };
        for (int i = wave; i < MT; i += W) {   // thread (i, lane): channels 16 i + 4 q4 .. + 3 of row n
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float4 x = reinterpret_cast<const float4 *>(smem)[(w * MT + i) * 64 + lane];
                v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
            }
            if (!mine) continue;
            if (whole) {
                store_row(n, 16 * i + 4 * q4, v, sum == 0.f ? 0.f : 1.f / sum);
            } else {
                float *to_part = part + n * HD + 16 * i + 4 * q4;
                put(to_part, v.x, v.y), put(to_part + 2, v.z, v.w);
            }
        }
        if (!whole) {
            if (wave == 0 && q4 == 0 && mine) {
                put(part + kKv4Rows * HD + 2 * n, best, sum);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wavefront's stores are where everyone sees them
            __syncthreads();
            const int64_t w0 = kv4_div(u.before, share), w1 = kv4_div(u.before + steps - 1, share);   // the workgroups that have parts of it
            if (tid == 0) {
                const uint32_t others = __hip_atomic_fetch_add(a.arrived + w0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last_here = others == (uint32_t)(w1 - w0);
                if (last_here) __hip_atomic_store(a.arrived + w0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next call
            }
            __syncthreads();
            if (last_here) {
                for (int i = tid; i < rows * (HD / 4); i += 64 * W) {
                    const int r = i / (HD / 4), c = (i - r * (HD / 4)) * 4;
                    float top = -INFINITY, all = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    constexpr int N = 8;   // parts on their way together
                    for (int64_t w = w0; w <= w1; w += N) {
                        float2 msum[N], x01[N], x23[N];
#pragma unroll
                        for (int e = 0; e < N; e++) {
                            const int64_t at_w = w + e < w1 ? w + e : w1;
                            const float *x = part_of(at_w, cut == 0 && at_w == w0);
                            msum[e] = get(x + kKv4Rows * HD + 2 * r), x01[e] = get(x + r * HD + c), x23[e] = get(x + r * HD + c + 2);
                            if (w + e > w1) msum[e] = make_float2(-INFINITY, 0.f);
                        }
                        float higher = top;
#pragma unroll
                        for (int e = 0; e < N; e++) higher = fmaxf(higher, msum[e].x);
                        const float back = all == 0.f ? 0.f : __builtin_amdgcn_exp2f(top - higher);
                        top = higher, all *= back, v.x *= back, v.y *= back, v.z *= back, v.w *= back;
#pragma unroll
                        for (int e = 0; e < N; e++) {
                            if (msum[e].y == 0.f) continue;   // nothing the row sees
                            const float keep = __builtin_amdgcn_exp2f(msum[e].x - top);
                            all += msum[e].y * keep, v.x += x01[e].x * keep, v.y += x01[e].y * keep, v.z += x23[e].x * keep, v.w += x23[e].y * keep;
                        }
                    }
                    store_row(r, c, v, all == 0.f ? 0.f : 1.f / all);
                }
            }
        }
        __syncthreads();   // LDS is free for the next unit

        at = u.before + steps;
        if (at >= run1) break;
        if (++u.inner < per_seq) u.before = at;
        else if (!kv4_next(a, at, cut, &u)) break;
    }
}

template <int HD>
void kv4_launch(hipc_ctx *ctx, const Kv4Attend &a, int dtype, bool alone) {
    auto launch = [&](auto waves) {
        constexpr int W = decltype(waves)::value;
        const unsigned grid = kKv4PerCu * ctx->cu_count / W;
        if (dtype == HIPC_F16) hipLaunchKernelGGL((kv4_attend_kernel<HD, 1, W>), grid, 64 * W, 0, ctx->stream, a);
        else hipLaunchKernelGGL((kv4_attend_kernel<HD, 2, W>), grid, 64 * W, 0, ctx->stream, a);
    };
    if (alone) launch(std::integral_constant<int, 1>());
    else launch(std::integral_constant<int, 4>());
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
        a.tokens = (int)tokens, a.n_q_heads = heads->n_q_heads, a.group = (int)group, a.window = std::min(heads->window, kKv4MaxPositions);
        a.row_blocks = (int)ceil_div(tokens * group, kKv4Rows);
        const int64_t unit = dtype == HIPC_F16 ? 8 : 4;
        a.wide = aligned(Q, 16) && aligned(Y, 16) && q_stride % unit == 0 && y_stride % unit == 0;
        // what workgroups exchange, and the words they count in, in a scratch slot of this operator's own: the words are zero
        // between calls, so a new block is cleared once
        const unsigned grid = kKv4PerCu * ctx->cu_count;   // at most
        const size_t count_bytes = (grid * 4 + 255) & ~(size_t)255;
        const void *before = ctx->scratch[kScratchKv4].ptr;
        void *block = nullptr;
        if (int rc = scratch_get(ctx, kScratchKv4, count_bytes + (size_t)grid * 2 * kKv4Rows * (kKv4MaxHead + 2) * 4, &block)) return rc;
        a.arrived = static_cast<uint32_t *>(block), a.parts = reinterpret_cast<float *>(static_cast<char *>(block) + count_bytes);
        if (block != before) {
            hipLaunchKernelGGL((fill_words), 1, 256, 0, ctx->stream, a.arrived, count_bytes / 4, 0u);
            HIPC_LAUNCHED(ctx);
        }
        const int64_t units = (int64_t)cache->n_seqs * cache->n_kv_heads * a.row_blocks;
        const bool alone = units * 2 >= 3 * (int64_t)ctx->cu_count;
        switch (heads->head_dim / 32) {
            case 1: kv4_launch<32>(ctx, a, dtype, alone); break;
            case 2: kv4_launch<64>(ctx, a, dtype, alone); break;
            case 3: kv4_launch<96>(ctx, a, dtype, alone); break;
            case 4: kv4_launch<128>(ctx, a, dtype, alone); break;
            case 5: kv4_launch<160>(ctx, a, dtype, alone); break;
            case 6: kv4_launch<192>(ctx, a, dtype, alone); break;
            case 7: kv4_launch<224>(ctx, a, dtype, alone); break;
            default: kv4_launch<256>(ctx, a, dtype, alone); break;
        }
        HIPC_LAUNCHED(ctx);
        return HIPC_OK;
    });
}

}  // extern "C"
