// Attention over packed prompts (hipc_prompt_attention).
#include <algorithm>
#include <type_traits>

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
    // on the matrix cores
    int tiles, splits, by_keys;   // query tiles at most; workgroups that share the keys of a tile; tiles are started in the order of the keys they see
    float *part_o, *part_ml;   // of each: [split][row][head][channel] sums, (maximum, sum) pairs
};
constexpr int kScratchPrompt = 3;   // scratch slot of the parts

constexpr int kScratchPadded = 8;   // ... and of the operands in rows of the matrix cores' kind

// A factor of what a row sees is above 0, however small: where the type has no number for it, the least one stands in, so that an infinity times it
// stays one. (A NaN stays a NaN.)
__device__ __forceinline__ float above_zero(float w) { return w == 0.f ? 0x1p-149f : w; }

// Heads too wide for the matrix cores, and calls without scratch memory for aligned rows (in a recording, or where the device has no more): one wavefront per query row and head, a lane a channel of every
// 64, KEYS keys on their way at once. Bound by the trips to memory: 1000 rows of 4 / 2 heads of 264 in f16 726 us, 1145 with one key at a time.
template <typename T, int C>
__global__ void __launch_bounds__(64) prompt_rows_kernel(const PromptArgs a) {
    constexpr int KEYS = 32 / C;
    const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, kvh = h / a.group;
    int seq, first, end;
    if (!packed_sequence(a.q_starts, a.n_seqs, a.total_q, row, &seq, &first, &end)) return;
    const int k0 = max(a.k_starts[seq], 0), k1 = min(a.k_starts[seq + 1], a.total_k);
    const int keys = max(k1 - k0, 0);
    const int pos = keys - (end - first) + (row - first);
    const T *q = static_cast<const T *>(a.q) + a.q_stride * row + (int64_t)h * a.dim;
    T *y = static_cast<T *>(a.y) + a.y_stride * row + (int64_t)h * a.dim;
    float qv[C], acc[C] = {};
#pragma unroll
    for (int i = 0; i < C; i++) qv[i] = lane + 64 * i < a.dim ? (float)q[lane + 64 * i] * a.scale : 0.f;
    float m = -INFINITY, l = 0.f;
    const int from = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0, to = a.causal ? pos + 1 : keys;
    for (int t0 = from; t0 < to; t0 += KEYS) {
        // (behind the last key that is seen that one stands in, and does not count)
        auto load = [&](const void *base, int64_t stride, T (&x)[KEYS][C]) {
#pragma unroll
            for (int e = 0; e < KEYS; e++) {
                const T *from_row = static_cast<const T *>(base) + stride * (k0 + min(t0 + e, to - 1)) + (int64_t)kvh * a.dim;
#pragma unroll
                for (int i = 0; i < C; i++) {
                    const T there = from_row[min(lane + 64 * i, a.dim - 1)];
                    x[e][i] = lane + 64 * i < a.dim ? there : (T)0.f;
                }
            }
        };
        T k[KEYS][C], v[KEYS][C];
        load(a.k, a.k_stride, k);
        load(a.v, a.v_stride, v);
        float s[KEYS], grown = m;
#pragma unroll
        for (int e = 0; e < KEYS; e++) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < C; i++) sum = __builtin_fmaf(qv[i], (float)k[e][i], sum);
            s[e] = lean_wave_sum(sum);
            if (t0 + e < to) grown = fmaxf(grown, s[e]);
        }
        const float keep = m == -INFINITY ? 0.f : above_zero(expf(m - grown));
        m = grown, l *= keep;
#pragma unroll
        for (int i = 0; i < C; i++) acc[i] *= keep;
#pragma unroll
        for (int e = 0; e < KEYS; e++) {
            if (t0 + e >= to) break;
            // (a score of -inf has no weight, also before any other has one)
            const float p = s[e] == -INFINITY ? 0.f : above_zero(expf(s[e] - grown));
            l += p;
#pragma unroll
            for (int i = 0; i < C; i++) acc[i] = __builtin_fmaf(p, (float)v[e][i], acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < C; i++)
        if (lane + 64 * i < a.dim) y[lane + 64 * i] = (T)(l > 0.f ? acc[i] / l : l);
}

// Rows that are not as the matrix cores' kernels take them (heads of a multiple of 8 channels, on 16 bytes) pass through scratch memory as such rows, with
// zeros behind a head's channels, and the result comes back the same way: two launches more, 1000 rows of 12 heads of 100 in f16 32 us where the kernel
// above took 1420. A lane moves eight channels; rows outside every sequence are left alone.
struct PromptPadded {
    void *rows[3], *padded[3];   // Q, K, V, or Y; null: as they are
    int64_t stride[3];           // of rows
    const int *starts[3];
    int total[3], heads[3];
    int n_seqs, dim, units;      // channels of a head, and the padded head's units of eight
};
template <typename T, bool IN>
__global__ void __launch_bounds__(256) prompt_pad_kernel(const PromptPadded a) {
    typedef T T8 __attribute__((ext_vector_type(8)));
    const int z = blockIdx.y, row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (!a.rows[z] || row >= a.total[z]) return;
    int seq, first, end;
    if (!packed_sequence(a.starts[z], a.n_seqs, a.total[z], row, &seq, &first, &end)) return;
    T *rows = static_cast<T *>(a.rows[z]) + a.stride[z] * row;
    T8 *padded = static_cast<T8 *>(a.padded[z]) + (int64_t)row * a.heads[z] * a.units;
    for (int u = threadIdx.x & 63; u < a.heads[z] * a.units; u += 64) {
        const int h = u / a.units, c = (u - h * a.units) * 8;
        T *at = rows + (int64_t)h * a.dim + c;
        T8 v;
        if (IN) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = c + j < a.dim ? at[j] : (T)0.f;
            padded[u] = v;
        } else {
            v = padded[u];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (c + j < a.dim) at[j] = v[j];
        }
    }
}

// ---------------------------------------------------------------------------------- on the matrix cores, f16
//
// A wavefront has 32 query rows -- (token, head of the group) pairs, the group's heads of a token side by side, so that keys are
// fetched once for all heads that share them -- and walks the keys KT at a time, both products turned around:
//   S^T = K Q^T      32x32x16: a lane's 16 results are one query's scores (query = lane % 32) of keys 8 (r / 4) + 4 (lane / 32) + r % 4
//   O^T = V^T P^T    the lane's weights are the second operand as they lie, with the keys of a step numbered the way the scores came out;
//                    V^T is read from row-major LDS rows by the transposing loads
// so maximum, sum and rescale of the softmax are numbers of one lane, exchanged once between the two halves of the wavefront.
// The running maximum is let grow by up to 2^8 before sums are rescaled, and weights are kept 2^7 times as large: up to 2^15 in f16, whose ordinary
// numbers then reach down to 2^-21 of the heaviest weight and whose subnormal ones, off by up to 2^-32 of it, to 2^-31. (Around 1, f16 loses weights below
// 2^-25: of 60000 keys that together weigh 2^-10 of one more, all.) That weights are rounded to f16 at all is a choice: as two terms each they would take half as
// many products again of a kernel that these bound, to bring errors of 1.1 to 1.35 times what rounding the results alone makes down to that.
// Tiles of K and V go from memory to LDS without a register, one tile ahead; 16-byte chunks of a row lie at chunk ^ f(row), so
// that the eight (K) and four (V) rows a read takes per cycle lie in different banks. Chunks behind head_dim and rows behind the
// sequence are zeros (the buffer's range check).
typedef _Float16 ph8 __attribute__((ext_vector_type(8)));
typedef _Float16 ph4 __attribute__((ext_vector_type(4)));
typedef _Float16 ph2 __attribute__((ext_vector_type(2)));
typedef short ps4 __attribute__((ext_vector_type(4)));
typedef float pf16 __attribute__((ext_vector_type(16)));
typedef uint32_t pu4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleAt = 8.f;   // in powers of two
constexpr float kWeightUp = 7.f;    // ... f16 weights

// Which ROWS query rows of one kv head a workgroup has; the tiles are started in the order of `at`.
struct PromptTile {
    int seq, q0, len_q, k0, keys;   // the sequence's rows of Q and K
    int r0, rows;                   // first row of the tile, rows of the sequence (tokens * group)
};
// what a lane knows of a sequence
struct PromptLengths {
    int from, keys_from, len, keys, tiles;
    __device__ __forceinline__ PromptLengths(const PromptArgs &a, int seq, int rows) {
        const int s = min(seq, a.n_seqs - 1);
        // (all four on their way together)
        const int q_from = a.q_starts[s], q_to = a.q_starts[s + 1], k_from = a.k_starts[s], k_to = a.k_starts[s + 1];
        from = max(q_from, 0), keys_from = max(k_from, 0);
        const int to = min(q_to, a.total_q);
        len = seq < a.n_seqs && to > from ? to - from : 0, keys = max(min(k_to, a.total_k) - keys_from, 0);
        tiles = (len * a.group + rows - 1) / rows;
    }
    __device__ __forceinline__ void of_lane(const PromptArgs &a, int l, PromptTile *out) const {
        out->q0 = __builtin_amdgcn_readlane(from, l);
        out->len_q = __builtin_amdgcn_readlane(len, l);
        out->rows = out->len_q * a.group;
        out->k0 = __builtin_amdgcn_readlane(keys_from, l);
        out->keys = __builtin_amdgcn_readlane(keys, l);
    }
};
template <int ROWS>
__device__ __forceinline__ bool prompt_tile(const PromptArgs &a, int at, PromptTile *out) {
    const int lane = threadIdx.x & 63;
    if (a.by_keys) {
        // (64 sequences at most) Tiles that see the most keys first, of all sequences: a lane knows how many tiles of its sequence see more than some number of keys, and the
        // number below which the wanted one lies is found by halving, in steps of 64 keys. (In the sequences' order the first sequence's last tiles,
        // as long as any, came last: eight of up to 1024, 32 / 8 heads of 128, 61.5 us and 58.7 this way; four of up to 3000, 14 / 2 heads of 64, 79 and 70.)
        const PromptLengths s(a, lane, ROWS);
        const int past = s.keys - s.len;
        // (j + 1) * ROWS / group + past keys are seen by tile j; the clamp keeps the product within the rows' own count
        auto above = [&](int level) { return s.tiles - (int)min((uint32_t)s.tiles, (uint32_t)(min(max(64 * level - past, 0), s.len + ROWS) * a.group) / ROWS); };
        auto all = [&](int n) { return __builtin_amdgcn_readlane(wave_scan(n), 63); };
        if (at >= all(s.tiles)) return false;
        int low = -1, high = (int)lean_wave_max((float)((max(s.keys, 0) + ROWS) / 64 + 1)) + 1;   // (rounded up past 2^24)
        while (high - low > 1) {
            const int mid = (low + high) / 2;
            if (all(above(mid)) <= at) high = mid;
            else low = mid;
        }
        const int n = above(high), here = (low < 0 ? s.tiles : above(low)) - n, scan = wave_scan(here);
        const int rank = at - all(n), l = __builtin_ctzll(__ballot(scan > rank));
        s.of_lane(a, l, out);
        out->seq = l;
        out->r0 = (__builtin_amdgcn_readlane(s.tiles - n - 1 - (rank - (scan - here)), l)) * ROWS;
        return true;
    }
    // the last tiles of a causal sequence are the heaviest
    const int tile = a.tiles - 1 - at;
    int before = 0;
    auto in = [&](int base, const PromptLengths &s) {
        const int sum = wave_scan(s.tiles);
        const uint64_t over = __ballot(before + sum > tile);
        if (over) {
            const int l = __builtin_ctzll(over);
            s.of_lane(a, l, out);
            out->seq = base + l;
            out->r0 = (tile - (before + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(s.tiles, l))) * ROWS;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
        return over != 0;
    };
    if (in(0, PromptLengths(a, lane, ROWS))) return true;
    for (int base = 64; base < a.n_seqs; base += 256) {   // (four chunks on their way at once)
        const PromptLengths s[4] = {{a, base + lane, ROWS}, {a, base + 64 + lane, ROWS}, {a, base + 128 + lane, ROWS}, {a, base + 192 + lane, ROWS}};
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (in(base + 64 * e, s[e])) return true;
    }
    return false;
}

__device__ __forceinline__ float halves_max(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 16 bytes a lane from memory to LDS (lane l's to `to` + 16 l), zeros where the offset is outside the descriptor; arrived when vmcnt says so
__device__ __forceinline__ void to_lds(uint32_t to, pu4 rsrc, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(rsrc) : "memory");
}
__device__ __forceinline__ pu4 descriptor(const void *p, uint32_t bytes) {
    const uint64_t at = (uint64_t)p;
    return pu4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at), (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(at >> 32) & 0xffffu)),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

// what one key range of a row left for the join: sums not divided yet
__device__ __forceinline__ size_t prompt_part(const PromptArgs &a, int z, int row, int head) { return ((size_t)z * a.total_q + row) * a.n_q_heads + head; }

// the key tiles of a workgroup of `rows` query rows: what its rows see together, or one of a.splits parts of it
struct PromptSpan {
    int t0, t1;
    __device__ __forceinline__ PromptSpan(const PromptArgs &a, const PromptTile &pt, int rows, int key_tile) {
        const int past = pt.keys - pt.len_q, last = (min(pt.r0 + rows, pt.rows) - 1) / a.group;
        const int end = a.causal ? min(max(past + last + 1, 0), pt.keys) : pt.keys;
        const int begin = a.window > 0 ? max(past + pt.r0 / a.group - a.window + 1, 0) : 0;
        t0 = begin / key_tile, t1 = end > begin ? (end + key_tile - 1) / key_tile : t0;
        if (a.splits > 1) {
            const int per = (t1 - t0 + a.splits - 1) / a.splits;
            t0 += (int)blockIdx.y * per, t1 = min(t1, t0 + per);
        }
    }
};
// a lane's query row and the keys it sees; those some and those all of its wavefront's 32 rows see
struct PromptRow {
    bool mine, any;
    int token, head, lane_begin, lane_end, begin, end, all_begin, all_end;
    __device__ __forceinline__ PromptRow(const PromptArgs &a, const PromptTile &pt, int first, int n, int kvh) {
        const int past = pt.keys - pt.len_q, row = first + n;
        any = first < pt.rows, mine = row < pt.rows;
        token = row / a.group, head = kvh * a.group + (row - token * a.group);
        const int p0 = past + first / a.group, p1 = past + min(first + 31, pt.rows - 1) / a.group;
        auto ends = [&](int pos) { return a.causal ? min(pos + 1, pt.keys) : pt.keys; };
        auto begins = [&](int pos) { return a.window > 0 ? max(pos - a.window + 1, 0) : 0; };
        lane_begin = begins(past + token), lane_end = ends(past + token);
        begin = begins(p0), end = ends(p1), all_begin = begins(p1), all_end = ends(p0);
    }
};
// counts of visible values that are not finite (1 of +inf, 128 of -inf, 16384 of NaN, of at most 64 keys), added to sums
__device__ __forceinline__ void add_kinds(const pf16 &kinds, pf16 &o) {
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int k = (int)kinds[r];
        if (k) o[r] += k >= 16384 || ((k & 127) && k >= 128) ? NAN : k >= 128 ? -INFINITY : INFINITY;
    }
}
// the lane's row, done: divided into Y, or as it is for the join
template <typename T, int HC>
__device__ __forceinline__ void prompt_rows_out(const PromptArgs &a, const PromptTile &pt, const PromptRow &pr, int h, int c0, float m, float l, const pf16 (&o)[HC / 32]) {
    l = halves_sum(l);
    if (!pr.mine) return;
    if (a.splits > 1) {
        const size_t part = prompt_part(a, blockIdx.y, pt.q0 + pr.token, pr.head);
        if (h == 0 && c0 == 0) a.part_ml[2 * part] = m, a.part_ml[2 * part + 1] = l;
        float *to = a.part_o + part * a.dim;
#pragma unroll
        for (int ot = 0; ot < HC / 32; ot++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int c = c0 + 32 * ot + 8 * (r / 4) + 4 * h;
                if (c < a.dim) *reinterpret_cast<float4 *>(to + c) = make_float4(o[ot][r], o[ot][r + 1], o[ot][r + 2], o[ot][r + 3]);
            }
        return;
    }
    typedef T T4 __attribute__((ext_vector_type(4)));
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T *y = static_cast<T *>(a.y) + a.y_stride * (pt.q0 + pr.token) + (int64_t)pr.head * a.dim;
#pragma unroll
    for (int ot = 0; ot < HC / 32; ot++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int c = c0 + 32 * ot + 8 * (r / 4) + 4 * h;
            if (c < a.dim) *reinterpret_cast<T4 *>(y + c) = T4{(T)(o[ot][r] * inv), (T)(o[ot][r + 1] * inv), (T)(o[ot][r + 2] * inv), (T)(o[ot][r + 3] * inv)};
        }
}

// A wavefront's 32 query rows, HC channels of them from channel c0 on, over key tiles of KT rows of PITCH halfs in LDS.
template <int HC, int KT, int PITCH>
struct PromptRows {
    ph8 qf[HC / 16];
    pf16 o[HC / 32];
    float m = -INFINITY, l = 0.f, c2, down = -kWeightUp;   // down: what is taken off a score before the exponential
    uint32_t k_at[4], v_at[2];
    int h;

    __device__ __forceinline__ PromptRows(const PromptArgs &a, int lane, int c0) {
        const int n = lane & 31, i16 = lane & 15;
        h = lane >> 5;
        c2 = fabsf(a.scale) * kLog2e;
        // where the lane reads: K row n, chunk 2 c + h; V rows 4 h + i / 4 (+ 8, + 16 u), 16 channels of 32 ot a half of the 32 lanes
#pragma unroll
        for (int c = 0; c < 4; c++) k_at[c] = n * PITCH * 2 + (((2 * c + h) ^ (n & 7)) * 16) + 2 * c0;
#pragma unroll
        for (int i = 0; i < 2; i++) v_at[i] = (4 * h + (i16 >> 2)) * PITCH * 2 + (((4 * i + 2 * ((lane >> 4) & 1) + ((i16 >> 1) & 1)) ^ ((i16 >> 2) << 1)) * 16) + (i16 & 1) * 8 + 2 * c0;
#pragma unroll
        for (int i = 0; i < HC / 32; i++) o[i] = pf16{};
    }
    __device__ __forceinline__ void queries(const PromptArgs &a, const PromptTile &pt, const PromptRow &pr, int c0) {
        const _Float16 *q = static_cast<const _Float16 *>(a.q) + a.q_stride * (pt.q0 + (pr.mine ? pr.token : 0)) + (int64_t)(pr.mine ? pr.head : 0) * a.dim;
#pragma unroll
        for (int c = 0; c < HC / 16; c++) {
            ph8 v = {};
            if (pr.mine && c0 + 16 * c + 8 * h < a.dim) v = *reinterpret_cast<const ph8 *>(q + c0 + 16 * c + 8 * h);
            qf[c] = a.scale < 0.f ? -v : v;
        }
    }
    __device__ __forceinline__ void scores(const char *ks, pf16 (&s)[KT / 32]) const {
#pragma unroll
        for (int b = 0; b < KT / 32; b++) {
            s[b] = pf16{};
#pragma unroll
            for (int c = 0; c < HC / 16; c++)
                s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const ph8 *>(ks + k_at[c & 3] + (c >> 2) * 128 + b * 64 * PITCH), qf[c], s[b], 0, 0, 0);
        }
    }
    // the scores of keys key0 .. become weights
    __device__ __forceinline__ void weights(pf16 (&s)[KT / 32], int key0, bool masked, const PromptRow &pr, ph8 (&p)[KT / 16]) {
        if (masked) {
#pragma unroll
            for (int b = 0; b < KT / 32; b++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int key = key0 + 32 * b + 8 * (r / 4) + 4 * h + r % 4;
                    s[b][r] = key >= pr.lane_begin && key < pr.lane_end ? s[b][r] : -INFINITY;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < KT / 32; b++)
#pragma unroll
            for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[b][r]);
        mx = halves_max(mx) * c2;
        if (__any(mx > m + kRescaleAt)) {
            const float grown = mx > m + kRescaleAt ? mx : m, keep = grown == m ? 1.f : above_zero(__builtin_amdgcn_exp2f(m - grown));   // (a row goes by its own scores)
            m = grown, l *= keep, down = (m == -INFINITY ? 0.f : m) - kWeightUp;
#pragma unroll
            for (int i = 0; i < HC / 32; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[i][r] *= keep;
        }
#pragma unroll
        for (int u = 0; u < KT / 16; u++)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                typedef float f2 __attribute__((ext_vector_type(2)));
                const f2 w = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[u / 2][8 * (u & 1) + j], c2, -down)),
                              __builtin_amdgcn_exp2f(__builtin_fmaf(s[u / 2][8 * (u & 1) + j + 1], c2, -down))};
                const ph2 w16 = __builtin_convertvector(w, ph2);   // the second product's operand; the sum is that of the same rounded weights
                p[u][j] = w16.x, p[u][j + 1] = w16.y;
                l = __builtin_amdgcn_fdot2(w16, ph2{(_Float16)1.f, (_Float16)1.f}, l, false);
            }
    }
    __device__ __forceinline__ ph8 v_part(const char *vs, int ot, int u) const {
        const char *at = vs + v_at[ot & 1] + (ot >> 1) * 128 + u * 32 * PITCH;
        const ps4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ps4 *)(at));
        const ps4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ps4 *)(at + 16 * PITCH));
        return __builtin_bit_cast(ph8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ __forceinline__ void values(const char *vs, int key0, bool masked, const PromptRow &pr, const ph8 (&p)[KT / 16]) {
        if (masked) {
            // A hidden key's weight is zero, but zero times an infinity is not: where the tile has such values, the product takes
            // zeros in their places, and a second one finds out what the rows that see them get.
            uint32_t bad = 0;
#pragma unroll
            for (int ot = 0; ot < HC / 32; ot++)
#pragma unroll
                for (int u = 0; u < KT / 16; u++) {
                    const pu4 w = __builtin_bit_cast(pu4, v_part(vs, ot, u));
#pragma unroll
                    for (int j = 0; j < 4; j++) bad |= ((w[j] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
                }
            if (__any(bad != 0)) {
#pragma unroll
                for (int ot = 0; ot < HC / 32; ot++) {
                    pf16 kinds = pf16{};
#pragma unroll
                    for (int u = 0; u < KT / 16; u++) {
                        ph8 v = v_part(vs, ot, u), kind = {}, seen = {};
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const uint16_t bits = __builtin_bit_cast(uint16_t, (_Float16)v[j]);
                            // 1 of +inf, 128 of -inf, 16384 of NaN: a tile's counts of each stay apart
                            if ((bits & 0x7c00) == 0x7c00) kind[j] = (_Float16)((bits & 0x3ff) ? 16384.f : bits >> 15 ? 128.f : 1.f), v[j] = (_Float16)0;
                            const int key = key0 + 16 * u + 8 * (j / 4) + 4 * h + j % 4;
                            seen[j] = (_Float16)(key >= pr.lane_begin && key < pr.lane_end ? 1.f : 0.f);
                        }
                        o[ot] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[u], o[ot], 0, 0, 0);
                        kinds = __builtin_amdgcn_mfma_f32_32x32x16_f16(kind, seen, kinds, 0, 0, 0);
                    }
                    add_kinds(kinds, o[ot]);
                }
                return;
            }
        }
#pragma unroll
        for (int ot = 0; ot < HC / 32; ot++)
#pragma unroll
            for (int u = 0; u < KT / 16; u++) o[ot] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v_part(vs, ot, u), p[u], o[ot], 0, 0, 0);
    }
    // Tiles that all rows see whole are not looked through, and an infinity under a weight that f16 rounded to zero has made NaN of its channel there. Where a
    // row's sums (not its weights) are NaN, the values under them are read once more, and infinities of one sign stand for the sum. (Each wavefront by itself, behind
    // the tiles: going over these again with every one looked through cost 2 % of 8192 rows' time and a microsecond of a short call's, this less than half of
    // that. 8192 rows of 32 / 8 heads of 128 that all see a key whose values are NaN take 2.1 ms beside 0.6.)
    __device__ __forceinline__ void settle(const PromptArgs &a, const PromptTile &pt, const PromptRow &pr, const PromptSpan &sp, int kvh, int c0) {
        float most = 0.f;   // a NaN wins
#pragma unroll
        for (int i = 0; i < HC / 32; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) most = __builtin_elementwise_maximum(most, o[i][r]);
        const bool odd = pr.mine && l == l && most != most;
        if (__builtin_expect(!__any(odd), 1)) return;
        // a bit for each of the lane's sums: it is NaN, and there is an infinity of that sign under it, or a NaN (both)
        static_assert(HC / 2 <= 64, "of 64");
        uint64_t left = 0, up = 0, down = 0;
#pragma unroll
        for (int i = 0; i < HC / 32; i++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (odd && o[i][r] != o[i][r]) left |= (uint64_t)1 << (16 * i + r);
        const int from = max(pr.lane_begin, sp.t0 * KT), to = min(pr.lane_end, sp.t1 * KT);
        while (left) {   // four channels at a time, eight keys on their way at once
            const int at = __builtin_ctzll(left) & ~3, c = c0 + 32 * (at / 16) + 8 * (at / 4 % 4) + 4 * h;
            const uint32_t sums = (uint32_t)(left >> at) & 15u;
            const _Float16 *v = static_cast<const _Float16 *>(a.v) + a.v_stride * pt.k0 + (int64_t)kvh * a.dim + c;
            uint32_t u = 0, d = 0;
            for (int key = from; key < to && (u & d & sums) != sums && c < a.dim; key += 8) {
                uint64_t w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] = *reinterpret_cast<const uint64_t *>(v + a.v_stride * min(key + e, to - 1));
#pragma unroll 1
                for (int e = 0; e < 8; e++) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t bits = (uint32_t)(w[0] >> (16 * j)) & 0xffffu;
                        if (bits > 0xfc00u || (bits >= 0x7c00u && bits < 0x8000u)) u |= 1u << j;   // +inf, NaN
                        if (bits >= 0xfc00u || (bits > 0x7c00u && bits < 0x8000u)) d |= 1u << j;   // -inf, NaN
                    }
#pragma unroll
                    for (int f = 0; f < 7; f++) w[f] = w[f + 1];
                }
            }
            up |= (uint64_t)u << at, down |= (uint64_t)d << at;
            left &= ~((uint64_t)15 << at);
        }
#pragma unroll
        for (int i = 0; i < HC / 32; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const bool p = up >> (16 * i + r) & 1, n = down >> (16 * i + r) & 1;
                if (odd && p != n && o[i][r] != o[i][r]) o[i][r] = p ? INFINITY : -INFINITY;
            }
    }
};

// The loads of KT rows of K and V by W wavefronts, of which this is number `wave`: offsets stay, the descriptors' bases move along the keys.
template <int KT, int PITCH, int W>
struct PromptFetch {
    static constexpr int CHUNKS = PITCH / 8, RPI = 512 / PITCH;   // 16-byte chunks of a row; rows of a 1 KiB load
    static constexpr int LOADS = KT / RPI, EACH = (LOADS + W - 1) / W;
    const char *k, *v;
    uint32_t k_row, v_row, k_off[EACH], v_off[EACH];
    int keys, width, wave;

    __device__ __forceinline__ PromptFetch(const PromptArgs &a, const PromptTile &pt, int kvh, int wave_, int lane) : keys(pt.keys), width(2 * a.dim), wave(wave_) {
        k_row = (uint32_t)a.k_stride * 2, v_row = (uint32_t)a.v_stride * 2;
        k = static_cast<const char *>(a.k) + (a.k_stride * pt.k0 + (int64_t)kvh * a.dim) * 2;
        v = static_cast<const char *>(a.v) + (a.v_stride * pt.k0 + (int64_t)kvh * a.dim) * 2;
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int r = (wave + e * W) * RPI + lane / CHUNKS, chunk = lane % CHUNKS;
            const int kc = chunk ^ (r & 7), vc = chunk ^ ((r & 3) << 1);
            k_off[e] = 8 * kc < a.dim ? r * k_row + 16 * kc : 0x80000000u;
            v_off[e] = 8 * vc < a.dim ? r * v_row + 16 * vc : 0x80000000u;
        }
    }
    __device__ __forceinline__ void rows(const char *base, uint32_t row, const uint32_t (&off)[EACH], int t, uint32_t to) const {
        const pu4 r = descriptor(base + (int64_t)t * KT * row, (uint32_t)(min(keys - t * KT, KT) - 1) * row + width);
#pragma unroll
        for (int e = 0; e < EACH; e++)
            if (LOADS % W == 0 || wave + e * W < LOADS) to_lds(to + (wave + e * W) * 1024, r, off[e]);
    }
    __device__ __forceinline__ void keys_of(int t, uint32_t to) const { rows(k, k_row, k_off, t, to); }
    __device__ __forceinline__ void values_of(int t, uint32_t to) const { rows(v, v_row, v_off, t, to); }
};

// Heads wider than 128 channels are shared by C = 2 wavefronts: each multiplies its half of the channels, they add up their scores through
// LDS, and each sums its half of the channels of the result (one wavefront with all 256 needs 512 registers and has its SIMD to itself:
// 4096 rows of 16 query and 4 kv heads 280 us, shared 235).
template <int HD, int W, int KT>
__global__ void __launch_bounds__(64 * W, 2) prompt_tiles_kernel(const PromptArgs a) {
    constexpr int C = HD > 128 ? 2 : 1, HC = HD / C;               // wavefronts of a row, channels of each
    constexpr int PITCH = HD <= 64 ? 64 : HD <= 128 ? 128 : 256;   // halfs of an LDS row
    constexpr int TILE = KT * PITCH * 2;                           // bytes of a tile of K, or of V
    __shared__ __attribute__((aligned(1024))) char smem[4 * TILE];   // [buffer][K, V]
    __shared__ float4 scores[C > 1 ? W : 1][KT / 8][64];              // a wavefront's own, for the other
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_char *)smem;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    // the heaviest tiles first; kv heads change fastest, so a head stays with its XCDs
    const int heads = a.n_q_heads / a.group, kvh = (int)(blockIdx.x % heads);
    PromptTile pt;
    if (!prompt_tile<32 * W / C>(a, (int)(blockIdx.x / heads), &pt)) return;
    const PromptSpan sp(a, pt, 32 * W / C, KT);
    const PromptRow pr(a, pt, pt.r0 + 32 * (wave / C), lane & 31, kvh);
    const int c0 = C > 1 ? (wave & 1) * HC : 0;   // the wavefront's first channel
    const PromptFetch<KT, PITCH, W> from(a, pt, kvh, wave, lane);
    PromptRows<HC, KT, PITCH> rows(a, lane, c0);
    auto fetch = [&](int t, int buf) {
        from.keys_of(t, lds + buf * 2 * TILE);
        from.values_of(t, lds + buf * 2 * TILE + TILE);
    };
    if (sp.t0 < sp.t1) fetch(sp.t0, 0);
    rows.queries(a, pt, pr, c0);
    for (int t = sp.t0; t < sp.t1; t++) {
        const int buf = (t - sp.t0) & 1;
        // this tile has arrived, and every wavefront is done with the other buffer
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (t + 1 < sp.t1) fetch(t + 1, buf ^ 1);
        const bool active = pr.any && t * KT < pr.end && (t + 1) * KT > pr.begin;
        if (C == 1 && !active) continue;
        const char *ks = smem + buf * 2 * TILE;
        pf16 s[KT / 32];
        rows.scores(ks, s);
        if (C > 1) {
#pragma unroll
            for (int i = 0; i < KT / 8; i++) scores[wave][i][lane] = make_float4(s[i / 4][i % 4 * 4], s[i / 4][i % 4 * 4 + 1], s[i / 4][i % 4 * 4 + 2], s[i / 4][i % 4 * 4 + 3]);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (!active) continue;
#pragma unroll
            for (int i = 0; i < KT / 8; i++) {
                const float4 v = scores[wave ^ 1][i][lane];
                s[i / 4][i % 4 * 4] += v.x, s[i / 4][i % 4 * 4 + 1] += v.y, s[i / 4][i % 4 * 4 + 2] += v.z, s[i / 4][i % 4 * 4 + 3] += v.w;
            }
        }
        const bool masked = (t + 1) * KT > pr.all_end || t * KT < pr.all_begin;
        ph8 p[KT / 16];
        rows.weights(s, t * KT, masked, pr, p);
        rows.values(ks + TILE, t * KT, masked, pr, p);
    }
    rows.settle(a, pt, pr, sp, kvh, c0);
    prompt_rows_out<_Float16, HC>(a, pt, pr, rows.h, c0, rows.m, rows.l, rows.o);
}

// Few rows: a workgroup has 32 of them, and its four wavefronts take the key tiles in turn, each through LDS of its own, so that none waits for
// another before the end. The keys' half of that LDS is free for the next tile once they are multiplied, the values' half once those are; both are
// asked for then, and waited for by count (loads end in the order they were issued in).
// W == 1: a workgroup is one wavefront with all keys of its rows, for short prompts in great number. (1024 of up to 16 rows, 32 / 8 heads of 128: 55 us, with tiles of four wavefronts 130.)
template <int HD, int W>
__global__ void __launch_bounds__(64 * W, 2) prompt_few_kernel(const PromptArgs a) {
    constexpr int KT = 32, PITCH = HD <= 64 ? 64 : 128, TILE = KT * PITCH * 2;
    constexpr int SUMS = W > 1 ? W * HD * 32 * 4 : 0;
    __shared__ __attribute__((aligned(1024))) char smem[2 * W * TILE > SUMS ? 2 * W * TILE : SUMS];   // [wavefront][K, V]; at last the sums
    __shared__ float ml[W][2][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int heads = a.n_q_heads / a.group, kvh = (int)(blockIdx.x % heads);
    PromptTile pt;
    if (!prompt_tile<32>(a, (int)(blockIdx.x / heads), &pt)) return;
    const PromptSpan sp(a, pt, 32, KT);
    const PromptRow pr(a, pt, pt.r0, lane & 31, kvh);
    const PromptFetch<KT, PITCH, 1> from(a, pt, kvh, 0, lane);
    constexpr int LOADS = PromptFetch<KT, PITCH, 1>::LOADS;
    PromptRows<HD, KT, PITCH> rows(a, lane, 0);
    const char *ks = smem + wave * 2 * TILE, *vs = ks + TILE;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_char *)smem + wave * 2 * TILE;
    int t = sp.t0 + wave;
    if (t < sp.t1) from.keys_of(t, lds), from.values_of(t, lds + TILE);
    rows.queries(a, pt, pr, 0);
    for (; t < sp.t1; t += W) {
        const bool masked = (t + 1) * KT > pr.all_end || t * KT < pr.all_begin, more = t + W < sp.t1;
        pf16 s[1];
        ph8 p[2];
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");   // the keys are there; the values may be on their way
        rows.scores(ks, s);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");             // (the keys have been read)
        if (more) from.keys_of(t + W, lds);
        rows.weights(s, t * KT, masked, pr, p);
        if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        rows.values(vs, t * KT, masked, pr, p);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) from.values_of(t + W, lds + TILE);
    }
    rows.settle(a, pt, pr, sp, kvh, 0);   // (the keys of the workgroup's other wavefronts too: these add up)
    if (W == 1) {
        prompt_rows_out<_Float16, HD>(a, pt, pr, rows.h, 0, rows.m, rows.l, rows.o);
        return;
    }
    // the wavefronts' sums, joined in LDS
    rows.l = halves_sum(rows.l);
    if (lane < 32) ml[wave][0][lane] = rows.m, ml[wave][1][lane] = rows.l;
    __syncthreads();
    const int n = lane & 31;
    float best = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; w++) best = fmaxf(best, ml[w][0][n]);
#pragma unroll
    for (int w = 0; w < W; w++) sum += ml[w][1][n] == 0.f ? 0.f : ml[w][1][n] * __builtin_amdgcn_exp2f(ml[w][0][n] - best);
    const float keep = rows.l == 0.f ? 0.f : above_zero(__builtin_amdgcn_exp2f(rows.m - best));
    float4 *sums = reinterpret_cast<float4 *>(smem);   // [wavefront][four results of a lane][lane]
#pragma unroll
    for (int i = 0; i < HD / 8; i++) {
        const pf16 &x = rows.o[i / 4];
        const int r = i % 4 * 4;
        sums[(wave * (HD / 8) + i) * 64 + lane] = rows.l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x[r] * keep, x[r + 1] * keep, x[r + 2] * keep, x[r + 3] * keep);
    }
    __syncthreads();
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const size_t part = prompt_part(a, blockIdx.y, pt.q0 + (pr.mine ? pr.token : 0), pr.mine ? pr.head : 0);
    if (a.splits > 1 && wave == 0 && lane < 32 && pr.mine) a.part_ml[2 * part] = best, a.part_ml[2 * part + 1] = sum;
#pragma unroll
    for (int j = 0; j < HD / 8 / W; j++) {
        const int i = j * W + wave, c = 32 * (i / 4) + 8 * (i % 4) + 4 * rows.h;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float4 x = sums[(w * (HD / 8) + i) * 64 + lane];
            v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        if (!pr.mine || c >= a.dim) continue;
        if (a.splits > 1) {
            *reinterpret_cast<float4 *>(a.part_o + part * a.dim + c) = v;
        } else {
            _Float16 *y = static_cast<_Float16 *>(a.y) + a.y_stride * (pt.q0 + pr.token) + (int64_t)pr.head * a.dim;
            *reinterpret_cast<ph4 *>(y + c) = ph4{(_Float16)(v.x * inv), (_Float16)(v.y * inv), (_Float16)(v.z * inv), (_Float16)(v.w * inv)};
        }
    }
}

// ---------------------------------------------------------------------------------- on the matrix cores, f32
//
// The same products of f32 factors, each as three bf16 terms (8 bits a term, together the value's 24): of the nine products of
// terms six are formed, smallest first; the three left out are below 2^-21 of the whole together (2^-23 on average). K and V are split once on their way into LDS, a plane a term; a
// tile's values wait in registers while the tile before is multiplied.
typedef __bf16 pb8 __attribute__((ext_vector_type(8)));

// Two values as three pairs of bf16, cut off rather than rounded: 8 bits each, so their sum is the value, and no term passes the type's range. (A
// value that is not finite is its first term; the others are NaN.)
__device__ __forceinline__ void split3(float x, float y, uint32_t (&term)[3]) {
    auto top = [](float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); };
    auto pair = [](float v, float w) { return __builtin_amdgcn_perm(__float_as_uint(w), __float_as_uint(v), 0x07060302u); };   // the upper halves
    const float rx = x - top(x), ry = y - top(y);
    term[0] = pair(x, y), term[1] = pair(rx, ry), term[2] = pair(rx - top(rx), ry - top(ry));
}
__device__ __forceinline__ pf16 mfma_terms(const pb8 (&x)[3], const pb8 (&y)[3], pf16 acc) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[2], y[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[0], y[2], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[1], y[1], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[1], y[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[0], y[1], acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[0], y[0], acc, 0, 0, 0);
}

template <int HD, int W>
__global__ void __launch_bounds__(64 * W, HD > 128 && W == 4 ? 1 : 2) prompt_terms_kernel(const PromptArgs a) {
    constexpr int C = HD > 128 ? 2 : 1, HC = HD / C;
    constexpr int KT = 32;
    constexpr int PITCH = HD <= 64 ? 64 : HD <= 128 ? 128 : 256;   // bf16 of an LDS row
    constexpr int PLANE = KT * PITCH * 2;                          // bytes of a term of a tile
    constexpr int CHUNKS = HD / 8;                                 // units of eight channels of a row
    constexpr int EACH = (KT * CHUNKS + 64 * W - 1) / (64 * W);    // ... of a tile, per thread
    __shared__ __attribute__((aligned(1024))) char smem[6 * PLANE];   // [K, V][term]
    __shared__ float4 scores[C > 1 ? W : 1][4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;

    const int heads = a.n_q_heads / a.group, kvh = (int)(blockIdx.x % heads);
    PromptTile pt;
    if (!prompt_tile<32 * W / C>(a, (int)(blockIdx.x / heads), &pt)) return;
    const PromptSpan sp(a, pt, 32 * W / C, KT);
    const PromptRow pr(a, pt, pt.r0 + 32 * (wave / C), n, kvh);
    const int c0 = C > 1 ? (wave & 1) * HC : 0;

    const float c2 = a.scale * kLog2e;

    const float *kb = static_cast<const float *>(a.k) + a.k_stride * pt.k0 + (int64_t)kvh * a.dim;
    const float *vb = static_cast<const float *>(a.v) + a.v_stride * pt.k0 + (int64_t)kvh * a.dim;
    float4 held[2][EACH][2];
    auto fetch = [&](int t) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int unit = tid + e * 64 * W, r = unit / CHUNKS, c = (unit - r * CHUNKS) * 8;
            const bool there = unit < KT * CHUNKS && t * KT + r < pt.keys && c < a.dim;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                held[0][e][j] = there ? *reinterpret_cast<const float4 *>(kb + a.k_stride * (t * KT + r) + c + 4 * j) : float4{};
                held[1][e][j] = there ? *reinterpret_cast<const float4 *>(vb + a.v_stride * (t * KT + r) + c + 4 * j) : float4{};
            }
        }
    };
    auto store = [&]() {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int unit = tid + e * 64 * W, r = unit / CHUNKS, chunk = unit - r * CHUNKS;
            if (unit >= KT * CHUNKS) break;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const float *x = reinterpret_cast<const float *>(held[w][e]);
                uint32_t term[4][3];
#pragma unroll
                for (int j = 0; j < 4; j++) split3(x[2 * j], x[2 * j + 1], term[j]);
                char *to = smem + w * 3 * PLANE + r * PITCH * 2 + (chunk ^ (w ? (r & 3) << 1 : r & 7)) * 16;
#pragma unroll
                for (int k = 0; k < 3; k++) *reinterpret_cast<pu4 *>(to + k * PLANE) = pu4{term[0][k], term[1][k], term[2][k], term[3][k]};
            }
        }
    };

    const int i16 = lane & 15;
    uint32_t k_at[4], v_at[2];
#pragma unroll
    for (int c = 0; c < 4; c++) k_at[c] = n * PITCH * 2 + (((2 * c + h) ^ (n & 7)) * 16) + 2 * c0;
#pragma unroll
    for (int o = 0; o < 2; o++) v_at[o] = (4 * h + (i16 >> 2)) * PITCH * 2 + (((4 * o + 2 * ((lane >> 4) & 1) + ((i16 >> 1) & 1)) ^ ((i16 >> 2) << 1)) * 16) + (i16 & 1) * 8 + 2 * c0;

    pf16 o[HC / 32];
#pragma unroll
    for (int i = 0; i < HC / 32; i++) o[i] = pf16{};
    float m = -INFINITY, l = 0.f;
    if (sp.t0 < sp.t1) fetch(sp.t0);
    pb8 qf[HC / 16][3];
    {
        const float *q = static_cast<const float *>(a.q) + a.q_stride * (pt.q0 + (pr.mine ? pr.token : 0)) + (int64_t)(pr.mine ? pr.head : 0) * a.dim;
#pragma unroll
        for (int c = 0; c < HC / 16; c++) {
            float4 v[2] = {};
            if (pr.mine && c0 + 16 * c + 8 * h < a.dim) {
                v[0] = *reinterpret_cast<const float4 *>(q + c0 + 16 * c + 8 * h);
                v[1] = *reinterpret_cast<const float4 *>(q + c0 + 16 * c + 8 * h + 4);
            }
            const float *x = reinterpret_cast<const float *>(v);
            uint32_t term[4][3];
#pragma unroll
            for (int j = 0; j < 4; j++) split3(x[2 * j], x[2 * j + 1], term[j]);
#pragma unroll
            for (int e = 0; e < 3; e++) qf[c][e] = __builtin_bit_cast(pb8, pu4{term[0][e], term[1][e], term[2][e], term[3][e]});
        }
    }
    for (int t = sp.t0; t < sp.t1; t++) {
        __syncthreads();   // everybody is done with the tile before
        store();
        __syncthreads();
        if (t + 1 < sp.t1) fetch(t + 1);
        const bool active = pr.any && t * KT < pr.end && (t + 1) * KT > pr.begin;
        if (C == 1 && !active) continue;

        pf16 s = pf16{}, odd = pf16{};   // (two chains of products, which wait for each other's results half as long)
#pragma unroll
        for (int c = 0; c < HC / 16; c++) {
            pb8 kf[3];
#pragma unroll
            for (int e = 0; e < 3; e++) kf[e] = *reinterpret_cast<const pb8 *>(smem + e * PLANE + k_at[c & 3] + (c >> 2) * 128);
            if (c & 1) odd = mfma_terms(kf, qf[c], odd);
            else s = mfma_terms(kf, qf[c], s);
        }
        s += odd;
        if (C > 1) {
#pragma unroll
            for (int i = 0; i < 4; i++) scores[wave][i][lane] = make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
            __syncthreads();
            if (!active) continue;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 v = scores[wave ^ 1][i][lane];
                s[4 * i] += v.x, s[4 * i + 1] += v.y, s[4 * i + 2] += v.z, s[4 * i + 3] += v.w;
            }
        }
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] *= c2;
        const bool masked = (t + 1) * KT > pr.all_end || t * KT < pr.all_begin;
        if (masked) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int key = t * KT + 8 * (r / 4) + 4 * h + r % 4;
                s[r] = key >= pr.lane_begin && key < pr.lane_end ? s[r] : -INFINITY;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) mx = fmaxf(mx, s[r]);
        mx = halves_max(mx);
        if (__any(mx > m + kRescaleAt)) {
            const float grown = mx > m + kRescaleAt ? mx : m, keep = grown == m ? 1.f : above_zero(__builtin_amdgcn_exp2f(m - grown));
            m = grown, l *= keep;
#pragma unroll
            for (int i = 0; i < HC / 32; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[i][r] *= keep;
        }
        const float shift = m == -INFINITY ? 0.f : m;
        pb8 p[2][3];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            uint32_t term[4][3];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float x = __builtin_amdgcn_exp2f(s[8 * u + 2 * j] - shift), y = __builtin_amdgcn_exp2f(s[8 * u + 2 * j + 1] - shift);
                l += x + y;
                split3(x, y, term[j]);
            }
#pragma unroll
            for (int e = 0; e < 3; e++) p[u][e] = __builtin_bit_cast(pb8, pu4{term[0][e], term[1][e], term[2][e], term[3][e]});
        }
        auto v_part = [&](int e, int ot, int u) {
            const char *at = smem + (3 + e) * PLANE + v_at[ot & 1] + (ot >> 1) * 128 + u * 32 * PITCH;
            const ps4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ps4 *)(at));
            const ps4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ps4 *)(at + 16 * PITCH));
            return __builtin_bit_cast(pb8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        // Infinities and NaN of V (whole in its first term): in the product zeros stand for them -- a weight's later terms may be
        // zero -- and a second product finds out what the rows that see them get.
        uint32_t bad = 0;
#pragma unroll
        for (int ot = 0; ot < HC / 32; ot++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const pu4 w = __builtin_bit_cast(pu4, v_part(0, ot, u));
#pragma unroll
                for (int j = 0; j < 4; j++) bad |= ((w[j] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
            }
        const bool any_bad = __any(bad != 0);
#pragma unroll
        for (int ot = 0; ot < HC / 32; ot++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                pb8 v[3];
#pragma unroll
                for (int e = 0; e < 3; e++) v[e] = v_part(e, ot, u);
                if (any_bad) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if ((__builtin_bit_cast(uint16_t, (__bf16)v[0][j]) & 0x7f80) == 0x7f80) v[0][j] = v[1][j] = v[2][j] = (__bf16)0.f;
                }
                o[ot] = mfma_terms(v, p[u], o[ot]);
            }
        if (any_bad) {
#pragma unroll
            for (int ot = 0; ot < HC / 32; ot++) {
                pf16 kinds = pf16{};
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const pb8 v = v_part(0, ot, u);
                    pb8 kind = {}, seen = {};
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint16_t bits = __builtin_bit_cast(uint16_t, (__bf16)v[j]);
                        if ((bits & 0x7f80) == 0x7f80) kind[j] = (__bf16)((bits & 0x7f) ? 16384.f : bits >> 15 ? 128.f : 1.f);
                        const int key = t * KT + 16 * u + 8 * (j / 4) + 4 * h + j % 4;
                        seen[j] = (__bf16)(key >= pr.lane_begin && key < pr.lane_end ? 1.f : 0.f);
                    }
                    kinds = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kind, seen, kinds, 0, 0, 0);
                }
                add_kinds(kinds, o[ot]);
            }
        }
    }
    prompt_rows_out<float, HC>(a, pt, pr, h, c0, m, l, o);
}

// The ranges of keys that several workgroups had of the same rows, joined: four channels of a row and head per thread. What a range counts for and its
// part are on their way together, AT_ONCE ranges at a time, and rows are looked up meanwhile. (Looked up, weighed and read one behind the other,
// 31 ranges of 64 rows of four heads of 256 took 40 us of the call's 54.)
template <typename T, int AT_ONCE>
__global__ void __launch_bounds__(256) prompt_join_kernel(const PromptArgs a) {
    const int quads = a.dim / 4;
    const int64_t rows = (int64_t)a.total_q * a.n_q_heads, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const bool in = at < rows * quads;
    const int64_t of = in ? at / quads : rows - 1;   // row and head, as in the parts
    const int c = in ? (int)(at - of * quads) * 4 : 0, row = (int)(of / a.n_q_heads), head = (int)(of - (int64_t)row * a.n_q_heads);
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto join = [&](int z0, const float2 (&ml)[AT_ONCE], const float4 (&o)[AT_ONCE]) {
        float most = m;
#pragma unroll
        for (int e = 0; e < AT_ONCE; e++)
            if (z0 + e < a.splits && ml[e].y != 0.f) most = fmaxf(most, ml[e].x);
        const float before = m == most ? 1.f : above_zero(__builtin_amdgcn_exp2f(m - most));
        m = most;
        if (l != 0.f) l *= before, acc.x *= before, acc.y *= before, acc.z *= before, acc.w *= before;
#pragma unroll
        for (int e = 0; e < AT_ONCE; e++) {
            if (z0 + e >= a.splits || ml[e].y == 0.f) continue;   // (the range has nothing the row sees, and its part may hold anything)
            const float keep = ml[e].x == m ? 1.f : above_zero(__builtin_amdgcn_exp2f(ml[e].x - m));
            l = __builtin_fmaf(ml[e].y, keep, l);
            acc.x = __builtin_fmaf(keep, o[e].x, acc.x), acc.y = __builtin_fmaf(keep, o[e].y, acc.y);
            acc.z = __builtin_fmaf(keep, o[e].z, acc.z), acc.w = __builtin_fmaf(keep, o[e].w, acc.w);
        }
    };
    float2 ml[AT_ONCE];
    float4 o[AT_ONCE];
    auto load = [&](int z0) {
#pragma unroll
        for (int e = 0; e < AT_ONCE; e++) {
            const int64_t part = min(z0 + e, a.splits - 1) * rows + of;
            ml[e] = reinterpret_cast<const float2 *>(a.part_ml)[part];
            o[e] = *reinterpret_cast<const float4 *>(a.part_o + part * a.dim + c);
        }
    };
    load(0);
    // (a wavefront's lanes may lie in several rows)
    bool mine = false;
    const int last = __builtin_amdgcn_readlane(row, 63);
    for (int r = __builtin_amdgcn_readfirstlane(row); r <= last; r++) {
        int seq, first, end;
        const bool has = packed_sequence(a.q_starts, a.n_seqs, a.total_q, r, &seq, &first, &end);
        mine |= has && r == row;
    }
    join(0, ml, o);
    for (int z = AT_ONCE; z < a.splits; z += AT_ONCE) {
        load(z);
        join(z, ml, o);
    }
    if (!in || !mine) return;
    typedef T T4 __attribute__((ext_vector_type(4)));
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<T4 *>(static_cast<T *>(a.y) + a.y_stride * row + (int64_t)head * a.dim + c) = T4{(T)(acc.x * inv), (T)(acc.y * inv), (T)(acc.z * inv), (T)(acc.w * inv)};
}

size_t prompt_parts_bytes(const PromptArgs &a, int splits) { return splits > 1 ? (size_t)splits * a.total_q * a.n_q_heads * (a.dim + 2) * 4 : 0; }

// W == 1: the kernel for few rows; 2: the same with a wavefront by itself
template <typename T, int HD, int W>
int prompt_launch(hipc_ctx *ctx, PromptArgs a, int splits, void *parts) {
    const int64_t tiles = ceil_div((int64_t)a.total_q * a.group, W <= 2 ? 32 : 32 * W / (HD > 128 ? 2 : 1)) + a.n_seqs;   // (at most: a sequence may leave one unfinished)
    a.tiles = (int)tiles, a.splits = splits;
    // (where all tiles run at once, their order is not worth the microsecond that it takes to find it)
    a.by_keys = W > 2 && a.causal && a.window == 0 && a.n_seqs > 1 && a.n_seqs <= 64 && tiles * (a.n_q_heads / a.group) > 2 * ctx->cu_count;
    if (splits > 1) {
        a.part_o = static_cast<float *>(parts), a.part_ml = a.part_o + (size_t)splits * a.total_q * a.n_q_heads * a.dim;
    }
    const dim3 grid((unsigned)(tiles * (a.n_q_heads / a.group)), splits);
    if constexpr (sizeof(T) == 2 && W <= 2) hipLaunchKernelGGL((prompt_few_kernel<HD, W == 1 ? 4 : 1>), grid, W == 1 ? 256 : 64, 0, ctx->stream, a);
    else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((prompt_tiles_kernel<HD, W, (HD > 128 ? 32 : 64)>), grid, 64 * W, 0, ctx->stream, a);
    else hipLaunchKernelGGL((prompt_terms_kernel<HD, W>), grid, 64 * W, 0, ctx->stream, a);
    HIPC_LAUNCHED(ctx);
    if (splits > 1) {
        const unsigned threads = (unsigned)ceil_div((int64_t)a.total_q * a.n_q_heads * a.dim / 4, 256);
        if (splits <= 4) hipLaunchKernelGGL((prompt_join_kernel<T, 4>), threads, 256, 0, ctx->stream, a);
        else hipLaunchKernelGGL((prompt_join_kernel<T, 8>), threads, 256, 0, ctx->stream, a);
        HIPC_LAUNCHED(ctx);
    }
    return HIPC_OK;
}

// How many wavefronts a workgroup has, and how many workgroups share the keys of a tile of rows. Both go by what the host knows:
// rows, keys and sequences in all. Measured in us, inputs not in the caches nearest the CUs, heads 32 / 8 of 128 in f16 unless said.
// Wavefronts (4 / 8): 8192 rows in one sequence 607 / 585; eight sequences of up to 1024 58.5 / 61.7; two of up to 1500 in f32, whose tiles are split once for
// all wavefronts, 239 / 217. A wavefront by itself for prompts of few rows (with their heads 256 on average), against four: 1024 of up to 16 rows
// 55 / 130, 256 of up to 64 41 / 51, 64 of up to 256 58 / 54; of 14 / 2 heads of 64 15 / 31.
// The kernel for few rows against four wavefronts: 16 rows behind 4000 keys 15 / 17, 60 20 / 23, 500 alone 11 / 18; 200 seeing 512 keys 12 / 20;
// past 512 workgroups it loses: four prompts of up to 400 22 / 17. Channels up to 64 carry it to twice as many (two prompts of up to 1000, 14 / 2 heads 13 / 20);
// wider than 128, its 32 rows a workgroup take in the keys too often (two pieces of 1000 that see 512 keys, 4 / 1 heads of 256: 33 / 25).
// Sharing keys costs the parts' way out and back and a join, and pays while CUs are left and there are keys enough (alone / 2 / 4 / 8 / 16):
// 64 rows behind 4000 keys, 4 / 1 heads of 256 173 / 94 / 52 / 32 / 23; 600 rows behind 4000 keys 100 / 82 / 79; 600 that see 512 21 / 30 / 32.
template <typename T>
int prompt_matrix(hipc_ctx *ctx, const PromptArgs &a) {
    const int64_t rows = (int64_t)a.total_q * a.group, kv = a.n_q_heads / a.group, cus = ctx->cu_count;
    const int shared = a.dim > 128 ? 2 : 1;   // wavefronts of a row
    const bool brief = sizeof(T) == 2 && a.dim <= 128 && rows <= 256 * (int64_t)a.n_seqs;
    int waves = brief ? 2 : 4;
    if (waves == 4 && rows * kv * shared >= 256 * cus * (sizeof(T) == 2 ? 4 : 1) &&
        (sizeof(T) == 2 ? a.total_k >= 2048 * (int64_t)a.n_seqs : rows >= 1024 * (int64_t)a.n_seqs))
        waves = 8;
    if (sizeof(T) == 2 && a.dim <= 128 && std::max<int64_t>(ceil_div(rows, 32), a.n_seqs) * kv <= (a.dim <= 64 ? 4 : 2) * cus &&
        !(brief && a.total_k <= 128 * (int64_t)a.n_seqs))
        waves = 1;
    if (ctx->tune.prompt_waves > 0) waves = ctx->tune.prompt_waves;
    if (waves < 4 && (sizeof(T) != 2 || a.dim > 128)) waves = 4;
    const int tile_rows = waves <= 2 ? 32 : 32 * waves / shared;
    const int64_t groups = std::max<int64_t>(ceil_div(rows, tile_rows), a.n_seqs) * kv;
    int64_t keys = a.total_k / a.n_seqs;
    if (a.window > 0) keys = std::min<int64_t>(keys, a.window + tile_rows / a.group);
    const int64_t key_tiles = ceil_div(keys, waves == 1 ? 128 : sizeof(T) == 2 && a.dim <= 128 ? 64 : 32);
    // us: a tile of keys 1.2 (f32: 4), the join 4, and for each range its part out and in, at 4.4 TB/s, and its start
    const double tile = sizeof(T) == 2 ? 1.2 : 4.0, part = (double)a.total_q * a.n_q_heads * a.dim * 4 / 2.2e6 + 0.15;
    int splits = 1;
    double best = tile * key_tiles;
    for (int s = 2; s <= std::min<int64_t>(32, key_tiles) && s * groups <= 2 * cus && groups < cus; s++) {
        const double time = tile * ceil_div(key_tiles, s) + 4.0 + s * part;
        if (time < best) best = time, splits = s;
    }
    if (ctx->tune.prompt_split > 0) splits = std::min(ctx->tune.prompt_split, 256);
    void *parts = nullptr;
    if (splits > 1 && !scratch_have(ctx, kScratchPrompt, prompt_parts_bytes(a, splits), &parts)) splits = 1;
    auto launch = [&](auto width) -> int {
        constexpr int HD = decltype(width)::value;
        if (waves >= 8) return prompt_launch<T, HD, 8>(ctx, a, splits, parts);
        if constexpr (sizeof(T) == 2 && HD <= 128) {
            if (waves == 1) return prompt_launch<T, HD, 1>(ctx, a, splits, parts);
            if (waves < 4) return prompt_launch<T, HD, 2>(ctx, a, splits, parts);
        }
        return prompt_launch<T, HD, 4>(ctx, a, splits, parts);
    };
    // (96 beside 128: 6000 rows of 16 / 8 heads of 96 in f16 147 us, as heads of 128 166; two prompts of up to 1500 in f32 135 and 194. A wavefront of
    // its own for 160 channels spills: 119 us where 256 shared by two take 88.)
    return a.dim <= 64    ? launch(std::integral_constant<int, 64>())
           : a.dim <= 96  ? launch(std::integral_constant<int, 96>())
           : a.dim <= 128 ? launch(std::integral_constant<int, 128>())
                          : launch(std::integral_constant<int, 256>());
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
        HIPC_REQUIRE(ctx, n_seqs >= 0 && n_seqs <= 1 << 20 && total_q >= 0 && total_q <= 1 << 30 && total_k >= 0 && total_k <= 1 << 30,
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
        a.dim = heads->head_dim, a.causal = heads->causal != 0, a.window = std::min(heads->window, 1 << 30);
        const int64_t unit = dtype == HIPC_F16 ? 8 : 4;   // elements of 16 bytes
        auto matrix = [&](const PromptArgs &m) { return dtype == HIPC_F16 ? prompt_matrix<_Float16>(ctx, m) : prompt_matrix<float>(ctx, m); };
        const int dim8 = (int)ceil_div(a.dim, 8) * 8;
        if (a.dim <= 256 && heads->n_kv_heads * (int64_t)dim8 <= 1 << 23 && grid_fits((total_q * a.group / 32 + n_seqs + 1) * heads->n_kv_heads, 512) && grid_fits(ceil_div(total_q * heads->n_q_heads * dim8, 1024), 256) &&
            grid_fits(ceil_div(std::max(total_q, total_k), 4), 256)) {
            auto fits = [&](const void *p, int64_t stride, int64_t most) { return a.dim % 8 == 0 && aligned(p, 16) && stride % unit == 0 && stride <= most; };
            // Q, K, V, and Y: padded where they do not fit
            const bool pad[4] = {!fits(Q, q_stride, far), !fits(K, k_stride, 1 << 23) && total_k > 0, !fits(V, v_stride, 1 << 23) && total_k > 0, !fits(Y, y_stride, far)};
            if (!pad[0] && !pad[1] && !pad[2] && !pad[3]) return matrix(a);
            const int64_t count[4] = {total_q, total_k, total_k, total_q};
            const int of_heads[4] = {heads->n_q_heads, heads->n_kv_heads, heads->n_kv_heads, heads->n_q_heads};
            size_t at[4], bytes = 0;
            for (int i = 0; i < 4; i++) {
                at[i] = bytes;
                if (pad[i]) bytes += (size_t)count[i] * of_heads[i] * dim8 * size;
            }
            void *block = nullptr;
            if (scratch_have(ctx, kScratchPadded, bytes, &block)) {
                PromptPadded in{{}, {}, {q_stride, k_stride, v_stride}, {a.q_starts, a.k_starts, a.k_starts}, {a.total_q, a.total_k, a.total_k}, {of_heads[0], of_heads[1], of_heads[2]}, a.n_seqs, a.dim, dim8 / 8};
                PromptPadded out{{Y}, {static_cast<char *>(block) + at[3]}, {y_stride}, {a.q_starts}, {a.total_q}, {of_heads[3]}, a.n_seqs, a.dim, dim8 / 8};
                PromptArgs m = a;
                const void **operands[3] = {&m.q, &m.k, &m.v};
                int64_t *strides[3] = {&m.q_stride, &m.k_stride, &m.v_stride}, rows = 0;
                for (int i = 0; i < 3; i++) {
                    if (!pad[i]) continue;
                    in.rows[i] = const_cast<void *>(*operands[i]), in.padded[i] = static_cast<char *>(block) + at[i];
                    *operands[i] = in.padded[i], *strides[i] = (int64_t)of_heads[i] * dim8;
                    rows = std::max(rows, count[i]);
                }
                m.dim = dim8;
                auto move = [&](auto into, const PromptPadded &p, int64_t n, int operands_of) -> int {
                    constexpr bool IN = decltype(into)::value;
                    const dim3 grid((unsigned)ceil_div(n, 4), operands_of);
                    if (dtype == HIPC_F16) hipLaunchKernelGGL((prompt_pad_kernel<_Float16, IN>), grid, 256, 0, ctx->stream, p);
                    else hipLaunchKernelGGL((prompt_pad_kernel<float, IN>), grid, 256, 0, ctx->stream, p);
                    HIPC_LAUNCHED(ctx);
                    return HIPC_OK;
                };
                if (rows > 0)
                    if (int rc = move(std::true_type(), in, rows, 3)) return rc;
                if (pad[3]) m.y = out.padded[0], m.y_stride = (int64_t)of_heads[3] * dim8;
                if (int rc = matrix(m)) return rc;
                return pad[3] ? move(std::false_type(), out, total_q, 1) : HIPC_OK;
            }
        }
        HIPC_REFUSE(ctx, !grid_fits(total_q, 64), "%s: %lld rows: too many for one call of such heads", who, (long long)total_q);
        const dim3 grid((unsigned)total_q, heads->n_q_heads);
        auto launch = [&](auto channels) {
            constexpr int C = decltype(channels)::value;
            if (dtype == HIPC_F16) hipLaunchKernelGGL((prompt_rows_kernel<_Float16, C>), grid, 64, 0, ctx->stream, a);
            else hipLaunchKernelGGL((prompt_rows_kernel<float, C>), grid, 64, 0, ctx->stream, a);
        };
        if (a.dim <= 64 * 4) launch(std::integral_constant<int, 4>());
        else launch(std::integral_constant<int, kPromptMaxHead / 64>());
        HIPC_LAUNCHED(ctx);
        return HIPC_OK;
    });
}

}  // extern "C"
