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
    // on the matrix cores
    int tiles, splits;         // query tiles at most; workgroups that share the keys of a tile
    float *part_o, *part_ml;   // of each: [split][row][head][channel] sums, (maximum, sum) pairs
};
constexpr int kScratchPrompt = 3;   // scratch slot of the parts

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


// ---------------------------------------------------------------------------------- on the matrix cores, f16
//
// A wavefront has 32 query rows -- (token, head of the group) pairs, the group's heads of a token side by side, so that keys are
// fetched once for all heads that share them -- and walks the keys KT at a time, both products turned around:
//   S^T = K Q^T      32x32x16: a lane's 16 results are one query's scores (query = lane % 32) of keys 8 (r / 4) + 4 (lane / 32) + r % 4
//   O^T = V^T P^T    the lane's weights are the second operand as they lie, with the keys of a step numbered the way the scores came out;
//                    V^T is read from row-major LDS rows by the transposing loads
// so maximum, sum and rescale of the softmax are numbers of one lane, exchanged once between the two halves of the wavefront.
// The running maximum is let grow by up to 2^8 before sums are rescaled (weights up to 2^8 in f16 round like others).
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

// which rows a workgroup of `rows` query rows of one kv head has: tiles are counted through the sequences in order
struct PromptTile {
    int seq, q0, len_q, k0, keys;   // the sequence's rows of Q and K
    int r0, rows;                   // first row of the tile, rows of the sequence (tokens * group)
};
__device__ __forceinline__ bool prompt_tile(const PromptArgs &a, int tile, int rows_per_tile, PromptTile *out) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.n_seqs; base += 64) {
        const int s = min(base + lane, a.n_seqs - 1);
        const int from = max(a.q_starts[s], 0), to = min(a.q_starts[s + 1], a.total_q);
        const int n = base + lane < a.n_seqs && to > from ? ((to - from) * a.group + rows_per_tile - 1) / rows_per_tile : 0;
        int sum = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int up = __shfl_up(sum, d);
            if (lane >= d) sum += up;
        }
        const uint64_t over = __ballot(before + sum > tile);
        if (over) {
            const int l = __builtin_ctzll(over);
            const int first = before + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(n, l);
            out->seq = base + l;
            out->q0 = __builtin_amdgcn_readlane(from, l);
            out->len_q = __builtin_amdgcn_readlane(to, l) - out->q0;
            out->rows = out->len_q * a.group;
            out->r0 = (tile - first) * rows_per_tile;
            out->k0 = max(a.k_starts[out->seq], 0);
            out->keys = max(min(a.k_starts[out->seq + 1], a.total_k) - out->k0, 0);
            return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
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

template <int HD, int W, int KT>
__global__ void __launch_bounds__(64 * W) prompt_tiles_kernel(const PromptArgs a) {
    constexpr int PITCH = HD <= 64 ? 64 : HD <= 128 ? 128 : 256;   // halfs of an LDS row
    constexpr int TILE = KT * PITCH * 2;                           // bytes of a tile of K, or of V
    constexpr int CHUNKS = PITCH / 8, RPI = 512 / PITCH;           // 16-byte chunks of a row; rows of a 1 KiB load
    constexpr int LOADS = TILE / 1024;                             // loads of a tile
    constexpr int EACH = (LOADS + W - 1) / W;
    __shared__ __attribute__((aligned(1024))) char smem[4 * TILE];   // [buffer][K, V]
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_char *)smem;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;

    // the heaviest tiles (the last of a causal sequence) first; kv heads change fastest, so a head stays with its XCDs
    const int heads = a.n_q_heads / a.group, kvh = (int)(blockIdx.x % heads);
    PromptTile pt;
    if (!prompt_tile(a, a.tiles - 1 - (int)(blockIdx.x / heads), 32 * W, &pt)) return;

    const int past = pt.keys - pt.len_q;                              // position of the sequence's first query row
    const int last_row = min(pt.r0 + 32 * W, pt.rows) - 1;
    const int k_end = a.causal ? min(max(past + last_row / a.group + 1, 0), pt.keys) : pt.keys;
    const int k_begin = a.window > 0 ? max(past + pt.r0 / a.group - a.window + 1, 0) : 0;
    int t0 = k_begin / KT, t1 = k_end > k_begin ? (k_end + KT - 1) / KT : t0;
    if (a.splits > 1) {
        const int per = (t1 - t0 + a.splits - 1) / a.splits;
        t0 += (int)blockIdx.y * per, t1 = min(t1, t0 + per);
    }

    // the lane's query row
    const int wr0 = pt.r0 + 32 * wave, row = wr0 + n;
    const bool mine = row < pt.rows;
    const int token = row / a.group, head = kvh * a.group + (row - token * a.group), pos = past + token;
    const int lane_end = a.causal ? min(pos + 1, pt.keys) : pt.keys, lane_begin = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
    // ... and the wavefront's: the first row's and the last's ends
    const int w_last = min(wr0 + 31, pt.rows - 1);
    const int w_pos0 = past + wr0 / a.group, w_pos1 = past + w_last / a.group;
    const bool w_any = wr0 < pt.rows;
    const int w_end = a.causal ? min(w_pos1 + 1, pt.keys) : pt.keys, w_begin = a.window > 0 ? max(w_pos0 - a.window + 1, 0) : 0;
    const int w_all_end = a.causal ? min(w_pos0 + 1, pt.keys) : pt.keys, w_all_begin = a.window > 0 ? max(w_pos1 - a.window + 1, 0) : 0;

    ph8 qf[HD / 16];
    {
        const _Float16 *q = static_cast<const _Float16 *>(a.q) + a.q_stride * (pt.q0 + (mine ? token : 0)) + (int64_t)(mine ? head : 0) * a.dim;
#pragma unroll
        for (int c = 0; c < HD / 16; c++) {
            ph8 v = {};
            if (mine && 16 * c + 8 * h < a.dim) v = *reinterpret_cast<const ph8 *>(q + 16 * c + 8 * h);
            qf[c] = a.scale < 0.f ? -v : v;
        }
    }
    const float c2 = fabsf(a.scale) * kLog2e;

    // the tile's loads of this wavefront: offsets stay, the descriptor's base moves along the keys
    const uint32_t k_row = (uint32_t)a.k_stride * 2, v_row = (uint32_t)a.v_stride * 2;
    const char *kb = static_cast<const char *>(a.k) + (a.k_stride * pt.k0 + (int64_t)kvh * a.dim) * 2;
    const char *vb = static_cast<const char *>(a.v) + (a.v_stride * pt.k0 + (int64_t)kvh * a.dim) * 2;
    uint32_t k_off[EACH], v_off[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int r = (wave + e * W) * RPI + lane / CHUNKS, chunk = lane % CHUNKS;
        const int kc = chunk ^ (r & 7), vc = chunk ^ ((r & 3) << 1);
        k_off[e] = 8 * kc < a.dim ? r * k_row + 16 * kc : 0x80000000u;
        v_off[e] = 8 * vc < a.dim ? r * v_row + 16 * vc : 0x80000000u;
    }
    auto fetch = [&](int t, int buf) {
        const int left = min(pt.keys - t * KT, KT);
        const pu4 kr = descriptor(kb + (int64_t)t * KT * k_row, (uint32_t)(left - 1) * k_row + 2 * a.dim);
        const pu4 vr = descriptor(vb + (int64_t)t * KT * v_row, (uint32_t)(left - 1) * v_row + 2 * a.dim);
#pragma unroll
        for (int e = 0; e < EACH; e++)
            if (LOADS % W == 0 || wave + e * W < LOADS) {
                const uint32_t to = lds + buf * 2 * TILE + (wave + e * W) * 1024;
                to_lds(to, kr, k_off[e]);
                to_lds(to + TILE, vr, v_off[e]);
            }
    };

    // where the lane reads: K row n, chunk 2 c + h; V rows 4 h + i / 4 (+ 8, + 16 u), 16 channels of 32 ot a half of the 32 lanes
    const int i16 = lane & 15;
    uint32_t k_at[4], v_at[2];
#pragma unroll
    for (int c = 0; c < 4; c++) k_at[c] = n * PITCH * 2 + (((2 * c + h) ^ (n & 7)) * 16);
#pragma unroll
    for (int o = 0; o < 2; o++) v_at[o] = (4 * h + (i16 >> 2)) * PITCH * 2 + (((4 * o + 2 * ((lane >> 4) & 1) + ((i16 >> 1) & 1)) ^ ((i16 >> 2) << 1)) * 16) + (i16 & 1) * 8;

    pf16 o[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; i++) o[i] = pf16{};
    float m = -INFINITY, l = 0.f;

    if (t0 < t1) fetch(t0, 0);
    for (int t = t0; t < t1; t++) {
        const int buf = (t - t0) & 1;
        // this tile has arrived, and every wavefront is done with the other buffer
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (t + 1 < t1) fetch(t + 1, buf ^ 1);
        if (!w_any || t * KT >= w_end || (t + 1) * KT <= w_begin) continue;
        const char *ks = smem + buf * 2 * TILE, *vs = ks + TILE;

        pf16 s[KT / 32];
#pragma unroll
        for (int b = 0; b < KT / 32; b++) {
            s[b] = pf16{};
#pragma unroll
            for (int c = 0; c < HD / 16; c++)
                s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const ph8 *>(ks + k_at[c & 3] + (c >> 2) * 128 + b * 64 * PITCH), qf[c], s[b], 0, 0, 0);
        }
        const bool masked = (t + 1) * KT > w_all_end || t * KT < w_all_begin;
        if (masked) {
#pragma unroll
            for (int b = 0; b < KT / 32; b++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int key = t * KT + 32 * b + 8 * (r / 4) + 4 * h + r % 4;
                    s[b][r] = key >= lane_begin && key < lane_end ? s[b][r] : -INFINITY;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < KT / 32; b++)
#pragma unroll
            for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[b][r]);
        mx = halves_max(mx) * c2;
        if (__any(mx > m + kRescaleAt)) {
            const float grown = mx > m + kRescaleAt ? mx : m, keep = grown == m ? 1.f : __builtin_amdgcn_exp2f(m - grown);   // (a row goes by its own scores)
            m = grown, l *= keep;
#pragma unroll
            for (int i = 0; i < HD / 32; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[i][r] *= keep;
        }
        const float shift = m == -INFINITY ? 0.f : m;
        ph8 p[KT / 16];
#pragma unroll
        for (int u = 0; u < KT / 16; u++)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                typedef float f2 __attribute__((ext_vector_type(2)));
                const f2 w = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[u / 2][8 * (u & 1) + j], c2, -shift)),
                              __builtin_amdgcn_exp2f(__builtin_fmaf(s[u / 2][8 * (u & 1) + j + 1], c2, -shift))};
                const ph2 w16 = __builtin_convertvector(w, ph2);   // the second product's operand; the sum is that of the same rounded weights
                p[u][j] = w16.x, p[u][j + 1] = w16.y;
                l = __builtin_amdgcn_fdot2(w16, ph2{(_Float16)1.f, (_Float16)1.f}, l, false);
            }
        auto v_part = [&](int ot, int u) {
            const char *at = vs + v_at[ot & 1] + (ot >> 1) * 128 + u * 32 * PITCH;
            const ps4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ps4 *)(at));
            const ps4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ps4 *)(at + 16 * PITCH));
            return __builtin_bit_cast(ph8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        if (masked) {
            // A hidden key's weight is zero, but zero times an infinity is not: where the tile has such values, the product takes
            // zeros in their places, and a second one finds out what the rows that see them get.
            uint32_t bad = 0;
#pragma unroll
            for (int ot = 0; ot < HD / 32; ot++)
#pragma unroll
                for (int u = 0; u < KT / 16; u++) {
                    const pu4 w = __builtin_bit_cast(pu4, v_part(ot, u));
#pragma unroll
                    for (int j = 0; j < 4; j++) bad |= ((w[j] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
                }
            if (__any(bad != 0)) {
#pragma unroll
                for (int ot = 0; ot < HD / 32; ot++) {
                    pf16 kinds = pf16{};
#pragma unroll
                    for (int u = 0; u < KT / 16; u++) {
                        ph8 v = v_part(ot, u), kind = {}, seen = {};
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const uint16_t bits = __builtin_bit_cast(uint16_t, (_Float16)v[j]);
                            // 1 of +inf, 128 of -inf, 16384 of NaN: a tile's counts of each stay apart
                            if ((bits & 0x7c00) == 0x7c00) kind[j] = (_Float16)((bits & 0x3ff) ? 16384.f : bits >> 15 ? 128.f : 1.f), v[j] = (_Float16)0;
                            const int key = t * KT + 16 * u + 8 * (j / 4) + 4 * h + j % 4;
                            seen[j] = (_Float16)(key >= lane_begin && key < lane_end ? 1.f : 0.f);
                        }
                        o[ot] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[u], o[ot], 0, 0, 0);
                        kinds = __builtin_amdgcn_mfma_f32_32x32x16_f16(kind, seen, kinds, 0, 0, 0);
                    }
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int k = (int)kinds[r];
                        if (k) o[ot][r] += k >= 16384 || ((k & 127) && k >= 128) ? NAN : k >= 128 ? -INFINITY : INFINITY;
                    }
                }
                continue;
            }
        }
#pragma unroll
        for (int ot = 0; ot < HD / 32; ot++)
#pragma unroll
            for (int u = 0; u < KT / 16; u++) o[ot] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v_part(ot, u), p[u], o[ot], 0, 0, 0);
    }
    l = halves_sum(l);
    if (!mine) return;
    if (a.splits > 1) {
        const size_t part = prompt_part(a, blockIdx.y, pt.q0 + token, head);
        if (h == 0) a.part_ml[2 * part] = m, a.part_ml[2 * part + 1] = l;
        float *to = a.part_o + part * a.dim;
#pragma unroll
        for (int ot = 0; ot < HD / 32; ot++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int c = 32 * ot + 8 * (r / 4) + 4 * h;
                if (c < a.dim) *reinterpret_cast<float4 *>(to + c) = make_float4(o[ot][r], o[ot][r + 1], o[ot][r + 2], o[ot][r + 3]);
            }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    _Float16 *y = static_cast<_Float16 *>(a.y) + a.y_stride * (pt.q0 + token) + (int64_t)head * a.dim;
#pragma unroll
    for (int ot = 0; ot < HD / 32; ot++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int c = 32 * ot + 8 * (r / 4) + 4 * h;
            if (c < a.dim)
                *reinterpret_cast<ph4 *>(y + c) = ph4{(_Float16)(o[ot][r] * inv), (_Float16)(o[ot][r + 1] * inv), (_Float16)(o[ot][r + 2] * inv), (_Float16)(o[ot][r + 3] * inv)};
        }
}

// The ranges of keys that several workgroups had of the same rows, joined: one wavefront per row and head.
template <typename T>
__global__ void __launch_bounds__(256) prompt_join_kernel(const PromptArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int row = __builtin_amdgcn_readfirstlane((int)(w / a.n_q_heads)), head = __builtin_amdgcn_readfirstlane((int)(w % a.n_q_heads));
    if (row >= a.total_q) return;
    int seq, first, end;
    if (!packed_sequence(a.q_starts, a.n_seqs, a.total_q, row, &seq, &first, &end)) return;
    float m = -INFINITY, l = 0.f;
    for (int z = 0; z < a.splits; z++) m = fmaxf(m, a.part_ml[2 * prompt_part(a, z, row, head)]);
    float acc[kPromptMaxHead / 64] = {};
    for (int z = 0; z < a.splits; z++) {
        const size_t part = prompt_part(a, z, row, head);
        const float pm = a.part_ml[2 * part], pl = a.part_ml[2 * part + 1];
        if (pl == 0.f) continue;   // the range has nothing the row sees
        const float keep = pm == m ? 1.f : __builtin_amdgcn_exp2f(pm - m);
        l += pl * keep;
#pragma unroll
        for (int i = 0; i < kPromptMaxHead / 64; i++)
            if (lane + 64 * i < a.dim) acc[i] += keep * a.part_o[part * a.dim + lane + 64 * i];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T *y = static_cast<T *>(a.y) + a.y_stride * row + (int64_t)head * a.dim;
#pragma unroll
    for (int i = 0; i < kPromptMaxHead / 64; i++)
        if (lane + 64 * i < a.dim) y[lane + 64 * i] = (T)(acc[i] * inv);
}

template <int HD, int W, int KT>
int prompt_tiles(hipc_ctx *ctx, PromptArgs a, int splits) {
    const int64_t tiles = ceil_div((int64_t)a.total_q * a.group, 32 * W) + a.n_seqs;   // (at most: a sequence may leave one unfinished)
    a.tiles = (int)tiles, a.splits = splits;
    if (splits > 1) {
        const size_t rows = (size_t)splits * a.total_q * a.n_q_heads;
        void *s = nullptr;
        if (int rc = scratch_get(ctx, kScratchPrompt, rows * (a.dim + 2) * 4, &s)) return rc;
        a.part_o = static_cast<float *>(s), a.part_ml = a.part_o + rows * a.dim;
    }
    hipLaunchKernelGGL((prompt_tiles_kernel<HD, W, KT>), dim3((unsigned)(tiles * (a.n_q_heads / a.group)), splits), 64 * W, 0, ctx->stream, a);
    HIPC_LAUNCHED(ctx);
    if (splits > 1) {
        hipLaunchKernelGGL((prompt_join_kernel<_Float16>), (unsigned)ceil_div((int64_t)a.total_q * a.n_q_heads, 4), 256, 0, ctx->stream, a);
        HIPC_LAUNCHED(ctx);
    }
    return HIPC_OK;
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
        if (dtype == HIPC_F16 && heads->head_dim % 8 == 0 && heads->head_dim <= 256 && aligned(Q, 16) && aligned(K, 16) && aligned(V, 16) && aligned(Y, 8) &&
            q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0 && y_stride % 4 == 0 && k_stride <= 1 << 23 && v_stride <= 1 << 23 &&
            (total_q * a.group + (int64_t)n_seqs * 256) * heads->n_kv_heads < (int64_t)1 << 31) {
            const int d = heads->head_dim;
            return d <= 64 ? prompt_tiles<64, 8, 64>(ctx, a, 1) : d <= 128 ? prompt_tiles<128, 8, 64>(ctx, a, 1) : prompt_tiles<256, 4, 32>(ctx, a, 1);
        }
        const dim3 grid((unsigned)total_q, heads->n_q_heads);
        if (dtype == HIPC_F16) hipLaunchKernelGGL((prompt_rows_kernel<_Float16>), grid, 64, 0, ctx->stream, a);
        else hipLaunchKernelGGL((prompt_rows_kernel<float>), grid, 64, 0, ctx->stream, a);
        HIPC_LAUNCHED(ctx);
        return HIPC_OK;
    });
}

}  // extern "C"
