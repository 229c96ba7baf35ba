// Attention of packed new rows over the paged 4-bit cache (hipc_kv4_prompt_attention): the sequences that bring many. Those that bring few are
// kv4_attention.hip's.
//
//   y_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale q_i.k_j - m_i)      over the keys j that row i sees, m_i the running maximum
//
// The matrix cores bound it: of a key tile of 64 a wavefront's 32 rows of 128 channels take 48 products of 32x32x16 -- weights enter as two terms each -- beside some 290 vector
// instructions, an exponential and some six others a score and a quarter of them to unpack codes. So codes become f16 once a workgroup, in LDS, not once a wavefront, and eight
// wavefronts share them where there are rows for that. 2048 rows behind 30000 keys, 32 / 8 heads of 128 in f16: 1500 us, 0.69 PFLOP/s of the operation's, 1.04 of the products that it takes
// (a product of 8192^3: 1.21); matrix cores busy 52 % of the cycles, vector instructions 51 %, LDS 44 %, half of that bank conflicts (Kv4TileReads). 500 rows behind 8000: 120 us.
// Short prompts are chains: 2.4 us a key tile, 5 to start; a chain is cut only where query tiles are fewer than half of the workgroups that run at once.
#include <algorithm>
#include <type_traits>

#include "kv4.h"
#include "kv4_prompt.h"
#include "lanes.h"

namespace hipc {

namespace {

typedef _Float16 th8 __attribute__((ext_vector_type(8)));
typedef _Float16 th2 __attribute__((ext_vector_type(2)));
typedef short ts4 __attribute__((ext_vector_type(4)));
typedef float tf16 __attribute__((ext_vector_type(16)));
typedef uint32_t tu4 __attribute__((ext_vector_type(4)));

constexpr float kTileLog2e = 1.4426950408889634f;
constexpr float kTileRescaleAt = 8.f;   // in powers of two (see Kv4TileRows)
constexpr float kTileUp = 7.f;

__device__ __forceinline__ float tile_halves_max(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float tile_halves_sum(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// What a lane knows of a sequence: its rows (none, where it brings few), how many tiles of ROWS (row, head of the group) pairs they make.
struct TileSequence {
    int row0, tokens, length, tiles;
    // what memory says of it (of the last one, behind it)
    struct Asked {
        int from, to, length;
    };
    static __device__ __forceinline__ Asked ask(const Kv4Tiles &a, int seq) {
        const int s = min(seq, a.cache.n_seqs - 1);
        return {a.starts[s], a.starts[s + 1], a.cache.n_pages > 0 ? kv4_length(a.cache, s) : 0};
    }
    __device__ __forceinline__ TileSequence(const Kv4Tiles &a, int seq, int rows, const Asked &q) {
        length = q.length, row0 = max(q.from, 0);
        const int end = min(q.to, a.total), brought = end > row0 && seq < a.cache.n_seqs ? end - row0 : 0;
        tokens = (int64_t)brought * a.group > a.most ? brought : 0;
        tiles = (int)(((int64_t)tokens * a.group + rows - 1) / rows);
    }
};
// body(base, sequence) for the sequences in chunks of 64, a lane's is base + lane: the first 64 are there, of the others eight chunks are asked for at once (a token of each of 4096
// short sequences, both kernels: 146 us, one chunk behind the other 163). Ends where body is true.
template <int ROWS, typename Body>
__device__ __forceinline__ void tile_sequences(const Kv4Tiles &a, const TileSequence &early, Body body) {
    if (body(0, early)) return;
    const int lane = threadIdx.x & 63;
    for (int base = 64; base < a.cache.n_seqs; base += 512) {
        TileSequence::Asked asked[8];
#pragma unroll
        for (int e = 0; e < 8; e++) asked[e] = TileSequence::ask(a, base + 64 * e + lane);
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (base + 64 * e < a.cache.n_seqs && body(base + 64 * e, TileSequence(a, base + 64 * e + lane, ROWS, asked[e]))) return;
    }
}
// Which rows of one kv head a workgroup has, and which key tiles of KT: the first `sink_tiles`, then those from first + sink_tiles on, `count` in all.
struct Tile {
    int seq, row0, tokens, length, r0, rows;   // rows: of the sequence (tokens times group)
    int first, count, sink_tiles;
};
template <int ROWS, int KT>
__device__ __forceinline__ void tile_keys(const Kv4Tiles &a, Tile *t) {
    const int past = t->length - t->tokens, held = kv4_held(a.cache, t->length);
    const int last = (min(t->r0 + ROWS, t->rows) - 1) / a.group, end = min(past + last + 1, held);
    const int begin = a.window > 0 ? max(past + t->r0 / a.group - a.window + 1, 0) : 0, first = begin / KT;
    t->sink_tiles = a.window > 0 && end > 0 ? min((min(a.sinks, end) + KT - 1) / KT, first) : 0;
    t->first = first - t->sink_tiles;
    t->count = t->sink_tiles + (end > begin ? (end + KT - 1) / KT - first : 0);
}
// all tiles, and how many key tiles the longest of them has
template <int ROWS, int KT>
__device__ __forceinline__ int tile_total(const Kv4Tiles &a, const TileSequence &early, int *longest) {
    int total = 0;
    float most = 0.f;
    tile_sequences<ROWS>(a, early, [&](int, const TileSequence &s) {
        if (!__any(s.tiles > 0)) return false;
        total += __builtin_amdgcn_readlane(wave_scan(s.tiles), 63);
        const int keys = min(s.length, a.window > 0 ? min(a.window, 1 << 29) + ROWS / a.group + min(a.sinks, 1 << 29) : kKv4MaxPositions);
        most = fmaxf(most, lean_wave_max(s.tiles > 0 ? (float)(keys / KT + 1) : 0.f));
        return false;
    });
    *longest = (int)most;
    return total;
}
// tile number `at` of those, the sequences' in their order
template <int ROWS>
__device__ __forceinline__ void tile_find(const Kv4Tiles &a, const TileSequence &early, int at, Tile *t) {
    int before = 0;
    tile_sequences<ROWS>(a, early, [&](int base, const TileSequence &s) {
        if (!__any(s.tiles > 0)) return false;
        const int sum = wave_scan(s.tiles);
        const uint64_t over = __ballot(before + sum > at);
        if (over) {
            const int l = __builtin_ctzll(over);
            t->seq = base + l;
            t->row0 = __builtin_amdgcn_readlane(s.row0, l), t->tokens = __builtin_amdgcn_readlane(s.tokens, l), t->length = __builtin_amdgcn_readlane(s.length, l);
            t->rows = t->tokens * a.group;
            t->r0 = (at - (before + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(s.tiles, l))) * ROWS;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
        return over != 0;
    });
}

// How many workgroups share the keys of a tile where tiles are fewer than workgroups run at once: every part costs its way out and, one behind the other, back into the
// workgroup that joins them (a.part_us), and pays while it takes more key tiles (a.tile_us) off the longest chain.
__device__ __forceinline__ int tile_splits(const Kv4Tiles &a, int units, int longest) {
    if (a.splits > 0) return min(a.splits, max(1, a.slots / units));
    const int most = min(a.slots / units, longest);
    int best = 1;
    float time = a.tile_us * longest;
    for (int s = 2; s <= most; s++) {
        const float t = a.tile_us * ((longest + s - 1) / s) + a.part_us * (s + 2);
        if (t < time) time = t, best = s;
    }
    return best;
}

// A lane's query row and what it sees: keys below `end` that are not below `begin`, or are below a.sinks; and what some and what all of its wavefront's rows see.
struct TileRow {
    bool mine, any;
    int token, head, lane_begin, lane_end, begin, end, all_begin, all_end;
    __device__ __forceinline__ TileRow(const Kv4Tiles &a, const Tile &t, int first, int n, int kvh) {
        const int past = t.length - t.tokens, held = kv4_held(a.cache, t.length), row = first + n;
        any = first < t.rows, mine = row < t.rows;
        token = row / a.group, head = kvh * a.group + (row - token * a.group);
        const int p0 = past + first / a.group, p1 = past + min(first + 31, t.rows - 1) / a.group;
        auto ends = [&](int pos) { return min(pos + 1, held); };
        auto begins = [&](int pos) { return a.window > 0 ? max(pos - a.window + 1, 0) : 0; };
        lane_begin = begins(past + token), lane_end = ends(past + token);
        begin = begins(p0), end = ends(p1), all_begin = begins(p1), all_end = ends(p0);
    }
    // the keys key0 .. key0 + 63 that the lane's row sees, a bit each; `there`: blocks of 16 that lie on pages
    __device__ __forceinline__ uint64_t seen(const Kv4Tiles &a, int key0, uint32_t there) const {
        auto below = [&](int end) { return end <= key0 ? 0 : end - key0 >= 64 ? ~(uint64_t)0 : ((uint64_t)1 << (end - key0)) - 1; };
        uint64_t pages = 0;
#pragma unroll
        for (int b = 0; b < 4; b++) pages |= there >> b & 1 ? (uint64_t)0xffff << (16 * b) : 0;
        return below(lane_end) & (~below(lane_begin) | below(a.sinks)) & pages;
    }
};

// Where a lane reads operands in key tiles of KT rows of PITCH halfs in LDS. 16-byte chunks of a row lie at chunk ^ f(row), three bits of it, so that rows of 128 bytes that a read
// takes at a time lie in different banks. In longer rows three bits leave a read in one 128-byte half of its rows: it has half of the banks, and takes twice as long as it would with all
// (2048 rows behind 30000 keys, 128 channels: 1.6e8 of LDS's 3.2e8 cycles are conflicts).
template <int KT, int PITCH>
struct Kv4TileReads {
    uint32_t k_at[4], v_at[2];
    __device__ __forceinline__ Kv4TileReads(int lane, int c0) {
        const int n = lane & 31, i16 = lane & 15, h = lane >> 5;
#pragma unroll
        for (int c = 0; c < 4; c++) k_at[c] = n * PITCH * 2 + (((2 * c + h) ^ (n & 7)) * 16) + 2 * c0;
#pragma unroll
        for (int i = 0; i < 2; i++) v_at[i] = (4 * h + (i16 >> 2)) * PITCH * 2 + (((4 * i + 2 * ((lane >> 4) & 1) + ((i16 >> 1) & 1)) ^ ((i16 >> 2) << 1)) * 16) + (i16 & 1) * 8 + 2 * c0;
    }
    // keys 32 b + lane % 32, channels 16 c + 8 (lane / 32) .. + 7
    __device__ __forceinline__ th8 keys(const char *ks, int b, int c) const { return *reinterpret_cast<const th8 *>(ks + k_at[c & 3] + (c >> 2) * 128 + b * 64 * PITCH); }
    // channels 32 ot + lane % 32 of the keys 16 u + 8 (j / 4) + 4 (lane / 32) + j % 4: the order in which scores come out
    __device__ __forceinline__ th8 values(const char *vs, int ot, int u) const {
        const char *at = vs + v_at[ot & 1] + (ot >> 1) * 128 + u * 32 * PITCH;
        const ts4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ts4 *)(at));
        const ts4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ts4 *)(at + 16 * PITCH));
        return __builtin_bit_cast(th8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// 32 query rows of a wavefront, HC channels of them from channel c0 on, both products turned around:
//   S^T = K Q^T      32x32x16: a lane's 16 results are one query's scores (query = lane % 32) of keys 8 (r / 4) + 4 (lane / 32) + r % 4
//   O^T = V^T P^T    the lane's weights are the second operand as they lie; V^T is read from row-major LDS rows by the transposing loads
// so maximum, sum and rescale of the softmax are numbers of one lane, exchanged once between the two halves of the wavefront.
// The running maximum may grow by 2^8 before sums are rescaled, and weights are kept 2^7 times as large: f16's ordinary numbers then reach down to 2^-21 of the
// heaviest weight, its subnormal ones to 2^-31. A weight enters as two f16 terms, 22 bits, as it does in the kernel for few rows: which of the two takes a row is decided by
// the rows beside it, and is not to be seen in the result. (One term a weight: errors 1.02 to 1.2 times those of the result's own rounding; 2048 rows behind 30000 keys 1128 us, two
// 1500.) QT = 1, f16 rows: queries as they are. QT = 2, f32 rows: two f16 terms of the row times a power of two.
// The eight channels of a word of codes lie in the order in which it unpacks, 0 4 1 5 2 6 3 7, in K's rows, V's and the queries alike.
template <int HC, int KT, int QT>
struct Kv4TileRows {
    th8 qf[HC / 16][QT];
    tf16 o[HC / 32];
    float m = -INFINITY, l = 0.f, c2, down = -kTileUp;

    __device__ __forceinline__ Kv4TileRows() {
#pragma unroll
        for (int i = 0; i < HC / 32; i++) o[i] = tf16{};
    }
    template <typename T>
    __device__ __forceinline__ void queries(const Kv4Tiles &a, const Tile &t, const TileRow &r, int h, int c0) {
        const T *q = static_cast<const T *>(a.q) + a.q_stride * (t.row0 + (r.mine ? r.token : 0)) + (int64_t)(r.mine ? r.head : 0) * a.cache.head_dim;
        const int dim = a.cache.head_dim;
        const float sign = a.scale < 0.f ? -1.f : 1.f;
        int up = 0;
        c2 = fabsf(a.scale) * kTileLog2e;
        if (QT == 2) {
            // The row's largest value into [2^14, 2^15); an infinity stays where it is. And no further up than leaves the scores' factor an ordinary number: at 0 it
            // would make NaN of what is hidden. (A wavefront with half of the channels looks at the whole row.)
            float most = 0.f;
            for (int c = 8 * h; c < dim; c += 16) {
                float x[8];
                kv4_load8(q + c, a.wide, x);
#pragma unroll
                for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(x[j]));
            }
            most = tile_halves_max(most);
            up = most > 0.f && most < INFINITY ? min(14 - ilogbf(most), 126 + ilogbf(fminf(c2, 0x1p126f))) : 0;
            c2 = ldexpf(c2, -up);
        }
#pragma unroll
        for (int c = 0; c < HC / 16; c++) {
            const int at = c0 + 16 * c + 8 * h;
            float x[8] = {};
            if (at < dim) kv4_load8(q + at, a.wide, x);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float v = x[(j & 1) * 4 + (j >> 1)] * sign;
                if (QT == 2) v = ldexpf(v, up);
                const _Float16 hi = (_Float16)v;
                qf[c][0][j] = r.mine ? hi : (_Float16)0;
                if (QT == 2) qf[c][QT - 1][j] = r.mine ? (_Float16)(v - (float)hi) : (_Float16)0;
            }
        }
    }
    // scores of keys that the lane's row does not see are -inf; `seen`: a bit for each key of the tile
    static __device__ __forceinline__ void hide(tf16 (&s)[KT / 32], uint64_t seen, int h) {
#pragma unroll
        for (int b = 0; b < KT / 32; b++) {
            const uint32_t hidden = ~(uint32_t)(seen >> (32 * b)) >> (4 * h);
#pragma unroll
            for (int r = 0; r < 16; r++) {   // (key 32 b + 8 (r / 4) + 4 h + r % 4)
                const uint32_t all = (uint32_t)((int32_t)(hidden << (31 - 8 * (r / 4) - r % 4)) >> 31);
                s[b][r] = __uint_as_float((all & 0xff800000u) | (~all & __float_as_uint(s[b][r])));
            }
        }
    }
    __device__ __forceinline__ void rise(const tf16 (&s)[KT / 32]) {
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < KT / 32; b++)
#pragma unroll
            for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[b][r]);
        mx = tile_halves_max(mx) * c2;
        if (__any(mx > m + kTileRescaleAt)) {
            const float grown = mx > m + kTileRescaleAt ? mx : m, keep = grown == m ? 1.f : __builtin_amdgcn_exp2f(m - grown);   // (a row goes by its own scores)
            m = grown, l *= keep, down = (m == -INFINITY ? 0.f : m) - kTileUp;
#pragma unroll
            for (int i = 0; i < HC / 32; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[i][r] *= keep;
        }
    }
    __device__ __forceinline__ void weights(const tf16 (&s)[KT / 32], th8 (&p)[KT / 16][2]) {
        float one = 1.f;
        HIPC_PIN_SGPR(one);   // (a product with it, not a subtraction: one instruction takes the f16 term as it is)
#pragma unroll
        for (int u = 0; u < KT / 16; u++)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                typedef float f2 __attribute__((ext_vector_type(2)));
                const f2 w = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[u / 2][8 * (u & 1) + j], c2, -down)),
                              __builtin_amdgcn_exp2f(__builtin_fmaf(s[u / 2][8 * (u & 1) + j + 1], c2, -down))};
                const th2 hi = __builtin_convertvector(w, th2);
                p[u][0][j] = hi.x, p[u][0][j + 1] = hi.y;
                l += w.x + w.y;
                p[u][1][j] = (_Float16)__builtin_fmaf(-(float)hi.x, one, w.x), p[u][1][j + 1] = (_Float16)__builtin_fmaf(-(float)hi.y, one, w.y);
            }
    }
    // Groups of values that are not all numbers are zeros in the product (zero times a NaN is none): the sums of the rows that see them are NaN. Lane l has the marks of
    // units 4 l .. + 3 of the tile, GP a key.
    template <int GP>
    __device__ __forceinline__ void odd_values(uint32_t marks, uint64_t seen, int c0) {
        for (uint64_t left = __ballot(marks != 0); left; left &= left - 1) {
            const int at = __builtin_ctzll(left);
            const uint32_t word = __builtin_amdgcn_readlane(marks, at);
            for (int j = 0; j < 4; j++) {
                const int g = (4 * at + j) % GP, r = (4 * at + j) / GP;
                if (!(word >> (8 * j) & 1)) continue;
                const float more = seen >> r & 1 ? NAN : 0.f;
#pragma unroll
                for (int ot = 0; ot < HC / 32; ot++)
                    if (c0 / 32 + ot == g) o[ot] += more;
            }
        }
    }
    // sums ot, r .. r + 3 (r a multiple of 4) as the channels 32 ot + 8 (r / 4) + 4 h .. + 3: the halves of the wavefront hold 0 4 1 5 and 2 6 3 7 of eight
    __device__ __forceinline__ float4 channels(int ot, int r) const {
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(o[ot][r]), __float_as_uint(o[ot][r + 1]), false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(o[ot][r + 2]), __float_as_uint(o[ot][r + 3]), false, false);
        return make_float4(__uint_as_float(x[0]), __uint_as_float(y[0]), __uint_as_float(x[1]), __uint_as_float(y[1]));
    }
};

// The codes of a key tile on their way from pages to f16 rows in LDS, by all threads of a workgroup: a thread takes 32 channels of a key or a value (16 bytes of codes and
// their parameters), EACH of them. Codes are asked for a tile before they are unpacked, page numbers another. Keys behind the sequence and on no page are zeros.
template <int HD, int KT, int PITCH, int W>
struct Kv4TileFetch {
    static constexpr int GP = HD <= 64 ? 2 : HD <= 128 ? 4 : 8;    // groups of a row, rounded up to a power of two
    static constexpr int UNITS = KT * GP;                          // of a tile of K, or of V
    static constexpr int EACH = W == 8 ? 1 : 2;
    static_assert(UNITS <= 256 && (W == 4 || W == 8), "one of each for 256 threads");
    tu4 codes[EACH];
    uint32_t params[EACH];
    bool none[EACH];   // nothing there: zeros
    int page[EACH], block_page;   // of the tiles asked for next
    const tu4 *codes_at[EACH];         // the unit's in page 0, place 0
    const uint32_t *params_at[EACH];   // ... a word beside every 16 bytes of codes, wherever one looks
    const int *table;
    uint32_t page_units, row_units;    // 16 bytes of codes; of a page (32 bits: where there is more than one, it holds less than 64 GB), of a row
    int shift, held, tid;

    __device__ __forceinline__ Kv4TileFetch(const Kv4Tiles &a, const Tile &t, int kvh, int tid_) : tid(tid_) {
        table = static_cast<const int *>(a.cache.table) + (int64_t)t.seq * a.cache.table_width;
        shift = 31 - __builtin_clz((unsigned)a.cache.page_size), row_units = a.cache.head_dim / 32, held = kv4_held(a.cache, t.length);
        page_units = (uint32_t)((uint64_t)(a.cache.n_kv_heads * row_units) << shift);
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const Unit u = unit(e);
            const int64_t at = ((int64_t)kvh * row_units << shift) + (u.g < (int)row_units ? u.g : 0);
            codes_at[e] = static_cast<const tu4 *>(u.value ? a.cache.v_codes : a.cache.k_codes) + at;
            params_at[e] = static_cast<const uint32_t *>(u.value ? a.cache.v_params : a.cache.k_params) + at;
        }
    }
    // the thread's units: of eight wavefronts the lower four have the keys', the upper ones the values'; of four all have one of each
    struct Unit {
        int g, r;
        bool value, any;
    };
    __device__ __forceinline__ Unit unit(int e) const {
        const int u = tid & 255;
        return {u % GP, (u / GP) % KT, W == 8 ? tid >= 256 : e == 1, u < UNITS};
    }
    // (what the table says is looked at a tile later: whether it is a page, too, so that nothing waits for it before)
    __device__ __forceinline__ int page_of(const Kv4Tiles &a, int key) const {
        const uint32_t at = (uint32_t)min(key >> shift, (int)a.cache.table_width - 1) * 4;   // (tables have up to 2^26 pages)
        return *reinterpret_cast<const int *>(reinterpret_cast<const char *>(table) + at);
    }
    __device__ __forceinline__ bool is_page(const Kv4Tiles &a, int p, int key) const { return (uint32_t)p < (uint32_t)a.cache.n_pages && key < held; }
    // (of unit e's tile)
    __device__ __forceinline__ void ask_page(const Kv4Tiles &a, int e, int tile) { page[e] = page_of(a, tile * KT + unit(e).r); }
    __device__ __forceinline__ void ask_blocks(const Kv4Tiles &a, int tile) { block_page = page_of(a, tile * KT + 16 * (tid % (KT / 16))); }
    // which blocks of 16 keys of the tile asked for lie on pages
    __device__ __forceinline__ uint32_t blocks_there(const Kv4Tiles &a, int tile) const {
        return (uint32_t)__ballot(is_page(a, block_page, tile * KT + 16 * (tid % (KT / 16)))) & ((1u << (KT / 16)) - 1);
    }
    __device__ __forceinline__ void ask_codes(const Kv4Tiles &a, int e, int tile) {
        const Unit u = unit(e);
        const int key = tile * KT + u.r;
        const bool there = is_page(a, page[e], key) && u.any && u.g < (int)row_units;
        const uint64_t at = (uint64_t)(uint32_t)(there ? page[e] : 0) * page_units + (uint64_t)(uint32_t)(key & (a.cache.page_size - 1)) * row_units;
        codes[e] = codes_at[e][at];
        params[e] = params_at[e][at];
        none[e] = !there;
    }
    // into a tile of K or of V; odd: marks of the tile's values, a byte a unit
    __device__ __forceinline__ void unpack(int e, char *to, uint8_t *odd) const {
        const Kv4Unpack take;
        const Unit u = unit(e);
        if (UNITS < 256 && !u.any) return;
        if (HD % (32 * GP) != 0 && 32 * u.g >= HD) return;   // (heads of 96 in rows of 128)
        kvh2 p = __builtin_bit_cast(kvh2, none[e] ? 0u : params[e]);
        // a group that has a NaN, or numbers past f16's range (its values lie between code 0's and code 15's): keys are NaN, values zeros with a mark
        const _Float16 top = __builtin_fmaf16((_Float16)15.f, p.x, p.y);
        const bool bad = (__builtin_bit_cast(uint16_t, top) & 0x7c00) == 0x7c00;
        p = __builtin_bit_cast(kvh2, bad ? (u.value ? 0u : 0x7e007e00u) : __builtin_bit_cast(uint32_t, p));
        if (u.value) odd[u.r * GP + u.g] = bad;
        char *row = to + u.r * PITCH * 2;
        const int turn = u.value ? (u.r & 3) << 1 : u.r & 7;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            kvh2 x[4];
            take(codes[e][j], kvh2{p.x, p.x}, kvh2{p.y, p.y}, x);
            *reinterpret_cast<th8 *>(row + ((4 * u.g + j) ^ turn) * 16) = th8{x[0].x, x[0].y, x[1].x, x[1].y, x[2].x, x[2].y, x[3].x, x[3].y};
        }
    }
};

// (Four wavefronts, the next tile's scores multiplied while this one's become weights: six prompts of up to 1024, 28 / 4 heads of 128 in f16, 46.0 us, in turn 43.8. Nor did it pay that
// the two wavefronts of a SIMD took turns at multiplying, with barriers in between, or that one had 64 rows and a SIMD to itself.)
// Workgroups that a CU runs at once: two wavefronts a SIMD, but one where heads are wider than 128 and four wavefronts have more than half of the LDS.
constexpr int tiles_per_cu(int hd, int w) { return hd > 128 ? 1 : 8 / w; }
template <int HD, int QT, int W>
__global__ void __launch_bounds__(64 * W, tiles_per_cu(HD, W) * W / 4) kv4_tiles_kernel(const Kv4Tiles a) {
    constexpr int C = HD > 128 ? 2 : 1, HC = HD / C;               // wavefronts of a row, channels of each
    constexpr int KT = HD > 128 ? 32 : 64;
    constexpr int PITCH = HD <= 64 ? 64 : HD <= 128 ? 128 : 256;   // halfs of an LDS row
    constexpr int TILE = KT * PITCH * 2, ROWS = 32 * W / C;
    constexpr int GP = HD <= 64 ? 2 : HD <= 128 ? 4 : 8;
    typedef typename std::conditional<QT == 1, _Float16, float>::type T;
    __shared__ __attribute__((aligned(1024))) char smem[4 * TILE];   // [K, V][buffer]
    __shared__ float4 scores[C > 1 ? W : 1][KT / 8][64];             // a wavefront's own, for the other
    __shared__ __attribute__((aligned(16))) uint8_t odd[2][256];     // [buffer][key][group]: values that are not all numbers
    static_assert(KT * GP <= 256, "a byte a unit");
    __shared__ int last_here;
    static_assert(tiles_per_cu(HD, W) * (sizeof smem + sizeof scores + sizeof odd + sizeof last_here) <= 160 * 1024, "a CU's LDS");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;

    const int heads = a.cache.n_kv_heads, kvh = (int)(blockIdx.x % heads);
    const TileSequence early(a, lane, ROWS, TileSequence::ask(a, lane));
    int longest;
    const int tiles = tile_total<ROWS, KT>(a, early, &longest);
    if (tiles == 0) return;
    const int splits = tile_splits(a, tiles * heads, longest);
    const int item = (int)(blockIdx.x / heads), at = item / splits, split = item - at * splits;
    if (at >= tiles) return;
    Tile t = {};
    tile_find<ROWS>(a, early, tiles - 1 - at, &t);   // the last tiles of a sequence are the heaviest
    tile_keys<ROWS, KT>(a, &t);
    const int per = max(1, (t.count + splits - 1) / splits), parts = max(1, (t.count + per - 1) / per);
    if (split >= parts) return;
    const int i0 = split * per, i1 = min(i0 + per, t.count);

    const TileRow row(a, t, t.r0 + 32 * (wave / C), lane & 31, kvh);
    const int c0 = C > 1 ? (wave & 1) * HC : 0;   // the wavefront's first channel
    // (behind the last tile of this workgroup that one stands in: it is unpacked once more, and not looked at)
    auto key_tile = [&](int i) {
        const int j = min(i, i1 - 1);
        return j < t.sink_tiles ? j : t.first + j;
    };
    Kv4TileFetch<HD, KT, PITCH, W> from(a, t, kvh, tid);
    constexpr int EACH = Kv4TileFetch<HD, KT, PITCH, W>::EACH;
    const Kv4TileReads<KT, PITCH> read(lane, c0);
    Kv4TileRows<HC, KT, QT> rows;
    auto k_buffer = [&](int i) { return smem + ((i - i0) & 1) * TILE; };
    auto v_buffer = [&](int i) { return smem + 2 * TILE + ((i - i0) & 1) * TILE; };
    auto odd_buffer = [&](int i) { return odd[(i - i0) & 1]; };
    auto score = [&](const char *ks, tf16 (&s)[KT / 32]) {
#pragma unroll
        for (int b = 0; b < KT / 32; b++) {
            s[b] = tf16{};
#pragma unroll
            for (int c = 0; c < HC / 16; c++) {
                const th8 k = read.keys(ks, b, c);
#pragma unroll
                for (int e = QT - 1; e >= 0; e--) s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, rows.qf[c][e], s[b], 0, 0, 0);
            }
        }
    };
    // what a wavefront of two that share a row has of a tile's scores, and the other's
    auto give = [&](const tf16 (&s)[KT / 32]) {
#pragma unroll
        for (int j = 0; j < KT / 8; j++) scores[wave][j][lane] = make_float4(s[j / 4][j % 4 * 4], s[j / 4][j % 4 * 4 + 1], s[j / 4][j % 4 * 4 + 2], s[j / 4][j % 4 * 4 + 3]);
    };
    auto take = [&](tf16 (&s)[KT / 32]) {
#pragma unroll
        for (int j = 0; j < KT / 8; j++) {
            const float4 v = scores[wave ^ 1][j][lane];
            s[j / 4][j % 4 * 4] += v.x, s[j / 4][j % 4 * 4 + 1] += v.y, s[j / 4][j % 4 * 4 + 2] += v.z, s[j / 4][j % 4 * 4 + 3] += v.w;
        }
    };
    // unit e's tile i to LDS, and what is behind it asked for
    auto unpack = [&](int e, int i) {
        from.unpack(e, from.unit(e).value ? v_buffer(i) : k_buffer(i), odd_buffer(i));
        from.ask_codes(a, e, key_tile(i + 1));
        from.ask_page(a, e, key_tile(i + 2));
    };
    // In turn i tile i + 1 is unpacked: into buffers whose tiles were last read in turn i - 1.
    auto unpack_all = [&](int i) {
#pragma unroll
        for (int e = 0; e < EACH; e++) unpack(e, i + 1);
    };
    // keys and values that this turn reads are there, and everybody is done with the other buffers (codes on their way are not waited for)
    auto meet = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    if (tid < 128) reinterpret_cast<uint32_t *>(odd)[tid] = 0;   // (units that heads of this width do not have stay so)
    if (i0 < i1) {
        from.ask_blocks(a, key_tile(i0));
#pragma unroll
        for (int e = 0; e < EACH; e++) from.ask_page(a, e, key_tile(i0));
#pragma unroll
        for (int e = 0; e < EACH; e++) from.ask_codes(a, e, key_tile(i0)), from.ask_page(a, e, key_tile(i0 + 1));
    }
    rows.template queries<T>(a, t, row, h, c0);
    if (i0 < i1) {
        meet();   // (the marks are cleared)
#pragma unroll
        for (int e = 0; e < EACH; e++) unpack(e, i0);
        for (int i = i0; i < i1; i++) {
            const int tile = key_tile(i), key0 = tile * KT;
            const uint32_t here = from.blocks_there(a, tile);
            from.ask_blocks(a, key_tile(i + 1));
            meet();
            const bool active = row.any && key0 < row.end && (key0 + KT > row.begin || key0 < a.sinks);
            if (C == 1 && !active) {
                unpack_all(i);
                continue;
            }
            tf16 s[KT / 32];
            score(k_buffer(i), s);
            unpack_all(i);   // (while the products are on their way)
            if (C > 1) {
                give(s);
                meet();   // (and the next turn's barrier keeps the next scores from being given before these are taken)
                if (!active) continue;
                take(s);
            }
            const bool masked = key0 + KT > row.all_end || (key0 < row.all_begin && key0 + KT > a.sinks) || here != (1u << (KT / 16)) - 1;
            uint64_t seen = ~(uint64_t)0;
            if (masked) {
                seen = row.seen(a, key0, here);
                rows.hide(s, seen, h);
            }
            rows.rise(s);
            th8 p[KT / 16][2];
            const uint32_t marks = *reinterpret_cast<const uint32_t *>(odd_buffer(i) + 4 * lane);
            rows.weights(s, p);
#pragma unroll
            for (int ot = 0; ot < HC / 32; ot++)
#pragma unroll
                for (int u = 0; u < KT / 16; u++) {
                    const th8 v = read.values(v_buffer(i), ot, u);
#pragma unroll
                    for (int e = 1; e >= 0; e--) rows.o[ot] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[u][e], rows.o[ot], 0, 0, 0);
                }
            if (__builtin_expect(__any(marks != 0), 0)) rows.template odd_values<GP>(marks, seen, c0);
        }
    }

    const float l = tile_halves_sum(rows.l);
    const int dim = a.cache.head_dim;
    auto store = [&](int token, int head, int c, const float4 &v, float inv) {
        T *y = static_cast<T *>(a.y) + a.y_stride * (t.row0 + token) + (int64_t)head * dim + c;
        typedef T T4 __attribute__((ext_vector_type(4)));
        const T4 out = {(T)(v.x * inv), (T)(v.y * inv), (T)(v.z * inv), (T)(v.w * inv)};
        if (a.wide) {
            *reinterpret_cast<T4 *>(y) = out;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = out[j];
        }
    };
    auto out = [&](float sum) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int ot = 0; ot < HC / 32; ot++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const float4 v = rows.channels(ot, r);
                const int c = c0 + 32 * ot + 8 * (r / 4) + 4 * h;
                if (row.mine && c < dim) store(row.token, row.head, c, v, inv);
            }
    };
    if (parts == 1) {
        out(l);
        return;
    }
    // Of several workgroups the one that comes last joins the parts, in their order: every thread stores what it has, two floats at a time, where every workgroup
    // sees them, and the last one's threads read what the same threads of the others had.
    constexpr int PAIRS = HC / 4 + 1;   // of a thread: its sums, then (maximum, sum)
    const int64_t unit = (int64_t)at * heads + kvh;
    auto part_of = [&](int z) { return reinterpret_cast<uint64_t *>(a.parts) + (unit * splits + z) * (int64_t)(PAIRS * 64 * W) + tid; };
    {
        uint64_t *part = part_of(split);
        auto put = [&](int i, float x, float y) {
            __hip_atomic_store(part + i * (64 * W), (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        if (row.mine) {
            put(PAIRS - 1, rows.m, l);
#pragma unroll
            for (int i = 0; i < HC / 4; i++) put(i, rows.o[i / 8][i % 8 * 2], rows.o[i / 8][i % 8 * 2 + 1]);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wavefront's stores are where everyone sees them
    __syncthreads();
    if (tid == 0) {
        const uint32_t others = __hip_atomic_fetch_add(a.arrived + unit, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_here = others == (uint32_t)(parts - 1);
        if (last_here) __hip_atomic_store(a.arrived + unit, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next call
    }
    __syncthreads();
    if (!last_here || !row.any) return;
    auto get = [&](int z, int i) {
        const uint64_t v = __hip_atomic_load(part_of(z) + i * (64 * W), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
    };
    float top = -INFINITY, all = 0.f;
    for (int z = 0; z < parts; z++) {
        const float2 ml = row.mine ? get(z, PAIRS - 1) : make_float2(-INFINITY, 0.f);
        if (ml.y != 0.f) top = fmaxf(top, ml.x);   // (else nothing that the row sees)
    }
#pragma unroll
    for (int i = 0; i < HC / 32; i++) rows.o[i] = tf16{};
    for (int z = 0; z < parts; z++) {
        if (!row.mine) break;
        const float2 ml = get(z, PAIRS - 1);
        float2 x[HC / 4];
#pragma unroll
        for (int i = 0; i < HC / 4; i++) x[i] = get(z, i);
        const bool counts = ml.y != 0.f;
        const float keep = counts ? __builtin_amdgcn_exp2f(ml.x - top) : 0.f;
        all += counts ? ml.y * keep : 0.f;
#pragma unroll
        for (int i = 0; i < HC / 4; i++) {
            float &x0 = reinterpret_cast<float *>(&rows.o[i / 8])[i % 8 * 2], &x1 = reinterpret_cast<float *>(&rows.o[i / 8])[i % 8 * 2 + 1];
            x0 += counts ? x[i].x * keep : 0.f, x1 += counts ? x[i].y * keep : 0.f;
        }
    }
    out(all);
}

template <int HD, int QT, int W>
int tiles_launch(hipc_ctx *ctx, Kv4Tiles a, size_t part_bytes) {
    constexpr int C = HD > 128 ? 2 : 1, HC = HD / C, ROWS = 32 * W / C;
    const int64_t rows = (int64_t)a.total * a.group, kv = a.cache.n_kv_heads;
    // tiles there can be: a sequence has some only if it brings more than a.most rows
    const int64_t tiles = rows / ROWS + std::min<int64_t>(a.cache.n_seqs, rows / (a.most + 1));
    a.slots = (int)std::min<int64_t>((int64_t)ctx->cu_count * tiles_per_cu(HD, W), part_bytes / ((size_t)(HC / 4 + 1) * 64 * W * 8));
    // us of a key tile (of half as many keys where heads are wider than 128), and of a part on its way through memory
    a.tile_us = (W == 8 ? (QT == 1 ? 3.1f : 5.2f) : QT == 1 ? 2.4f : 3.6f) * (HD <= 64 ? 0.6f : 1.f), a.part_us = 2.f;
    a.splits = ctx->tune.prompt_split;
    const int64_t groups = std::max<int64_t>(tiles * kv, ceil_div(a.slots, kv) * kv);
    HIPC_REFUSE(ctx, !grid_fits(groups, 64 * W), "hipc_kv4_prompt_attention: %d rows: too many for one call", a.total);
    hipLaunchKernelGGL((kv4_tiles_kernel<HD, QT, W>), (unsigned)groups, 64 * W, 0, ctx->stream, a);
    HIPC_LAUNCHED(ctx);
    return HIPC_OK;
}

}  // namespace

int kv4_tiles(hipc_ctx *ctx, const Kv4Tiles &a, int dtype, size_t part_bytes) {
    auto launch = [&](auto width) -> int {
        constexpr int HD = decltype(width)::value;
        // Eight wavefronts unpack a key tile once for twice as many rows as four and are half as many workgroups. us, four / eight: 2048 rows behind 30000 keys, 32 / 8 heads of 128 in
        // f16 1606 / 1505; 500 behind 8000 beside single tokens 160 / 155; prompts of up to 1024, 28 / 4 heads, 44 / 52; pieces of 1000 that see 512 keys, 4 / 1 heads of 256,
        // 31 / 38. How long sequences are is known on the device only: the table's room stands for it (a prompt of 1000, 28 / 4 heads of 128: 35.5, with a table of 32768 positions 39.7).
        const int64_t units = ceil_div((int64_t)a.total * a.group, HD > 128 ? 128 : 256) * a.cache.n_kv_heads;
        const int64_t room = a.cache.table_width * a.cache.page_size, keys = a.window > 0 ? std::min<int64_t>(room, a.window) : room;
        int waves = units >= (int64_t)ctx->cu_count || (keys >= 4096 && 4 * units >= (int64_t)ctx->cu_count) ? 8 : 4;
        if (ctx->tune.prompt_waves >= 4) waves = ctx->tune.prompt_waves;
        if (waves >= 8) return dtype == HIPC_F16 ? tiles_launch<HD, 1, 8>(ctx, a, part_bytes) : tiles_launch<HD, 2, 8>(ctx, a, part_bytes);
        return dtype == HIPC_F16 ? tiles_launch<HD, 1, 4>(ctx, a, part_bytes) : tiles_launch<HD, 2, 4>(ctx, a, part_bytes);
    };
    const int dim = a.cache.head_dim;
    return dim <= 64    ? launch(std::integral_constant<int, 64>())
           : dim <= 96  ? launch(std::integral_constant<int, 96>())
           : dim <= 128 ? launch(std::integral_constant<int, 128>())
                        : launch(std::integral_constant<int, 256>());
}

}  // namespace hipc
