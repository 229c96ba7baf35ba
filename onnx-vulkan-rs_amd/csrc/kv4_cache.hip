// The 4-bit key/value cache: storing rows (hipc_kv4_append) and reading them back (hipc_kv4_read).
//
// Both move bytes: 2 or 4 of a value on the outside, 5 bits in the cache, and memory bounds both (of two prompts of up to 8000 rows of 8 heads of 128
// in f32, 221 MB stored and read in 51 us, 4.3 TB/s; a copy's reading and writing 4.8). A wavefront takes 64 units of eight channels of one
// packed row (keys and values side by side), so a lane's outside access is 16 or 32 consecutive bytes and its codes one
// word; four neighbouring lanes hold a group and agree on its range without LDS.
#include <algorithm>

#include "kv4.h"
#include "lanes.h"

namespace hipc {

namespace {

struct Kv4Rows {
    hipc_kv4_cache cache;
    const int *starts;
    const void *k, *v;       // written by the reading kernel
    int64_t k_stride, v_stride;
    int total, units, chunks, wide;   // units of eight channels of a row, keys then values; wavefronts per row; rows on 16 bytes
};

// unit u of a row: which tensor, kv head, channel
struct Kv4Unit {
    int head, channel;
    bool value;
};
__device__ __forceinline__ Kv4Unit kv4_unit(const Kv4Rows &a, int u) {
    const int half = a.units >> 1, per_head = a.cache.head_dim >> 3;
    const bool value = u >= half;
    const int r = value ? u - half : u, h = r / per_head;
    return {h, (r - h * per_head) * 8, value};
}

template <typename T>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4Rows a) {
    const int w = kv4_wave(), lane = threadIdx.x & 63, row = w / a.chunks, u = (w - row * a.chunks) * 64 + lane;
    if (row >= a.total) return;
    const bool mine = u < a.units;
    const Kv4Unit unit = kv4_unit(a, mine ? u : 0);
    // the row's values are on their way while its place is looked up
    float x[8];
    const T *src = static_cast<const T *>(unit.value ? a.v : a.k) + (unit.value ? a.v_stride : a.k_stride) * row +
                   (int64_t)unit.head * a.cache.head_dim + unit.channel;
    kv4_load8(src, a.wide, x);
    int seq, first, end;
    if (!packed_sequence(a.starts, a.cache.n_seqs, a.total, row, &seq, &first, &end)) return;
    const Kv4Place place = kv4_place(a.cache, seq, kv4_length(a.cache, seq) - end + row);
    if (!place.there) return;

    uint32_t codes;
    const uint32_t params = kv4_quantize(x, &codes);
    if (!mine) return;
    const int64_t r = place.slot + (int64_t)unit.head * a.cache.page_size;
    uint8_t *to = static_cast<uint8_t *>(unit.value ? a.cache.v_codes : a.cache.k_codes) + r * (a.cache.head_dim / 2) + unit.channel / 2;
    *reinterpret_cast<uint32_t *>(to) = codes;
    if ((lane & 3) == 0) static_cast<uint32_t *>(unit.value ? a.cache.v_params : a.cache.k_params)[r * (a.cache.head_dim / kKv4Group) + unit.channel / kKv4Group] = params;
}

template <typename T>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Rows a) {
    const int w = kv4_wave(), lane = threadIdx.x & 63, row = w / a.chunks, u = (w - row * a.chunks) * 64 + lane;
    if (row >= a.total) return;
    int seq, first, end;
    if (!packed_sequence(a.starts, a.cache.n_seqs, a.total, row, &seq, &first, &end)) return;
    const Kv4Place place = kv4_place(a.cache, seq, kv4_length(a.cache, seq) - end + row);
    // Eight values a lane: of f16 a unit, 16 bytes; of f32 two halves of units, 64 lanes apart, so that a store is 1 KiB side by side either way. (The
    // codes unpack as pairs (i, i + 4): the halves' parameters go with them.)
    constexpr int HALF = sizeof(T) == 4 ? 2 : 1, N = 8 / HALF;
    typedef T TN __attribute__((ext_vector_type(N)));
    T *to[HALF];
    uint32_t codes = 0;
    kvh2 p[HALF] = {};
#pragma unroll
    for (int i = 0; i < HALF; i++) {
        const int at = HALF * (u - lane) + 64 * i + lane, half = HALF > 1 ? at & 1 : 0;   // in halves where there are such
        to[i] = nullptr;
        if (at >= HALF * a.units) continue;
        const Kv4Unit unit = kv4_unit(a, HALF > 1 ? at >> 1 : at);
        to[i] = static_cast<T *>(const_cast<void *>(unit.value ? a.v : a.k)) + (unit.value ? a.v_stride : a.k_stride) * row +
                (int64_t)unit.head * a.cache.head_dim + unit.channel + 4 * half;
        if (!place.there) continue;
        const int64_t r = place.slot + (int64_t)unit.head * a.cache.page_size;
        const uint8_t *from = static_cast<const uint8_t *>(unit.value ? a.cache.v_codes : a.cache.k_codes) + r * (a.cache.head_dim / 2) + unit.channel / 2 + 2 * half;
        if (HALF > 1) codes |= (uint32_t) * reinterpret_cast<const uint16_t *>(from) << (16 * i);
        else codes = *reinterpret_cast<const uint32_t *>(from);
        p[i] = static_cast<const kvh2 *>(unit.value ? a.cache.v_params : a.cache.k_params)[r * (a.cache.head_dim / kKv4Group) + unit.channel / kKv4Group];
    }
    kvh2 v[4];
    Kv4Unpack()(codes, kvh2{p[0].x, p[HALF - 1].x}, kvh2{p[0].y, p[HALF - 1].y}, v);
#pragma unroll
    for (int i = 0; i < HALF; i++) {
        if (!to[i]) continue;
        TN y;
#pragma unroll
        for (int j = 0; j < N; j++) y[j] = (T)v[j & 3][HALF > 1 ? i : j >> 2];
        if (a.wide) {
            __builtin_nontemporal_store(y, reinterpret_cast<TN *>(to[i]));
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) to[i][j] = y[j];
        }
    }
}

int rows_check(hipc_ctx *ctx, const char *who, const hipc_kv4_cache *c, int dtype, const void *starts, int64_t total, const void *K,
               int64_t k_stride, const void *V, int64_t v_stride, Kv4Rows *a) {
    if (int rc = kv4_check(ctx, who, c)) return rc;
    HIPC_REFUSE(ctx, dtype != HIPC_F16 && dtype != HIPC_F32, "%s: element type %d (f16 and f32 are taken)", who, dtype);
    HIPC_REQUIRE(ctx, total >= 0 && total <= 0x7fffffff, "%s: %lld rows", who, (long long)total);
    if (total == 0 || c->n_seqs == 0) return HIPC_OK;
    const size_t size = dtype == HIPC_F16 ? 2 : 4;
    const int64_t width = (int64_t)c->n_kv_heads * c->head_dim;
    HIPC_REQUIRE(ctx, K && V && starts, "%s: null pointer", who);
    HIPC_REQUIRE(ctx, k_stride >= width && v_stride >= width, "%s: rows %lld and %lld apart hold no %lld values", who, (long long)k_stride, (long long)v_stride, (long long)width);
    HIPC_REQUIRE(ctx, k_stride <= (int64_t)1 << 40 && v_stride <= (int64_t)1 << 40, "%s: rows too far apart", who);
    HIPC_REQUIRE(ctx, aligned(K, size) && aligned(V, size) && aligned(starts, 4), "%s: a pointer off its elements", who);
    a->cache = *c, a->starts = static_cast<const int *>(starts), a->k = K, a->v = V, a->k_stride = k_stride, a->v_stride = v_stride, a->total = (int)total;
    a->units = (int)(width / 4), a->chunks = (int)ceil_div(a->units, 64);
    a->wide = aligned(K, 16) && aligned(V, 16) && k_stride * size % 16 == 0 && v_stride * size % 16 == 0;
    HIPC_REFUSE(ctx, !grid_fits(ceil_div(total * a->chunks, 4), 256), "%s: %lld rows of %lld values: too many for one call", who, (long long)total, (long long)width);
    return HIPC_OK;
}

}  // namespace

int kv4_check(hipc_ctx *ctx, const char *who, const hipc_kv4_cache *c) {
    HIPC_REQUIRE(ctx, c, "%s: null cache", who);
    HIPC_REQUIRE(ctx, c->n_kv_heads > 0 && c->n_kv_heads <= 65535 && c->n_seqs >= 0 && c->n_seqs <= 1 << 20, "%s: %d kv heads, %d sequences", who, c->n_kv_heads, c->n_seqs);
    HIPC_REFUSE(ctx, c->head_dim <= 0 || c->head_dim > kKv4MaxHead || c->head_dim % kKv4Group != 0, "%s: head_dim %d (multiples of %d up to %d are taken)", who, c->head_dim, kKv4Group, kKv4MaxHead);
    HIPC_REFUSE(ctx, c->page_size < 16 || !is_pow2(c->page_size), "%s: pages of %d positions (powers of two from 16 on are taken)", who, c->page_size);
    HIPC_REQUIRE(ctx, c->n_pages >= 0 && c->n_pages <= 0x7fffffff && c->table_width >= 0, "%s: %lld pages, %lld a sequence", who, (long long)c->n_pages, (long long)c->table_width);
    HIPC_REQUIRE(ctx, c->table_width <= kKv4MaxPositions / c->page_size, "%s: a table of %lld pages of %d positions passes 2^30 positions", who, (long long)c->table_width, c->page_size);
    // (rows of the cache, one per position and kv head, are counted in 64 bits on the device)
    HIPC_REQUIRE(ctx, c->n_pages == 0 || (c->k_codes && c->k_params && c->v_codes && c->v_params), "%s: null pointer", who);
    HIPC_REQUIRE(ctx, aligned(c->k_codes, 16) && aligned(c->k_params, 16) && aligned(c->v_codes, 16) && aligned(c->v_params, 16), "%s: the cache's arrays lie on 16 bytes", who);
    HIPC_REQUIRE(ctx, c->n_seqs == 0 || (c->lengths && aligned(c->lengths, 4)), "%s: lengths", who);
    HIPC_REQUIRE(ctx, c->n_seqs == 0 || c->table_width == 0 || (c->table && aligned(c->table, 4)), "%s: page table", who);
    return HIPC_OK;
}

}  // namespace hipc

using namespace hipc;

extern "C" {

int hipc_kv4_append(hipc_ctx *ctx, const hipc_kv4_cache *cache, int dtype, const void *starts, int64_t total, const void *K,
                    int64_t k_stride, const void *V, int64_t v_stride) {
    return entry(ctx, [&]() -> int {
        Kv4Rows a{};
        if (int rc = rows_check(ctx, "hipc_kv4_append", cache, dtype, starts, total, K, k_stride, V, v_stride, &a)) return rc;
        if (a.total == 0) return HIPC_OK;
        const unsigned grid = (unsigned)ceil_div((int64_t)a.total * a.chunks, 4);
        if (dtype == HIPC_F16) hipLaunchKernelGGL((kv4_append_kernel<_Float16>), grid, 256, 0, ctx->stream, a);
        else hipLaunchKernelGGL((kv4_append_kernel<float>), grid, 256, 0, ctx->stream, a);
        HIPC_LAUNCHED(ctx);
        return HIPC_OK;
    });
}

int hipc_kv4_read(hipc_ctx *ctx, const hipc_kv4_cache *cache, int dtype, const void *starts, int64_t total, void *K, int64_t k_stride,
                  void *V, int64_t v_stride) {
    return entry(ctx, [&]() -> int {
        Kv4Rows a{};
        if (int rc = rows_check(ctx, "hipc_kv4_read", cache, dtype, starts, total, K, k_stride, V, v_stride, &a)) return rc;
        if (a.total == 0) return HIPC_OK;
        const unsigned grid = (unsigned)ceil_div((int64_t)a.total * a.chunks, 4);
        if (dtype == HIPC_F16) hipLaunchKernelGGL((kv4_read_kernel<_Float16>), grid, 256, 0, ctx->stream, a);
        else hipLaunchKernelGGL((kv4_read_kernel<float>), grid, 256, 0, ctx->stream, a);
        HIPC_LAUNCHED(ctx);
        return HIPC_OK;
    });
}

}  // extern "C"
