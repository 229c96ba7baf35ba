// Address model of the kernel that norms and turns heads (rotary.hip) behind gpu_model.h, driven through the entry points: rows,
// weights, frequencies, cache, page table and lengths in allocations of exactly their size, every load and store under
// AddressSanitizer; rows of every alignment and layout, heads of every size class, wavefronts that share rows, places that are
// none. Nothing between a row's heads and the next row is written. The refusals come first.
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "internal.h"

extern "C" {
const char *hipGetErrorString(hipError_t) { return "model"; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipStreamGetCaptureInfo_v2(hipStream_t, hipStreamCaptureStatus *status, unsigned long long *, hipGraph_t *, const hipGraphNode_t **, size_t *n) {
    *status = hipStreamCaptureStatusNone, *n = 0;
    return hipSuccess;
}
}

namespace {

hipc_ctx ctx;

void must(bool ok, const char *what) {
    if (ok) return;
    std::printf("FAILED %s (%s)\n", what, ctx.err.c_str());
    std::exit(1);
}

template <typename T>
struct Block {
    T *p;
    size_t n;
    explicit Block(size_t n_) : p(static_cast<T *>(gpu_model::alloc(n_ * sizeof(T)))), n(n_) {}
    ~Block() { gpu_model::release(p); }
    bool zero() const {
        for (size_t i = 0; i < n; i++)
            if (p[i] != T{}) return false;
        return true;
    }
};

struct Cache {
    Block<uint8_t> kc, vc;
    Block<uint32_t> kp, vp;
    Block<int> lengths, table;
    hipc_kv4_cache c;
    Cache(int pages, int page, int kv, int dim, int width)
        : kc((size_t)pages * page * kv * dim / 2), vc(kc.n), kp(kc.n / 16), vp(kp.n), lengths(1), table(width),
          c{kc.p, kp.p, vc.p, vp.p, pages, page, kv, dim, 1, lengths.p, table.p, width} {}
    bool zero() const { return kc.zero() && vc.zero() && kp.zero() && vp.zero(); }
};

void refusals() {
    Block<float> f(32), w(64);
    Block<uint16_t> q(4 * 128), k(4 * 128);
    Block<int> at(4), starts(2);
    Cache cache(2, 16, 2, 64, 2);
    const hipc_rotary_heads good{2, 2, 64, 64, 0, 1e-6f, 0.f, f.p, w.p, w.p};
    auto call = [&](const hipc_rotary_heads &h, int dtype = HIPC_F16, int64_t rows = 4, int64_t stride = 128, void *to = nullptr, const void *from = nullptr) {
        const int rc = hipc_rotary(&ctx, &h, dtype, at.p, rows, from ? from : q.p, stride, k.p, 128, to ? to : q.p, 128, k.p, 128);
        if (h.n_kv_heads == 2 && h.head_dim == 64)
            must(rc == hipc_kv4_append_rotary(&ctx, &cache.c, &h, dtype, starts.p, rows, from ? from : q.p, stride, k.p, 128, k.p, 128, to ? to : q.p, 128), "both calls refuse alike");
        return rc;
    };
    auto with = [&](auto change) {
        hipc_rotary_heads h = good;
        change(h);
        return call(h);
    };
    must(call(good) == HIPC_OK && with([](hipc_rotary_heads &h) { h.n_q_heads = 0; }) == HIPC_OK, "the call itself, and one of keys alone");
    must(with([](hipc_rotary_heads &h) { h.n_kv_heads = 0; }) == HIPC_OK, "one of queries alone");
    must(hipc_rotary(nullptr, &good, HIPC_F16, at.p, 4, q.p, 128, k.p, 128, q.p, 128, k.p, 128) == HIPC_ERR_INVALID, "no context");
    must(hipc_rotary(&ctx, nullptr, HIPC_F16, at.p, 4, q.p, 128, k.p, 128, q.p, 128, k.p, 128) == HIPC_ERR_INVALID, "no heads");
    must(hipc_rotary(&ctx, &good, HIPC_F16, nullptr, 4, q.p, 128, k.p, 128, q.p, 128, k.p, 128) == HIPC_ERR_INVALID, "no positions");
    must(hipc_rotary(&ctx, &good, HIPC_F16, (char *)at.p + 2, 4, q.p, 128, k.p, 128, q.p, 128, k.p, 128) == HIPC_ERR_INVALID, "positions off their elements");
    must(hipc_rotary(&ctx, &good, HIPC_F16, at.p, 4, q.p, 128, nullptr, 128, q.p, 128, k.p, 128) == HIPC_ERR_INVALID, "no keys");
    must(hipc_rotary(&ctx, &good, HIPC_F16, at.p, 4, q.p, 128, k.p, 128, q.p, 128, k.p, 127) == HIPC_ERR_INVALID, "rows that overlap");
    must(hipc_kv4_append_rotary(&ctx, nullptr, &good, HIPC_F16, starts.p, 4, q.p, 128, k.p, 128, k.p, 128, q.p, 128) == HIPC_ERR_INVALID, "no cache");
    must(hipc_kv4_append_rotary(&ctx, &cache.c, &good, HIPC_F16, nullptr, 4, q.p, 128, k.p, 128, k.p, 128, q.p, 128) == HIPC_ERR_INVALID, "no starts");
    must(hipc_kv4_append_rotary(&ctx, &cache.c, &good, HIPC_F16, starts.p, 4, q.p, 128, k.p, 128, nullptr, 128, q.p, 128) == HIPC_ERR_INVALID, "no values");
    hipc_rotary_heads other = good;
    other.n_kv_heads = 1;
    must(hipc_kv4_append_rotary(&ctx, &cache.c, &other, HIPC_F16, starts.p, 4, q.p, 128, k.p, 128, k.p, 128, q.p, 128) == HIPC_ERR_INVALID, "heads that are not the cache's");
    must(call(good, HIPC_I8) == HIPC_ERR_UNSUPPORTED, "types");
    must(call(good, HIPC_F16, -1) == HIPC_ERR_INVALID && call(good, HIPC_F16, (int64_t)INT_MAX + 1) == HIPC_ERR_INVALID, "row counts");
    must(call(good, HIPC_F16, 4, 127) == HIPC_ERR_INVALID && call(good, HIPC_F16, 4, ((int64_t)1 << 40) + 1) == HIPC_ERR_INVALID, "strides");
    must(call(good, HIPC_F16, 4, 128, (char *)q.p + 1) == HIPC_ERR_INVALID && call(good, HIPC_F16, 4, 128, nullptr, (char *)q.p + 1) == HIPC_ERR_INVALID, "pointers off their elements");
    for (int d : {0, -64}) must(with([&](hipc_rotary_heads &h) { h.head_dim = d, h.rotary_dim = 0; }) == HIPC_ERR_INVALID, "head sizes");
    must(with([](hipc_rotary_heads &h) { h.head_dim = 514; }) == HIPC_ERR_UNSUPPORTED, "a head too wide");
    for (int r : {-2, 33, 66}) must(with([&](hipc_rotary_heads &h) { h.rotary_dim = r; }) == HIPC_ERR_INVALID, "channels that turn");
    for (int n : {-1, 65536}) must(with([&](hipc_rotary_heads &h) { h.n_q_heads = n; }) == HIPC_ERR_INVALID, "head counts");
    for (float e : {-1e-6f, NAN, INFINITY}) must(with([&](hipc_rotary_heads &h) { h.norm_eps = e; }) == HIPC_ERR_INVALID, "eps");
    for (float v : {NAN, INFINITY}) must(with([&](hipc_rotary_heads &h) { h.amplitude = v; }) == HIPC_ERR_INVALID, "amplitude");
    must(with([](hipc_rotary_heads &h) { h.frequencies = nullptr; }) == HIPC_ERR_INVALID, "no frequencies");
    must(with([](hipc_rotary_heads &h) { h.q_norm = (const char *)h.q_norm + 2; }) == HIPC_ERR_INVALID, "weights off their elements");
    must(call(good, HIPC_F16, INT_MAX, 128) == HIPC_ERR_UNSUPPORTED, "launches that pass 32 bits");
    must(call(good, HIPC_F16, 0) == HIPC_OK && with([](hipc_rotary_heads &h) { h.rotary_dim = 0, h.frequencies = nullptr; }) == HIPC_OK, "no rows, nothing that turns");
    must(cache.zero(), "a refused call stores nothing");   // (and the ones above have no rows of the sequence's)
}

// rows `pad` values apart beyond their width, `off` values into their allocations, the last one ending it
template <typename T>
void turn(int dtype, int n_q, int n_kv, int dim, int rotary, int interleaved, bool norm, int rows, int pad, int off) {
    Block<float> f(rotary / 2 + (rotary == 0)), w(dim);
    Block<int> at(rows);
    for (int i = 0; i < rows; i++) at.p[i] = i * 7 - 3;
    const int qw = n_q * dim, kw = n_kv * dim, qs = qw + pad, ks = kw + pad;
    auto size = [&](int width, int stride) { return (size_t)off + (width ? (size_t)(rows - 1) * stride + width : 0); };
    Block<T> q(size(qw, qs)), k(size(kw, ks)), qo(size(qw, qs)), ko(size(kw, ks));
    for (size_t i = 0; i < q.n; i++) q.p[i] = (T)1;
    for (size_t i = 0; i < k.n; i++) k.p[i] = (T)1;
    for (size_t i = 0; i < qo.n; i++) qo.p[i] = (T)77;
    for (size_t i = 0; i < ko.n; i++) ko.p[i] = (T)77;
    const hipc_rotary_heads h{n_q, n_kv, dim, rotary, interleaved, 1e-6f, 1.5f, f.p, norm ? w.p : nullptr, norm ? w.p : nullptr};
    must(hipc_rotary(&ctx, &h, dtype, at.p, rows, q.p + off, qs, k.p + off, ks, qo.p + off, qs, ko.p + off, ks) == HIPC_OK, "rotary");
    auto check = [&](const Block<T> &b, int width, int stride) {
        for (size_t i = 0; i < b.n; i++) {
            const int64_t x = (int64_t)i - off;
            const bool inside = x >= 0 && x % stride < width;
            must(inside == (b.p[i] != (T)77), inside ? "every channel is written" : "what lies between rows stays");
        }
    };
    check(qo, qw, qs), check(ko, kw, ks);
}

template <typename T>
void store(int dtype, int n_q, int kv, int dim, int rotary, int interleaved, int page, std::vector<int> table, int pages, int length, int first, int n, int total, int pad, int off, bool stored) {
    Cache cache(pages, page, kv, dim, (int)table.size());
    std::memcpy(cache.table.p, table.data(), 4 * table.size());
    cache.lengths.p[0] = length;
    Block<int> starts(2);
    starts.p[0] = first, starts.p[1] = first + n;
    Block<float> f(rotary / 2 + (rotary == 0)), w(dim);
    for (int i = 0; i < dim; i++) w.p[i] = 1;
    const int qw = n_q * dim, kw = kv * dim, qs = qw + pad, ks = kw + pad;
    auto size = [&](int width, int stride) { return (size_t)off + (width ? (size_t)(total - 1) * stride + width : 0); };
    Block<T> q(size(qw, qs)), k(size(kw, ks)), v(k.n);
    for (size_t i = 0; i < q.n; i++) q.p[i] = (T)77;
    for (size_t i = 0; i < k.n; i++) k.p[i] = v.p[i] = (T)(1 + (int)(i % 97));
    const hipc_rotary_heads h{n_q, kv, dim, rotary, interleaved, 1e-6f, 0.f, f.p, nullptr, w.p};
    must(hipc_kv4_append_rotary(&ctx, &cache.c, &h, dtype, starts.p, total, q.p + off, qs, k.p + off, ks, v.p + off, ks, q.p + off, qs) == HIPC_OK, "append");
    must(stored != cache.zero(), stored ? "rows that have a place are stored" : "rows that have none are not");
}

template <typename T>
void all(int dtype) {
    for (int off : {0, 1, 4})
        for (int pad : {0, 4, 5})
            for (int interleaved : {0, 1})
                for (bool norm : {false, true}) {
                    turn<T>(dtype, 8, 2, 128, 128, interleaved, norm, 5, pad, off);
                    turn<T>(dtype, 3, 3, 96, 24, interleaved, norm, 3, pad, off);
                    turn<T>(dtype, 3, 1, 100, 36, interleaved, norm, 3, pad, off);
                    turn<T>(dtype, 2, 5, 33, 10, interleaved, norm, 3, pad, off);
                    turn<T>(dtype, 1, 1, 512, 512, interleaved, norm, 2, pad, off);
                    turn<T>(dtype, 1, 2, 510, 0, interleaved, norm, 2, pad, off);
                    turn<T>(dtype, 0, 2, 1, 0, interleaved, norm, 2, pad, off);
                    turn<T>(dtype, 70, 0, 2, 2, interleaved, norm, 2, pad, off);
                    for (int dim : {32, 96, 128, 160, 256}) {
                        store<T>(dtype, 3, 2, dim, dim, interleaved, 16, {2, 0, 1}, 3, 41, 0, 6, 6, pad, off, true);
                        store<T>(dtype, 3, 9, dim, 8, interleaved, 64, {0, 1}, 2, 70, 2, 5, 9, pad, off, true);
                        store<T>(dtype, 0, 1, dim, 10, interleaved, 16, {0}, 1, 3, 0, 8, 8, pad, off, true);
                        store<T>(dtype, 1, 1, dim, 0, interleaved, 16, {0, 1}, 2, 34, 0, 6, 6, pad, off, true);
                        store<T>(dtype, 1, 1, dim, 16, interleaved, 16, {0, 1}, 2, INT_MAX, 0, 6, 6, pad, off, false);
                        store<T>(dtype, 1, 1, dim, 16, interleaved, 16, {0, 1}, 2, INT_MIN, 0, 6, 6, pad, off, false);
                        store<T>(dtype, 1, 1, dim, 16, interleaved, 16, {-1, 2, INT_MAX, INT_MIN}, 2, 64, 0, 9, 9, pad, off, false);
                        store<T>(dtype, 1, 1, dim, 16, interleaved, 16, {0}, 1, 5, -3, 8, 5, pad, off, true);
                        store<T>(dtype, 1, 1, dim, 16, interleaved, 16, {0}, 1, 5, 3, -2, 5, pad, off, false);
                    }
                }
    turn<T>(dtype, 32, 8, 128, 128, 0, true, 3000, 0, 0);   // a row a wavefront
}

}  // namespace

int main() {
    for (int cus : {256, 1}) {
        ctx.cu_count = cus;
        refusals();
        all<_Float16>(HIPC_F16);
        all<float>(HIPC_F32);
    }
    std::printf("ok\n");
    return 0;
}
