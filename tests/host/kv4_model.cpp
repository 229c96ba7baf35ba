// Address model of the 4-bit cache's storing and reading kernels (kv4_cache.hip) behind gpu_model.h, driven through the entry
// points: rows, cache, page table and lengths in allocations of exactly their size, every load and store under AddressSanitizer.
// Page numbers outside the cache, lengths that pass the table or lie below zero, positions in front of a sequence, rows behind
// the last one, rows off 16 bytes: nothing outside the allocations is touched, and rows that lie nowhere change nothing. The
// refusals come first. (Votes of a wavefront are stubs here, which one sequence alone does not notice.)
#include <climits>
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
    Cache k(2, 16, 2, 64, 2);
    Block<uint16_t> rows(4 * 128);
    Block<int> starts(2);
    auto call = [&](const hipc_kv4_cache &c, int dtype = HIPC_F16, int64_t total = 4, int64_t stride = 128, void *at = nullptr, const void *s = nullptr) {
        if (!at) at = rows.p;
        if (!s) s = starts.p;
        const int rc = hipc_kv4_append(&ctx, &c, dtype, s, total, at, stride, rows.p, 128);
        must(rc == hipc_kv4_read(&ctx, &c, dtype, s, total, at, stride, rows.p, 128), "both calls refuse alike");
        return rc;
    };
    auto with = [&](auto change) {
        hipc_kv4_cache c = k.c;
        change(c);
        return call(c);
    };
    must(call(k.c) == HIPC_OK, "the call itself");
    must(hipc_kv4_append(&ctx, nullptr, HIPC_F16, starts.p, 4, rows.p, 128, rows.p, 128) == HIPC_ERR_INVALID, "no cache");
    must(hipc_kv4_append(nullptr, &k.c, HIPC_F16, starts.p, 4, rows.p, 128, rows.p, 128) == HIPC_ERR_INVALID, "no context");
    must(call(k.c, HIPC_I8) == HIPC_ERR_UNSUPPORTED, "types");
    must(call(k.c, HIPC_F16, -1) == HIPC_ERR_INVALID && call(k.c, HIPC_F16, (int64_t)INT_MAX + 1) == HIPC_ERR_INVALID, "row counts");
    must(call(k.c, HIPC_F16, 4, 127) == HIPC_ERR_INVALID && call(k.c, HIPC_F16, 4, ((int64_t)1 << 40) + 1) == HIPC_ERR_INVALID, "strides");
    must(call(k.c, HIPC_F16, 4, 128, (char *)rows.p + 1) == HIPC_ERR_INVALID && call(k.c, HIPC_F16, 4, 128, nullptr, (char *)starts.p + 2) == HIPC_ERR_INVALID, "pointers off their elements");
    must(hipc_kv4_append(&ctx, &k.c, HIPC_F16, nullptr, 4, rows.p, 128, rows.p, 128) == HIPC_ERR_INVALID, "no starts");
    must(hipc_kv4_append(&ctx, &k.c, HIPC_F16, starts.p, 4, rows.p, 128, nullptr, 128) == HIPC_ERR_INVALID, "no values");
    for (int d : {0, -32, 16, 48, 288}) must(with([&](hipc_kv4_cache &c) { c.head_dim = d; }) == HIPC_ERR_UNSUPPORTED, "head sizes");
    for (int p : {0, 8, 24, -16}) must(with([&](hipc_kv4_cache &c) { c.page_size = p; }) == HIPC_ERR_UNSUPPORTED, "page sizes");
    for (int h : {0, -1, 65536}) must(with([&](hipc_kv4_cache &c) { c.n_kv_heads = h; }) == HIPC_ERR_INVALID, "kv heads");
    for (int s : {-1, (1 << 20) + 1}) must(with([&](hipc_kv4_cache &c) { c.n_seqs = s; }) == HIPC_ERR_INVALID, "sequences");
    for (int64_t n : {(int64_t)-1, (int64_t)INT_MAX + 1}) must(with([&](hipc_kv4_cache &c) { c.n_pages = n; }) == HIPC_ERR_INVALID, "page counts");
    for (int64_t w : {(int64_t)-1, ((int64_t)1 << 26) + 1, (int64_t)1 << 62}) must(with([&](hipc_kv4_cache &c) { c.table_width = w; }) == HIPC_ERR_INVALID, "table widths");
    must(with([&](hipc_kv4_cache &c) { c.k_codes = nullptr; }) == HIPC_ERR_INVALID, "no memory for codes");
    must(with([&](hipc_kv4_cache &c) { c.v_params = (char *)c.v_params + 4; }) == HIPC_ERR_INVALID, "memory off 16 bytes");
    must(with([&](hipc_kv4_cache &c) { c.lengths = nullptr; }) == HIPC_ERR_INVALID && with([&](hipc_kv4_cache &c) { c.table = nullptr; }) == HIPC_ERR_INVALID, "no lengths, no table");
    must(with([&](hipc_kv4_cache &c) { c.table = (char *)c.table + 2; }) == HIPC_ERR_INVALID, "a table off 4 bytes");
    must(call(k.c, HIPC_F16, INT_MAX, 128) == HIPC_ERR_UNSUPPORTED, "launches that pass 32 bits");
    must(k.zero(), "a refused call stores nothing");
    // nothing to do
    must(call(k.c, HIPC_F16, 0) == HIPC_OK && with([&](hipc_kv4_cache &c) { c.n_seqs = 0, c.lengths = c.table = nullptr; }) == HIPC_OK, "no rows, no sequences");
}

// `rows` packed rows, `n` of them the sequence's, which has `length` positions
template <typename T>
void move(int dtype, int kv, int dim, int page, std::vector<int> table, int pages, int length, int first, int n, int total, int pad, int off, bool stored) {
    Cache k(pages, page, kv, dim, (int)table.size());
    std::memcpy(k.table.p, table.data(), 4 * table.size());
    k.lengths.p[0] = length;
    Block<int> starts(2);
    starts.p[0] = first, starts.p[1] = first + n;
    const int width = kv * dim, stride = width + pad;
    const size_t size = off + (size_t)(total - 1) * stride + width;   // the last row ends its allocation
    Block<T> K(size), V(size);
    for (size_t i = 0; i < size; i++) K.p[i] = V.p[i] = (T)(1 + (int)(i % 97));
    must(hipc_kv4_append(&ctx, &k.c, dtype, starts.p, total, K.p + off, stride, V.p + off, stride) == HIPC_OK, "append");
    must(stored != k.zero(), stored ? "rows that have a place are stored" : "rows that have none are not");
    std::vector<T> was(K.p, K.p + size);
    must(hipc_kv4_read(&ctx, &k.c, dtype, starts.p, total, K.p + off, stride, V.p + off, stride) == HIPC_OK, "read");
    for (size_t i = 0; i < size; i++) {
        const int64_t at = (int64_t)i - off, row = at >= 0 ? at / stride : -1;
        const bool inside = at >= 0 && at % stride < width && row >= std::max(first, 0) && row < std::min(first + n, total);
        must(inside || K.p[i] == was[i], "what lies outside every sequence stays");
        if (inside && !stored) must(K.p[i] == (T)0 && V.p[i] == (T)0, "rows that have no place read as zeros");
    }
}

template <typename T>
void moves(int dtype) {
    for (int off : {0, 1})
        for (int pad : {0, 3, 8}) {
            move<T>(dtype, 1, 32, 16, {0}, 1, 16, 0, 16, 16, pad, off, true);
            move<T>(dtype, 3, 96, 16, {2, 0, 1}, 3, 41, 0, 41, 41, pad, off, true);           // pages in any order, the last one in part
            move<T>(dtype, 2, 256, 64, {0, 1}, 2, 70, 2, 5, 9, pad, off, true);                // rows before and behind the sequence's
            move<T>(dtype, 1, 64, 16, {0}, 1, 3, 0, 8, 8, pad, off, true);                     // five rows in front of position 0
            move<T>(dtype, 1, 64, 16, {0, 1}, 2, 34, 0, 6, 6, pad, off, true);                 // two rows behind the table
            move<T>(dtype, 1, 64, 16, {0, 1}, 2, 1 << 30, 0, 6, 6, pad, off, false);
            move<T>(dtype, 1, 64, 16, {0, 1}, 2, INT_MAX, 0, 6, 6, pad, off, false);
            move<T>(dtype, 1, 64, 16, {0, 1}, 2, INT_MIN, 0, 6, 6, pad, off, false);
            move<T>(dtype, 1, 64, 16, {-1, 2, INT_MAX, INT_MIN}, 2, 64, 0, 64, 64, pad, off, false);   // no pages
            move<T>(dtype, 1, 64, 16, {7, 1}, 2, 20, 0, 20, 20, pad, off, true);               // one that is none, one that is
            move<T>(dtype, 1, 64, 16, {0}, 1, 5, -3, 8, 5, pad, off, true);                     // starts below 0, an end behind the rows
            move<T>(dtype, 1, 64, 16, {0}, 1, 5, 2, 40, 5, pad, off, true);
            move<T>(dtype, 1, 64, 16, {0}, 1, 5, 3, -2, 5, pad, off, false);                    // an end before the start
        }
    // one page a sequence, and rows of more than a wavefront's units
    move<T>(dtype, 8, 128, 1024, {0}, 1, 700, 0, 33, 33, 0, 0, true);
}

}  // namespace

int main() {
    ctx.cu_count = 256;
    refusals();
    moves<_Float16>(HIPC_F16);
    moves<float>(HIPC_F32);
    std::printf("ok\n");
    return 0;
}
