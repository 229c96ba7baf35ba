// The 4-bit key/value cache on the device: where a position's codes and parameters lie, which sequence a packed row
// belongs to, and what eight codes stand for. Shared by what stores, reads and attends to it (kv4_cache.hip,
// kv4_attention.hip) and, for the packed rows, by prompt_attention.hip.
#pragma once

#include <hip/hip_fp16.h>

#include "internal.h"
#include "lanes.h"

namespace hipc {

constexpr int kKv4Group = 32;      // channels that share a scale and a lowest value
constexpr int kKv4MaxHead = 256;
constexpr int kKv4MaxPositions = 1 << 30;   // of a sequence

typedef _Float16 kvh2 __attribute__((ext_vector_type(2)));

// Wave-wide: the sequence that packed row `row` belongs to, and its rows [first, end). The starts are counted 64 at a time;
// false where no sequence has the row (in front of the first, behind the last, or starts that do not ascend).
__device__ __forceinline__ bool packed_sequence(const int *starts, int n_seqs, int total, int row, int *seq, int *first, int *end) {
    const int lane = threadIdx.x & 63;
    int s = 0;
    for (int base = 1; base <= n_seqs; base += 64) {
        const int at = base + lane;
        const bool before = at <= n_seqs && starts[at < n_seqs ? at : n_seqs] <= row;
        const int c = __popcll(__ballot(before));
        s += c;
        if (c < 64) break;   // ascending starts: none behind this one is at or before the row
    }
    if (s >= n_seqs) return false;
    const int a = starts[s], b = starts[s + 1];
    *seq = s, *first = a < 0 ? 0 : a, *end = b > total ? total : b;
    return *first <= row && row < *end;
}

struct Kv4Place {
    int64_t slot;   // (page, kv head 0, place) as a row of heads: head h's row is slot + h * page_size
    bool there;
};
// position t of sequence s
__device__ __forceinline__ Kv4Place kv4_place(const hipc_kv4_cache &c, int s, int t) {
    const int shift = 31 - __builtin_clz((unsigned)c.page_size);
    if (t < 0 || (t >> shift) >= c.table_width) return {0, false};
    const int page = static_cast<const int *>(c.table)[(int64_t)s * c.table_width + (t >> shift)];
    if (page < 0 || page >= c.n_pages) return {0, false};
    return {((int64_t)page * c.n_kv_heads << shift) + (t & (c.page_size - 1)), true};
}
// what a sequence's length says, and the positions below it that the table has room for
__device__ __forceinline__ int kv4_length(const hipc_kv4_cache &c, int s) { return max(static_cast<const int *>(c.lengths)[s], 0); }
__device__ __forceinline__ int kv4_held(const hipc_kv4_cache &c, int length) { return min(length, (int)(c.table_width * c.page_size)); }

// Eight codes as f16 values, each lowest + code * scale rounded once: the code's bits under the exponent of 1024 (or, four
// bits further up, of 64) are that number plus the code; the subtraction is exact, and so is the product inside the fma.
// (A mask in a scalar register and the exponents in vector registers: one instruction takes the bits out and puts them in.)
struct Kv4Unpack {
    uint32_t low = 0x000f000fu, high = 0x00f000f0u, e1024 = 0x64006400u, e64 = 0x54005400u;
    __device__ __forceinline__ Kv4Unpack() {
        HIPC_PIN_SGPR(low);
        HIPC_PIN_SGPR(high);
        HIPC_PIN_VGPR(e1024);
        HIPC_PIN_VGPR(e64);
    }
    // nibbles 0 and 4, 1 and 5, 2 and 6, 3 and 7; a pair's scales and lowest values by scale(i), lowest(i)
    template <typename Scale, typename Lowest>
    __device__ __forceinline__ void operator()(uint32_t w, Scale scale, Lowest lowest, kvh2 (&v)[4]) const {
        auto part = [](uint32_t bits) { return __builtin_bit_cast(kvh2, bits); };
        const kvh2 k1024 = {(_Float16)1024.f, (_Float16)1024.f}, k64 = {(_Float16)64.f, (_Float16)64.f};
        v[0] = __builtin_elementwise_fma(part((w & low) | e1024) - k1024, scale(0), lowest(0));
        v[1] = __builtin_elementwise_fma(part((w & high) | e64) - k64, scale(1), lowest(1));
        w >>= 8;
        v[2] = __builtin_elementwise_fma(part((w & low) | e1024) - k1024, scale(2), lowest(2));
        v[3] = __builtin_elementwise_fma(part((w & high) | e64) - k64, scale(3), lowest(3));
    }
    __device__ __forceinline__ void operator()(uint32_t w, kvh2 scale, kvh2 lowest, kvh2 (&v)[4]) const {
        (*this)(w, [=](int) { return scale; }, [=](int) { return lowest; }, v);
    }
};

// eight elements as floats; `wide`: they lie on 16 bytes
template <typename T>
__device__ __forceinline__ void kv4_load8(const T *p, bool wide, float (&x)[8]) {
    typedef T T8 __attribute__((ext_vector_type(8)));
    if (wide) {
        const T8 v = *reinterpret_cast<const T8 *>(p);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)p[i];
    }
}

// Which wavefront of all this one is. Workgroups go round the eight XCDs; numbered so, the rows of an XCD lie side by side, and so do the cache
// lines that several positions share (a line of codes by two at 128 channels, one of parameters by eight). Two prompts of up to 8000 rows of 8 heads of
// 128 in f32, stored and read: 53.7 us, in the order of the workgroups 58.1.
__device__ __forceinline__ int kv4_wave() {
    const int each = (int)gridDim.x >> 3, b = blockIdx.x, at = b < each << 3 ? (b & 7) * each + (b >> 3) : b;
    return __builtin_amdgcn_readfirstlane(at * 4 + (threadIdx.x >> 6));
}

__device__ __forceinline__ float quad_min(float v) {
    v = fminf(v, lean_dpp<0xB1>(v));
    return fminf(v, lean_dpp<0x4E>(v));
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, lean_dpp<0xB1>(v));
    return fmaxf(v, lean_dpp<0x4E>(v));
}

// The quantizer's arithmetic is that of exact numbers up to its named roundings. A quotient is formed in f32 (off by less than 2^-17 below 31; beyond,
// the code is held to 0 or 15 either way) and decides unless it lies within 2^-14 of the border between two codes; then the remainder does, in 64 bits, where the difference and the
// product of a code (5 bits) and a scale (11) are exact. In 64 bits throughout, the kernel was bound by its 45 instructions a value
// (two prompts of up to 8000 rows of 8 heads of 128, f32, out of the nearest caches: 36.8 us, and 26.0 this way).
__device__ __forceinline__ int kv4_code(float x, float lowest, float scale, float inverse) {
    const float q = (x - lowest) * inverse, r = __builtin_rintf(q);
    int c = (int)r;
    if (__builtin_fabsf(__builtin_fabsf(q - r) - 0.5f) < 0x1p-14f) {
        const double d = (double)x - (double)lowest, rest = __builtin_fma(-(double)r, (double)scale, d), over = __builtin_fabs(rest) - 0.5 * (double)scale;
        if (over > 0.0 || (over == 0.0 && (c & 1))) c += rest > 0.0 ? 1 : -1;
    }
    return min(max(c, 0), 15);
}

// Eight channels a lane, a group of 32 of them in four neighbouring lanes (a quad): the lane's codes, and the group's parameters in all four.
__device__ __forceinline__ uint32_t kv4_quantize(float (&x)[8], uint32_t *codes_out) {
    bool nan = false;
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        nan |= x[i] != x[i];
        x[i] = fminf(fmaxf(x[i], -65408.f), 65408.f);
        lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
    }
    lo = quad_min(lo), hi = quad_max(hi);
    nan = quad_max(nan ? 1.f : 0.f) != 0.f;
    // (max - min) / 15: the product with 1 / 15, corrected by its remainder
    const double range = (double)hi - (double)lo, about = range * (1.0 / 15.0);
    float step = (float)__builtin_fma(__builtin_fma(-15.0, about, range), 1.0 / 15.0, about);
    HIPC_PIN_VGPR(step);   // the two roundings stay two (f32, then f16): left alone, the compiler makes one conversion of them
    const _Float16 lowest = (_Float16)lo, scale = (_Float16)step;
    const float inverse = scale > (_Float16)0 ? __builtin_amdgcn_rcpf((float)scale) : 0.f;
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) codes |= (uint32_t)kv4_code(x[i], (float)lowest, (float)scale, inverse) << (4 * i);
    *codes_out = codes;
    return nan ? 0x7e007e00u : __builtin_bit_cast(uint32_t, kvh2{scale, lowest});
}

// host side: what every call of the cache checks
int kv4_check(hipc_ctx *ctx, const char *who, const hipc_kv4_cache *c);
// the heads of an attention call, and the scale it uses
int attention_check(hipc_ctx *ctx, const char *who, const hipc_attention_heads *h, int dtype, float *scale);

}  // namespace hipc
