// Attention of packed new rows over the 4-bit cache: what the part for sequences that bring many rows (kv4_prompt.hip) gets from the entry point
// (kv4_attention.hip), which has the part for those that bring few.
#pragma once

#include "internal.h"

namespace hipc {

struct Kv4Tiles {
    hipc_kv4_cache cache;
    const void *q;
    void *y;
    int64_t q_stride, y_stride;
    const int *starts;
    int total, group, window, sinks, wide;   // wide: rows of Q and Y on 16 bytes
    int most;        // query rows (tokens times group) that a sequence has to pass to be in this part
    int slots;       // workgroups that run at once
    int splits;      // workgroups that share a tile's keys, or (not above 0) as many as tile_us and part_us say
    float tile_us, part_us;
    float scale;
    float *parts;    // what these exchange
    uint32_t *arrived;   // [slots]: parts of a unit that have come; all zero between calls
};
int kv4_tiles(hipc_ctx *ctx, const Kv4Tiles &a, int dtype, size_t part_bytes);

}  // namespace hipc
