// Attention over packed rows and over a paged cache, and the cache's rows: arguments of the launches, and what the serialiser, the
// validation and the launchers have to agree on.
#pragma once

#include "thip_kernels.h"

namespace thip {

constexpr int kMaxHeadDim = 256;

// Where the rows of a batch of sequences lie, and a paged cache of them.  A row of the cache is D elements: row (page * KVH + head) * PS + slot.
struct CacheArgs {
    const int32_t *starts;   // [S + 1]
    const int32_t *lengths;  // [S]; null: a row's position is its number in its sequence
    const int32_t *pages;    // [S][P]; null: key and value are rows [T][KVH][D]
    int32_t T, S, KVH, D;
    int32_t P, NP, PS;       // entries of a sequence's table, pages of the cache, positions of a page
    int32_t capacity;        // P * PS
    FastDiv ps;
};

struct CacheRowsArgs {
    CacheArgs c;
    uint16_t *key, *value;                 // rows; read by a write, written by a read
    void *key_cache, *value_cache;
    float *key_scales, *value_scales;      // null: the cache is bf16
    FastDiv kvh;
};
hipError_t launchCacheWrite(const CacheRowsArgs &a, const LaunchCtx &ctx);
hipError_t launchCacheRead(const CacheRowsArgs &a, const LaunchCtx &ctx);

struct AttentionArgs {
    CacheArgs c;
    const uint16_t *query;                 // [T][H][D]
    uint16_t *out;
    const void *key, *value;
    const float *key_scales, *value_scales;  // null: bf16
    int32_t H, G;                          // G: query heads of a key head
    float scale;
    int32_t window, sinks;                 // window 0: none (and sinks then 0)
    uint8_t *work;                         // attentionWorkspaceBytes
    size_t work_bytes;
};
hipError_t launchAttention(const AttentionArgs &a, const LaunchCtx &ctx);

// Bytes of partial results that a launch of these sizes may keep.  capacity: positions that a sequence can have.
inline uint64_t attentionWorkspaceBytes(int64_t T, int64_t S, int64_t H, int64_t KVH, int64_t D, int64_t capacity) { return 0; }

}  // namespace thip
