// Attention over packed rows and over a paged cache, and the cache's rows: arguments of the launches, and what the serialiser, the
// validation and the launchers have to agree on.
#pragma once

#include <math.h>

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
    FastDiv g;
    int32_t window, sinks;                 // window 0: none (and sinks then 0)
    uint8_t *work;                         // attentionWorkspaceBytes
    size_t work_bytes;
};
hipError_t launchAttention(const AttentionArgs &a, const LaunchCtx &ctx);

// How a launch shares its work out.  An item is a tile of `rows` of a sequence's rows (a row: one query head of one token, the heads of a key
// head next to one another) against a run of blocks of `keys` positions; a workgroup has one.  The device cuts runs that
// are longer than their share of the launch, so that there are about `items` of that share's length, and the last workgroup of a tile to finish joins the parts.
struct AttentionPlan {
    bool tiles;                  // attention_tiles, or attention_stream
    bool fine;                   // weights of tiles in two parts
    int32_t rowsLog, keysLog;
    int32_t windowBlocks;        // blocks that a tile can see at most (with a window)
    int32_t minBlocks, maxParts; // blocks that a part has at least, and parts of a run at most
    int32_t fewBlocks;           // the same where few tiles are full, and of a stream among tiles
    bool splits;                 // runs may be cut
    int32_t items, whole;        // the launch's blocks by these: a part's, and those up to which a tile's run stays whole
    // A run of b blocks, in parts of B, is ceil(b / B) items, less than one more than b / B; the b / B of all are no more than `items`.  So there are fewer
    // than `items` above one a run (of `grid`), and of runs that are cut (b > B), less than 2 b / B each, fewer than twice `items` (of `slots`).
    int64_t grid;                // items at most
    int64_t slots;               // parts of runs that are cut at most
    FastDiv kvh;
    __host__ __device__ int32_t rows() const { return 1 << rowsLog; }
    __host__ __device__ int32_t keys() const { return 1 << keysLog; }
};

// Blocks of a part of a tile's run (of a stream's where the launch is of streams), up to how many a tile's run stays whole, and blocks of a part of a stream
// among tiles.
struct PartBlocks {
    int32_t tile, tileWhole, stream;
};
// total: blocks of all tiles of a key head, those of streams among tiles counted a quarter; full: tiles that are more than a few rows.
__host__ __device__ inline PartBlocks partBlocks(const AttentionPlan &p, float total, float full, int32_t KVH) {
    const float all = total * (float)KVH * 1.001f;  // sums of 32 bits
    const int32_t part = (int32_t)fminf(ceilf(all / (float)p.items), 1e8f), whole = (int32_t)fminf(ceilf(all / (float)p.whole), 1e8f);
    const int32_t least = full * (float)KVH < 128.0f ? p.fewBlocks : p.minBlocks;
    return {part > least ? part : least, p.tiles && whole > least ? whole : least, 4 * part > p.fewBlocks ? 4 * part : p.fewBlocks};
}

// Parts of a run.
__host__ __device__ inline int32_t partsOf(const AttentionPlan &p, int32_t blocks, int32_t part, int32_t whole) {
    if (!p.splits || blocks <= part || blocks <= whole) return 1;
    const int32_t parts = (int32_t)(((uint32_t)blocks + (uint32_t)part - 1) / (uint32_t)part);
    return parts < p.maxParts ? parts : p.maxParts;
}

// capacity: positions that a sequence can have; quantised: the cache is int8 (for the launch only, what is asked of a workspace is the same)
inline AttentionPlan attentionPlan(int64_t T, int64_t S, int64_t H, int64_t KVH, int64_t D, int64_t capacity, int64_t window, int64_t sinks,
                                   bool quantised = false) {
    AttentionPlan p;
    const int64_t G = H / KVH, rows = T * G;  // of one key head
    // Streams read a sequence's keys once for every 16 of its rows, tiles once for 128, at the rate of one wave's row block.  With 32 rows a sequence both
    // take the same, with 64 streams took a third more (16 sequences of 4096 positions, four heads of 128: 56 us and 43); heads of 256 have the
    // slower tiles, and few rows of them too few (64 tokens over 4096 positions, four heads: 79 us in tiles, 42 in streams).
    p.tiles = rows > 32 * S && (D <= 128 || rows * KVH > 2048);
    // The second part costs a prompt of 8192 tokens with 32 heads of 128 a third (153 us, 201 with it), four chunks of up to 512 a quarter (167, 210); the error of a
    // result goes from 1.4 times that of its rounding alone to 1.0.  Over many rows that is what it is; over few it may be 1.7 times in one call.
    p.fine = T * H < 8192;
    p.rowsLog = p.tiles ? 7 : 4;
    p.keysLog = p.tiles && D <= 64 ? 6 : 5;
    // Tiles: a part's results are 34 (heads of 64) to 133 KB that are written, read and joined.  So parts are of 2048 positions or more (parts of 512 cost
    // a prompt of 2048 tokens with 16 heads of 128 another 13 us, with a window of 512 another 28), shorter where full tiles leave half the CUs without any;
    // and a run is cut only if it is longer than the launch's blocks shared out over `whole` tiles, half of those that are on the chip at once (three
    // workgroups a CU, two with bf16 heads of 256): runs that are alike are cut where their halves still go all at once.  us, whole / cut, runs of 8192
    // positions, 32 heads of 128 over 8: 264 tiles 309 / 214, 384 322 / 239, 432 322 / 338, 480 322 / 340; 16 heads of 256 over 4: 176 502 / 365,
    // 264 508 / 563, 320 515 / 564; int8, of which one workgroup of heads of 256 has a CU: 192 654 / 681, 264 1207 / 1030, 360 1227 / 1036.  A third of the
    // tiles with runs of 16384 and two thirds of 4096: 384 tiles 533 / 249, 720 553 / 410; heads of 256, 264 981 / 489, 512 989 / 686.
    // Streams cost less to join and are cut wherever they are longer than their share: a token for each of 72 sequences, eight heads of 128, one of 32768
    // positions and the others of 200: 457 / 40; all of up to 4096: 171 / 166; 65 of up to 4096: 175 / 141.  That a table has room for long runs costs
    // where there is none (256 sequences of up to 128 positions, a table for 32768: 32 / 37).
    p.items = p.tiles ? 512 : 1024;
    p.whole = D > 128 && !quantised ? 260 : 390;
    p.maxParts = p.tiles ? 16 : 64;
    const int64_t keys = p.keys();
    const int64_t most = (rows / p.rows() + (S < T ? S : T)) * KVH;
    // a tile's window reaches over its own tokens too, and its first and last block need not be whole
    const int64_t windowed = (sinks + keys - 1) / keys + (window + (p.rows() - 1) / G + keys) / keys + 1;
    p.windowBlocks = (int32_t)(windowed < 0x7fffffff ? windowed : 0x7fffffff);
    int64_t blocks = (capacity + keys - 1) / keys;
    if (window && windowed < blocks) blocks = windowed;
    // Streams: a wave of a workgroup has a block at least, but two of them none where all the parts then still are few (a token of one sequence of
    // 1024 positions with one head of 256: 12.3 us in parts of four blocks, 11.2 of two; of 32 such with a window of 512: 12 and 13.5)
    p.minBlocks = p.tiles ? (int32_t)(2048 / keys) : most * blocks <= 256 ? 2 : 4;
    p.fewBlocks = p.tiles ? (int32_t)(256 / keys) : p.minBlocks;
    int64_t parts = (blocks + p.fewBlocks - 1) / p.fewBlocks;
    if (parts > p.maxParts) parts = p.maxParts;
    // What is cut is settled on the device, where the lengths are.  (With more tiles than this sums of their parts might pass 31 bits where starts
    // do not ascend.)
    p.splits = parts > 1 && most <= 65536;
    p.grid = p.splits ? (most * parts < most + p.items ? most * parts : most + p.items) : most;
    p.slots = p.splits ? (p.grid < 2 * p.items ? p.grid : 2 * p.items) : 0;
    p.kvh = makeFastDiv((uint32_t)KVH);
    return p;
}

// Bytes of partial results that a launch of these sizes may keep: a counter for each slot, 0 before and after every launch, and behind the counters of as
// many slots as there can be, for each row of a slot D sums, a maximum and a sum of weights.  The counters lie alike whatever the sizes are: launches that
// follow one another have one workspace, as long as the longest.
constexpr uint64_t kAttentionCounterBytes = 4 * 2 * 1024;
inline uint64_t attentionWorkspaceBytes(int64_t T, int64_t S, int64_t H, int64_t KVH, int64_t D, int64_t capacity, int64_t window, int64_t sinks) {
    const AttentionPlan p = attentionPlan(T, S, H, KVH, D, capacity, window, sinks);
    return p.slots ? kAttentionCounterBytes + (uint64_t)p.slots * (uint64_t)p.rows() * (uint64_t)(D + 4) * 4 : 0;
}

}  // namespace thip
