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

// There is no tensor of rows, which row_starts would be kept inside of (CacheArgs::T).
constexpr int32_t kNoRows = 0x7fffffff;
struct CacheKeepArgs {
    CacheArgs c;
    const int32_t *accepted;               // [S][K]
    int32_t K;
    void *key_cache, *value_cache;
    float *key_scales, *value_scales;      // null: the cache is bf16
};
hipError_t launchCacheKeep(const CacheKeepArgs &a, const LaunchCtx &ctx);

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
    const int32_t *parents;                // [T]: the rows are trees; null: they follow one another
    int32_t tree_rows, tree_at;            // rows of a tree at most; where in LDS a workgroup has what it knows of its tree (set by the launch)
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
    int32_t fewBlocks;           // the same where few tiles are full, and of a stream among tiles; of trees' streams where the launch has less than manyBlocks
    int32_t manyBlocks, shortRun; // (0: no streams of trees) and the blocks of a run that stays whole
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

// Blocks in front of position `end`; a last block may pass 2^31.
__host__ __device__ inline int32_t blocksTo(const AttentionPlan &p, int32_t end) { return (int32_t)(((uint32_t)end + (uint32_t)p.keys() - 1) >> p.keysLog); }

// The blocks that rows at positions from `top` on (or at it) read, of which none sees a position behind `bottom`, of a sequence that has `length`: `sinks` blocks of the
// first positions that stay visible, then those from `window`, where the first row's window begins, on.  Rows below position 0 see nothing.
struct RowBlocks {
    int32_t sinks, window, all;
};
__host__ __device__ inline RowBlocks rowBlocks(const AttentionPlan &p, int32_t window, int32_t sinks, int32_t top, int32_t bottom, int32_t length) {
    const auto most = [](int32_t a, int32_t b) { return a > b ? a : b; };
    const auto least = [](int32_t a, int32_t b) { return a < b ? a : b; };
    const int32_t high = most(least(bottom + 1, length), 0), low = window ? most(most(top, -1) - window + 1, 0) : 0;
    const int32_t first = blocksTo(p, least(least(sinks, low), high)), from = most(low >> p.keysLog, first);
    return {first, from, first + most(blocksTo(p, high) - from, 0)};
}

// The blocks that a tile of a sequence can see at most.  treeRows: of its rows, those that can be a tree's; 0: rows follow one another.
__host__ __device__ inline int32_t seqBlocks(const AttentionPlan &p, int32_t window, int32_t sinks, int32_t treeRows, int32_t first, int32_t count, int32_t length) {
    const int32_t blocks = blocksTo(p, length);
    if (!window) return blocks;
    const int32_t some = blocks < p.windowBlocks ? blocks : p.windowBlocks;
    if (!treeRows) return some;
    // what the last tile reads; trees of a batch differ, and parts that are cut for the widest would be left empty (eight of up to 200 rows, windows
    // of 1024: 37.2 us, so 36.7; 33 to 60 tokens of ten sequences, eight heads of 128, windows of 40 41 and 25)
    const int32_t last = rowBlocks(p, window, sinks, first, first + (count < treeRows ? count : treeRows) - 1, length).all;
    return some < last ? some : last;
}

// Blocks of a part of a tile's run (of a stream's where the launch is of streams), up to how many a tile's run stays whole, and blocks of a part of a stream
// among tiles.
struct PartBlocks {
    int32_t tile, tileWhole, stream;
};
// total: blocks of all tiles of a key head, those of streams among tiles counted a quarter; full: tiles that are more than a few rows.
__host__ __device__ inline PartBlocks partBlocks(const AttentionPlan &p, float total, float full, int32_t KVH) {
    const float all = total * (float)KVH * 1.001f;  // sums of 32 bits
    const int32_t part = (int32_t)fminf(ceilf(all / (float)p.items), 1e8f), whole = (int32_t)fminf(ceilf(all / (float)p.whole), 1e8f);
    const int32_t least = (p.manyBlocks ? all < (float)p.manyBlocks : full * (float)KVH < 128.0f) ? p.fewBlocks : p.minBlocks;
    return {part > least ? part : least, p.tiles && whole > least ? whole : p.shortRun > least ? p.shortRun : least, 4 * part > p.fewBlocks ? 4 * part : p.fewBlocks};
}

// Parts of a run.
__host__ __device__ inline int32_t partsOf(const AttentionPlan &p, int32_t blocks, int32_t part, int32_t whole) {
    if (!p.splits || blocks <= part || blocks <= whole) return 1;
    const int32_t parts = (int32_t)(((uint32_t)blocks + (uint32_t)part - 1) / (uint32_t)part);
    return parts < p.maxParts ? parts : p.maxParts;
}

// capacity: positions that a sequence can have; quantised: the cache is int8 (but for trees the launch only knows it, what is asked of a workspace is the same)
// tree: rows of a tree at most (treeRows), 0: rows follow one another
constexpr int kTreeRows = 512;  // THIP_LM_TREE_ROWS
inline int64_t treeRows(int64_t T) { return T < kTreeRows ? T : kTreeRows; }
inline AttentionPlan attentionPlan(int64_t T, int64_t S, int64_t H, int64_t KVH, int64_t D, int64_t capacity, int64_t window, int64_t sinks,
                                   bool quantised = false, int64_t tree = 0) {
    AttentionPlan p;
    const int64_t G = H / KVH, rows = T * G;  // of one key head
    // Streams read a sequence's keys once for every 16 of its rows, tiles once for 128, at the rate of one wave's row block.  With 32 rows a sequence both
    // take the same, with 64 streams took a third more (16 sequences of 4096 positions, four heads of 128: 56 us and 43); heads of 256 have the
    // slower tiles, and few rows of them too few (64 tokens over 4096 positions, four heads: 79 us in tiles, 42 in streams).
    p.tiles = rows > 32 * S && (D <= 128 || rows * KVH > 2048);
    // The rows of a tree have all of the text before it to read, so few tiles are few workgroups with long runs, and streams the faster: up to 64 full tiles
    // (of heads above 128 32, of int8 128), but where the reading takes longer than the runs do, and a tile spares it for more streams than its work costs (four; of
    // int8, which streams read the better, six, and of its heads above 128, whose tiles are slow, where there are more blocks).  us, streams / tiles, by rows a sequence: 48 rows,
    // four key heads of 128, 2479 positions of int8 13 / 39; 516, one, 7323 with a window of 2275 17 / 50; 343, 20 sequences, eight of 80, 645 68 / 36; 257, three sequences,
    // eight of 256, 2909 166 / 77; 119, seven sequences, four of 128, 25556 260 / 121; 45, 46 sequences, two of 128, 19909 of int8 123 / 206; heads of 256 of int8: 205, eight
    // sequences, eight key heads, 4330 (17280 blocks of tiles) 188 / 212; 1538, two, four, 8192 (26624) 296 / 284; 553, two, eight, 20000 (50080) 557 / 437.  Not the faster
    // side: 37, 32 sequences, eight of 80, 1122 of int8, windows of 512, 31 / 34; 690, four sequences, eight of 256, 1024 of int8 81 / 90.
    if (tree) {
        const int64_t each = (rows - 1) / S + 1, streams = (each + 15) / 16, tiles = (each + 127) / 128, blocks = (window && window < capacity ? window : capacity) / 32;
        p.tiles = rows > 32 * S && (rows * KVH >= (D <= 128 ? 64 : quantised ? 128 : 32) * 128 ||
                                    (streams > (quantised ? 6 : 4) * tiles && tiles * S * KVH * blocks >= (!quantised ? 2048 : D <= 128 ? 16384 : 24576)));
    }
    // The second part costs a prompt of 8192 tokens with 32 heads of 128 a third (153 us, 201 with it), four chunks of up to 512 a quarter (167, 210); the error of a
    // result goes from 1.4 times that of its rounding alone to 1.0.  Over many rows that is what it is; over few it may be 1.7 times in one call.
    // Trees of as many rows pay 30.5 to 32.9 (eight of up to 200 rows, windows of 1024) and 159 to 230 (16 of up to 64 over int8: 25 registers spill, not 9).
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
    // Trees: parts of 512 positions or more (eight of up to 200 rows, four heads of 64, windows of 1024: 31.4, of 256 31.8, of 1024 32.9, of 2048 40.6), and of heads above 64
    // so that 640 are on the chip, nothing whole that is longer (16 of up to 64 rows over up to 8192 positions of int8, 32 heads of 128 over 8: 185 with up to half of
    // that whole, so 159).
    p.items = !p.tiles ? 1024 : tree && D > 64 ? 640 : 512;
    p.whole = tree && D > 64 ? 640 : D > 128 && !quantised ? 260 : 390;
    p.maxParts = p.tiles ? 16 : tree ? 32 : 64;
    const int64_t keys = p.keys();
    const int64_t most = (rows / p.rows() + (S < T ? S : T)) * KVH;
    // a tile's window reaches over its own tokens too (in a tree, whose rows may all stand at its first position, over those before it), and its first and
    // last block need not be whole
    const int64_t windowed = (sinks + keys - 1) / keys + (window + (tree ? tree : (p.rows() - 1) / G) + keys) / keys + 1;
    p.windowBlocks = (int32_t)(windowed < 0x7fffffff ? windowed : 0x7fffffff);
    int64_t blocks = (capacity + keys - 1) / keys;
    if (window && windowed < blocks) blocks = windowed;
    // Streams: a wave of a workgroup has a block at least, but two of them none where all the parts then still are few (a token of one sequence of
    // 1024 positions with one head of 256: 12.3 us in parts of four blocks, 11.2 of two; of 32 such with a window of 512: 12 and 13.5)
    // Trees' streams: 16 rows that are all there cost more to join than a token's few.  So parts are of eight blocks where those of four would be more workgroups than go
    // at once (two a CU, one of bf16 heads above 128), a run of up to eight stays whole, and one has up to 32.  us: 42 rows of two sequences over 2286 positions,
    // eight key heads of 80, 16.3 in parts of four, 14.3 of eight; 27 of 12 sequences over 1122, two of 256, 32 / 20; 64 of one sequence over 1024, one of 256, 16.7 /
    // 19.3; 16 of 15 sequences over up to 256, two of 96, 9.6 / 8.7 whole; 25 of one over 15087, two of 96, 64 parts 21.7, 32 17.9, 16 19.7.
    p.minBlocks = p.tiles ? (int32_t)((tree ? 512 : 2048) / keys) : tree ? 8 : most * blocks <= 256 ? 2 : 4;
    p.fewBlocks = p.tiles ? (int32_t)((tree ? 512 : 256) / keys) : tree ? 4 : p.minBlocks;
    p.manyBlocks = tree && !p.tiles ? (D > 128 && !quantised ? 1024 : 2048) : 0;
    p.shortRun = tree && !p.tiles ? 8 : 0;
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
inline uint64_t attentionWorkspaceBytes(int64_t T, int64_t S, int64_t H, int64_t KVH, int64_t D, int64_t capacity, int64_t window, int64_t sinks,
                                        int64_t tree = 0, bool quantised = false) {
    const AttentionPlan p = attentionPlan(T, S, H, KVH, D, capacity, window, sinks, quantised, tree);
    return p.slots ? kAttentionCounterBytes + (uint64_t)p.slots * (uint64_t)p.rows() * (uint64_t)(D + 4) * 4 : 0;
}

}  // namespace thip
