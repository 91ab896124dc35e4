// Attention of packed rows over themselves or over a paged cache (thip_lm_attention).
//
// o = sum_j w_j v_j / sum_j w_j, w_j = exp(scale (q . k_j) - m), over the positions j that the row sees; one pass over the keys with a
// running maximum m and a running sum, both scaled down where a later key raises m.  Exponents are to base 2, with log2(e) in the scale.
//
// Both products are taken transposed: S^T = K Q^T and O^T = V^T P^T.  A lane then holds scores of ONE query row (the result's column), so
// the softmax runs in the lane but for the maximum over the lanes that share the row, its scale of O is one number, and the scores it
// holds are, rounded to bf16, the right operand of the second product as they lie: the keys only have to be taken in the order in which the first
// product left them, which is the addresses of V's reads.  V's operand has a lane's values along the keys, across the rows that V lies in;
// ds_read_b64_tr turns them on the way out of LDS.
//
// Times below are means of calls one behind another, once the clocks have settled (the first ones after a pause take up to a tenth longer).  Where two
// forms are compared, both are of one call's inputs again and again, which the last cache helps by a few percent.
//
// Weights go into the second product as two bf16, one and what it leaves, in streams and in tiles of few rows, where that costs nothing; as one in tiles
// of many, where the second product's time counts (AttentionPlan::fine): off by half a step of 2^-8 each, which moves a result of independent values about as
// far as its own rounding does. Their sum is kept of the unrounded ones.  int8 keys and values are whole numbers that bf16 holds, so the scales are applied in fp32: a
// key's to its score, a value's to its weight.
#include "thip_attention.h"
#include "thip_attention_rows.h"
#include "thip_kernels_common.h"
#include "thip_lanes.h"

namespace thip {

constexpr float kLog2e = 1.4426950408889634f;

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

// Whether a row at position p sees position j (0 <= j): those of its window up to itself, and those before sinksOf(p).
__device__ __forceinline__ uint32_t windowOf(const AttentionArgs &a) { return a.window ? (uint32_t)a.window : 0x80000000u; }
__device__ __forceinline__ int sinksOf(const AttentionArgs &a, int p) { return min(a.sinks, p + 1); }
__device__ __forceinline__ bool sees(uint32_t window, int sinks, int p, int j) { return ((uint32_t)(p - j) < window) | (j < sinks); }

// ---- the work of a workgroup ----------------------------------------------------------------------------------------

// What sequence `s` brings: its rows, the positions it has, and the blocks that a tile of it can see at most.
struct SeqWork {
    int begin, count, first, length, tiles, blocks;
};
__device__ __forceinline__ SeqWork measureSeq(const AttentionArgs &a, const AttentionPlan &p, int s) {
    const CacheArgs &c = a.c;
    SeqWork w;
    const int there = min(s, c.S - 1);  // without a branch: of several sequences the loads go out together
    rowsOf(c, c.starts, there, &w.begin, &w.count);
    w.first = firstPosition(c, there, w.count);
    if (s >= c.S) w.count = 0;
    w.length = c.pages ? min(w.first + w.count, c.capacity) : w.count;
    w.tiles = (int)(((uint32_t)w.count * (uint32_t)a.G + (uint32_t)p.rows() - 1) >> p.rowsLog);
    w.blocks = seqBlocks(p, a.window, a.sinks, a.tree_rows, w.first, w.count, w.length);
    return w;
}

// Sum of the lanes up to this one.
template <typename T>
__device__ __forceinline__ T sumUpTo(T v) {
    v += moved<0x111>(v);       // from 1, 2, 4, 8 lanes down in the row of 16
    v += moved<0x112>(v);
    v += moved<0x114>(v);
    v += moved<0x118>(v);
    v += moved<0x142, 0xa>(v);  // the last of rows 0 and 2 to rows 1 and 3
    v += moved<0x143, 0xc>(v);  // the last of row 1 to rows 2 and 3
    return v;
}
__device__ __forceinline__ float sumOfWave(float v) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sumUpTo(v)), 63)); }

constexpr int kFewRows = 16;  // a stream's

// Among tiles, a sequence with few rows goes as a stream does, four blocks at once.
__device__ __forceinline__ bool goesByStream(const AttentionArgs &a, int count) { return a.c.pages && a.c.D <= 128 && count * a.G <= kFewRows; }

// A sequence's part of what blocksOfPart is made of: blocks, and tiles of more than a few rows.
__device__ __forceinline__ void addWork(const AttentionArgs &a, const AttentionPlan &p, const SeqWork &w, float *total, float *full) {
    const bool light = p.tiles && goesByStream(a, w.count);
    *total += (float)w.tiles * (float)w.blocks * (light ? 0.25f : 1.0f);
    if (w.count * a.G > kFewRows) *full += (float)w.tiles;
}

struct Item {
    SeqWork w;
    int seq, tile, head, split, splits, part;
    int slot;  // of its partial result; -1: the item is its rows' only one
};

// Items of a sequence, and those of them that are parts.
__device__ __forceinline__ int itemsOf(const AttentionArgs &a, const AttentionPlan &p, const PartBlocks &part, const SeqWork &w, int *splits, int *cut) {
    const bool light = p.tiles && goesByStream(a, w.count);
    *splits = partsOf(p, w.blocks, light ? part.stream : part.tile, light ? 0 : part.tileWhole);
    const int mine = w.tiles * *splits * a.c.KVH;
    *cut = *splits > 1 ? mine : 0;
    return mine;
}

// What a workgroup has in LDS while it looks for its item among more than 64 sequences.
struct Survey {
    float total[4], full[4];   // of each wave's
    int items[64], parts[64];  // of each group of sequences
};
constexpr int kManyItems = 1 << 24;  // more than a launch with parts has: where sums stop that starts which do not ascend make too large

// Item `index` of the launch.  Items lie sequence by sequence, a sequence's last tiles, which see most, first; key heads are next to one another, so
// that workgroups of one XCD (every eighth) read the same keys where there are eight heads.  Every wave of the workgroup comes to the same; false: there is
// none.  room: LDS, of which nothing is kept.
//
// A lane takes a sequence.  Of up to 64 each wave sums up all of them.  Of more the four waves share the sums, first the blocks, which the parts' length
// is made of, then the items of up to 64 groups; each goes on in the group that has its item.  A token for each of 1024 sequences of up to 128 positions,
// eight heads of 128: 121 us; with each wave going through all of them, 64 at a time, 148.
__device__ __forceinline__ bool findItem(const AttentionArgs &a, const AttentionPlan &p, int index, Item *out, void *room) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), S = a.c.S;
    PartBlocks part{0, 0, 0};
    int base = 0, end = S, before = 0, partsBefore = 0;  // sequences to look through, and what lies before them
    SeqWork w;
    if (S <= 64) {
        w = measureSeq(a, p, lane);
        if (p.splits) {
            float total = 0.0f, full = 0.0f;
            addWork(a, p, w, &total, &full);
            part = partBlocks(p, sumOfWave(total), sumOfWave(full), a.c.KVH);
        }
    } else {
        Survey *const held = (Survey *)room;
        const SeqWork own = measureSeq(a, p, threadIdx.x);  // in both sums
        if (p.splits) {
            float total = 0.0f, full = 0.0f;
            addWork(a, p, own, &total, &full);
#pragma unroll 4
            for (int s = threadIdx.x + 256; s < S; s += 256) addWork(a, p, measureSeq(a, p, s), &total, &full);
            total = sumOfWave(total);
            full = sumOfWave(full);
            if (lane == 0) {
                held->total[wave] = total;
                held->full[wave] = full;
            }
            __syncthreads();
            part = partBlocks(p, held->total[0] + held->total[1] + held->total[2] + held->total[3], held->full[0] + held->full[1] + held->full[2] + held->full[3], a.c.KVH);
        }
        const int group = 64 * ((S - 1) / (64 * 64) + 1), groups = (S - 1) / group + 1;
        for (int g = wave; g < groups; g += 4) {
            int items = 0, parts = 0;
            for (int s = g * group; s < min((g + 1) * group, S); s += 64) {
                int splits, cut;
                const SeqWork one = s + lane == (int)threadIdx.x ? own : measureSeq(a, p, s + lane);
                items += __builtin_amdgcn_readlane(sumUpTo(itemsOf(a, p, part, one, &splits, &cut)), 63);
                if (p.splits) {
                    parts += __builtin_amdgcn_readlane(sumUpTo(cut), 63);
                    items = min(items, kManyItems);
                    parts = min(parts, kManyItems);
                }
            }
            if (lane == 0) {
                held->items[g] = items;
                held->parts[g] = parts;
            }
        }
        __syncthreads();
        const int items = lane < groups ? held->items[lane] : 0, parts = lane < groups ? held->parts[lane] : 0;
        const int upTo = sumUpTo(items), partsUpTo = sumUpTo(parts);
        const uint64_t found = __ballot(upTo - items <= index && index < upTo);
        __syncthreads();
        if (!found) return false;
        const int g = __builtin_ctzll(found);
        before = __builtin_amdgcn_readlane(upTo - items, g);
        partsBefore = __builtin_amdgcn_readlane(partsUpTo - parts, g);
        base = g * group;
        end = min(base + group, S);
        w = measureSeq(a, p, base + lane);
    }
    for (;;) {
        int splits, cut;
        const int mine = itemsOf(a, p, part, w, &splits, &cut), upTo = sumUpTo(mine), cutUpTo = p.splits ? sumUpTo(cut) : 0, at = index - before;
        const uint64_t found = __ballot(upTo - mine <= at && at < upTo);
        if (found) {
            const int l = __builtin_ctzll(found);
            out->w.begin = __builtin_amdgcn_readlane(w.begin, l);
            out->w.count = __builtin_amdgcn_readlane(w.count, l);
            out->w.first = __builtin_amdgcn_readlane(w.first, l);
            out->w.length = __builtin_amdgcn_readlane(w.length, l);
            out->w.tiles = __builtin_amdgcn_readlane(w.tiles, l);
            out->w.blocks = __builtin_amdgcn_readlane(w.blocks, l);
            out->seq = base + l;
            out->splits = __builtin_amdgcn_readlane(splits, l);
            const uint32_t local = (uint32_t)(at - __builtin_amdgcn_readlane(upTo - mine, l));
            uint32_t rest = fastDiv(local, p.kvh);
            out->head = (int)(local - rest * (uint32_t)a.c.KVH);
            out->split = out->part = 0;
            out->slot = -1;
            if (out->splits > 1) {
                const uint32_t tile = rest / (uint32_t)out->splits;
                out->split = (int)(rest - tile * (uint32_t)out->splits);
                rest = tile;
                out->part = (int)(((uint32_t)out->w.blocks + (uint32_t)out->splits - 1) / (uint32_t)out->splits);
                out->slot = partsBefore + __builtin_amdgcn_readlane(cutUpTo - cut, l) + (int)local;
            }
            out->tile = out->w.tiles - 1 - (int)rest;
            // starts that do not ascend may make more of them: a run whose parts would not all have a place, or a workgroup, is left out whole, or its
            // counter would not come back to 0
            const int behind = (out->splits - 1 - out->split) * a.c.KVH;
            return out->splits == 1 || (out->slot + behind < p.slots && (int64_t)index + behind < p.grid);
        }
        const int these = __builtin_amdgcn_readlane(upTo, 63);
        base += 64;
        if (base >= end || at < these) return false;  // the second: sums that are too large
        before += these;
        partsBefore += __builtin_amdgcn_readlane(cutUpTo, 63);
        w = measureSeq(a, p, base + lane);
    }
}

// The blocks that a tile reads: those of the first positions that stay visible, then from its first row's window on.  Blocks [from, to)
// of that order are the item's.
struct Span {
    int rows;          // of the tile
    int sinkBlocks, windowBlock;
    int from, to;
};
template <bool TREE>
__device__ __forceinline__ Span spanOf(const AttentionArgs &a, const AttentionPlan &p, const Item &it) {
    Span s;
    const int r0 = it.tile << p.rowsLog;
    s.rows = min(p.rows(), it.w.count * a.G - r0);
    const int last = (int)fastDiv((uint32_t)(r0 + s.rows - 1), a.g);
    // of a tree places, whose rows may stand at any positions from the first on
    const int top = it.w.first + (TREE ? 0 : (int)fastDiv((uint32_t)r0, a.g)), bottom = it.w.first + (TREE ? min(last, a.tree_rows - 1) : last);
    const RowBlocks blocks = rowBlocks(p, a.window, a.sinks, top, bottom, it.w.length);
    s.sinkBlocks = blocks.sinks;
    s.windowBlock = blocks.window;
    const int all = blocks.all;
    s.from = min(it.splits > 1 ? it.split * it.part : 0, all);
    s.to = it.splits > 1 ? min(all, s.from + it.part) : all;
    return s;
}
__device__ __forceinline__ int blockStart(const AttentionPlan &p, const Span &s, int b) { return (b < s.sinkBlocks ? b : b - s.sinkBlocks + s.windowBlock) << p.keysLog; }

// Row of the keys (elements / D) that position j of a sequence has; -1: none.  In a loop a position is asked for a block ahead of the loads that
// need its row, and before the loads of the block before: loads come back in order, and a wait for an entry of the table would be one for all that
// were sent before it.
template <bool PAGED>
struct KeyAsk {
    PageAsk page;
};
template <>
struct KeyAsk<false> {
    int row;
};
template <bool PAGED>
__device__ __forceinline__ KeyAsk<PAGED> askKey(const AttentionArgs &a, const Item &it, int j, bool in) {
    if constexpr (PAGED) return {askPage(a.c, it.seq, j, in ? it.w.length : 0)};
    else return {(in & (j < it.w.length)) ? (it.w.begin + j) * a.c.KVH + it.head : -1};
}
template <bool PAGED>
__device__ __forceinline__ int keyRow(const AttentionArgs &a, const Item &it, const KeyAsk<PAGED> &q) {
    if constexpr (PAGED) return rowOf(a.c, q.page, it.head);
    else return q.row;
}

// ---- partial results ---------------------------------------------------------------------------------------------------

// A slot holds, for each row of a stream, D sums, then the maximum and the sum of weights; of a tile, the sums as a wave has them (16 bytes a lane,
// the waves' one behind the other, so that what is stored and read is whole lines), then the two of each row.  They go from workgroup to workgroup, which may be on
// different XCDs, past the caches, by loads and stores at the device's scope (a fence would write the XCD's whole L2 back).
constexpr int kDeviceScope = 16;  // sc1
__device__ __forceinline__ __amdgpu_buffer_rsrc_t slotsOf(const AttentionArgs &a, const AttentionPlan &p) {
    return __builtin_amdgcn_make_buffer_rsrc(a.work + kAttentionCounterBytes, 0, (int)((uint32_t)p.slots * (uint32_t)p.rows() * (uint32_t)(a.c.D + 4) * 4u), 0x00020000);
}
__device__ __forceinline__ uint32_t slotRow(const AttentionArgs &a, const AttentionPlan &p, int slot, int r) {
    return (((uint32_t)slot << p.rowsLog) + (uint32_t)r) * (uint32_t)(a.c.D + 4) * 4u;
}
// Of a tile: the sums, and its rows' maxima and sums of weights.
__device__ __forceinline__ uint32_t tileSums(const AttentionArgs &a, int slot) { return (uint32_t)slot * 128u * (uint32_t)(a.c.D + 4) * 4u; }
__device__ __forceinline__ uint32_t tileStats(const AttentionArgs &a, int slot, int r) { return tileSums(a, slot) + 512u * (uint32_t)a.c.D + 16u * (uint32_t)r; }
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void put4(__amdgpu_buffer_rsrc_t to, uint32_t at, float x, float y, float z, float w) {
    __builtin_amdgcn_raw_buffer_store_b128(v4u{__float_as_uint(x), __float_as_uint(y), __float_as_uint(z), __float_as_uint(w)}, to, (int)at, 0, kDeviceScope);
}
__device__ __forceinline__ v4f get4(__amdgpu_buffer_rsrc_t from, uint32_t at) {
    return __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(from, (int)at, 0, kDeviceScope));
}

// Every thread of a workgroup that has stored its part: the last one of the run's to come here adds the parts, in their order, scaled to
// their common maximum.  room: LDS that nobody uses any more, ROWS (PARTS + 1) floats and one.
template <int ROWS, int PARTS, int ELEMS>
__device__ __forceinline__ void joinParts(const AttentionArgs &a, const AttentionPlan &p, const Item &it, int rows, float *room) {
    constexpr int LANES = 256 / ROWS, EACH = PARTS / LANES;  // threads of a row, and parts of each
    const int tid = threadIdx.x, D = a.c.D, first = it.slot - it.split * a.c.KVH;
    const auto slots = slotsOf(a, p);
    uint32_t *const counter = (uint32_t *)a.work + first;
    int *const last = (int *)room;
    float *const factors = room + 1, *const totals = factors + ROWS * PARTS;
    waitVmcnt<0>();  // this wave's part is where the others will look
    __syncthreads();
    if (tid == 0) *last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u == (uint32_t)it.splits;
    __syncthreads();
    if (!*last) return;
    if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // Several elements of a thread's and several parts at once, the first of them while the factors are made.  Of a stream's 16 rows one element, as
    // the registers of more leave room for fewer workgroups (trees of 42 rows over 2286 positions, eight key heads of 80: 16.1 us, with four 17.8); but four in
    // trees' heads of 256, of which a CU has one workgroup in any case, and 16 rows' parts to join (16 rows over 1024 positions 17.3 us, with four 16.8).
    constexpr int BATCH = ROWS == 128 ? 4 : 8;
    constexpr bool TILE = ROWS == 128;
    const int pieces = D >> 2, all = TILE ? ((rows + 31) >> 5) * 8 * D : rows * pieces;
    const uint32_t step = TILE ? tileSums(a, a.c.KVH) : slotRow(a, p, a.c.KVH, 0), sums = TILE ? tileSums(a, first) : slotRow(a, p, first, 0);
    v4f part[ELEMS][BATCH];
    auto getParts = [&](int e0, int s) {
#pragma unroll
        for (int i = 0; i < ELEMS; i++) {
            if (ROWS < 128 && ELEMS > 1 && e0 - tid + 256 * i >= all) continue;
            const int e = min(e0 + 256 * i, all - 1);
            const uint32_t from = sums + (uint32_t)(TILE ? e : e + e / pieces) * 16u;  // a stream's rows are D + 4 long
#pragma unroll
            for (int k = 0; k < BATCH; k++) part[i][k] = get4(slots, from + min(s + k, it.splits - 1) * step);
        }
    };
    // row and first column of an element
    auto rowOf = [&](int e) { return TILE ? e / (8 * D) * 32 + (e & 31) : e / pieces; };
    auto columnOf = [&](int e, int r) { return TILE ? (e % (8 * D) >> 6) * 8 + ((e >> 5) & 1) * 4 : 4 * (e - r * pieces); };
    getParts(tid, 0);
    {
        const int r = tid / LANES, mine = tid % LANES;
        v4f stats[EACH];
        float most = -INFINITY, total = 0.0f;
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int s = e * LANES + mine;
            const int slot = first + min(s, it.splits - 1) * a.c.KVH, row = min(r, rows - 1);
            stats[e] = get4(slots, TILE ? tileStats(a, slot, row) : slotRow(a, p, slot, row) + D * 4);
            if (s >= it.splits) stats[e] = v4f{-INFINITY, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int e = 0; e < EACH; e++) most = fmaxf(most, stats[e][0]);
        most = overLanes<LANES>(most, [](float x, float y) { return fmaxf(x, y); });
        const float shift = most == -INFINITY ? 0.0f : most;
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const float f = __builtin_amdgcn_exp2f(stats[e][0] - shift);
            factors[r * PARTS + e * LANES + mine] = f;
            total += f * stats[e][1];
        }
        total = overLanes<LANES>(total, [](float x, float y) { return x + y; });
        if (mine == 0) totals[r] = total == 0.0f ? 0.0f : 1.0f / total;
    }
    __syncthreads();
    for (int e0 = tid; e0 < all; e0 += 256 * ELEMS) {
        v4f sum[ELEMS];
#pragma unroll
        for (int i = 0; i < ELEMS; i++) sum[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < it.splits; s += BATCH) {
            if (e0 != tid || s != 0) getParts(e0, s);
#pragma unroll
            for (int i = 0; i < ELEMS; i++) {
                const int r = rowOf(min(e0 + 256 * i, all - 1));
#pragma unroll
                for (int k = 0; k < BATCH; k++) {
                    if (s + k < it.splits) sum[i] += factors[r * PARTS + s + k] * part[i][k];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < ELEMS; i++) {
            const int e = e0 + 256 * i, r = rowOf(e), d = columnOf(e, r);
            if (e >= all || r >= rows) continue;
            const int mine = it.tile * ROWS + r, token = (int)fastDiv((uint32_t)mine, a.g);
            *(v2i *)(a.out + ((int64_t)(it.w.begin + token) * a.H + it.head * a.G + mine - token * a.G) * D + d) =
                v2i{packBf16(sum[i][0] * totals[r], sum[i][1] * totals[r]), packBf16(sum[i][2] * totals[r], sum[i][3] * totals[r])};
        }
    }
}

// ---- trees -------------------------------------------------------------------------------------------------------------

// What a workgroup knows of its tree, in LDS: for each row of the sequence up to its tile's last where the run of rows that ends in it begins (each the next one's
// parent, all in one word of a path) and that one's parent; then for each token of its tile the position in the text at which it stands (-1: it sees nothing) and a bit for
// each row of its path that it sees.  A lane follows its token's path by runs, so that a chain takes a step a word; windows are taken off here, where a row's depth is
// known, and cost the blocks of keys nothing.  (Row by row, with the words held back until they were whole: eight trees of 200 rows over 264 positions, 16 heads of 64 over
// 4: 22.2 us, so 21.3.)
struct Tree {
    const int32_t *position;  // [tokens]
    const uint32_t *seen;     // [tokens][stride]
    int words, stride, token0;
    bool all;                 // every row of the tile stands somewhere
    int bottom;               // with a window: none of them stands further down
};
__host__ __device__ constexpr int treeWords(int rows) { return (rows + 31) / 32; }
__host__ __device__ constexpr int treeStride(int rows) { return treeWords(rows) | 1; }  // odd: 32 rows at one word are in as many banks
__host__ __device__ constexpr int treeBytes(int rows, int tokens) { return 4 * (1 + rows + tokens * (1 + treeStride(rows))); }

// Every thread of the workgroup calls it.  paths: the item has keys of the tree, so the seen rows are asked for.
__device__ __forceinline__ Tree plantTree(const AttentionArgs &a, const Item &it, int8_t *smem, int r0, int rows, bool paths) {
    int32_t *const deepest = (int32_t *)(smem + a.tree_at);
    uint32_t *const runs = (uint32_t *)(deepest + 1);  // a row's run: its first row, the parent of that + 1 in the upper half
    const int tid = threadIdx.x, lane = tid & 63, count = min(it.w.count, a.tree_rows), base = it.w.first;
    Tree t;
    t.words = treeWords(a.tree_rows);
    t.stride = treeStride(a.tree_rows);
    t.token0 = (int)fastDiv((uint32_t)r0, a.g);
    const int tokens = (int)fastDiv((uint32_t)(r0 + rows - 1), a.g) - t.token0 + 1;
    int32_t *const position = (int32_t *)(runs + a.tree_rows);
    uint32_t *const seen = (uint32_t *)(position + tokens);
    t.position = position;
    t.seen = seen;
    t.all = base + t.token0 >= 0 && t.token0 + tokens <= count;
    const bool walks = paths || a.window;
    if (walks) {
        const int needed = min(count, t.token0 + tokens);
        for (int first = tid - lane; first < needed; first += 256) {
            const int i = first + lane;
            int parent = i < needed ? a.parents[it.w.begin + i] : -1;
            parent = parent < i ? max(parent, -1) : -1;
            const uint64_t linked = __ballot((lane & 31) && parent == i - 1);
            const uint32_t ends = ~(uint32_t)(linked >> (lane & 32)) & ((2u << (lane & 31)) - 1);  // rows of the word up to this one that begin a run
            const int begin = (lane & 32) + 31 - __builtin_clz(ends);
            const int above = __shfl(parent, begin);
            if (i < needed) runs[i] = (uint32_t)(first + begin) | (uint32_t)(above + 1) << 16;
        }
        if (paths) {
            for (int i = tid; i < tokens * t.stride; i += 256) seen[i] = 0;
        }
        if (tid == 0) *deepest = -1;
        __syncthreads();
    }
    if (tid < tokens) {
        const int row = t.token0 + tid;
        const bool stands = row < count && base + row >= 0;
        uint32_t *const mine = seen + tid * t.stride;
        int here = -1, depth = -1;
        auto bits = [](int from, int to) { return (2u << (to & 31)) - (1u << (from & 31)); };
        if (stands) {
            if (walks) {
                for (int r = row; r >= 0;) {
                    const uint32_t run = runs[r];
                    const int first = (int)(run & 0xffff);
                    if (paths) __hip_atomic_fetch_or(mine + (r >> 5), bits(first, r), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                    depth += r - first + 1;
                    r = (int)(run >> 16) - 1;
                }
            }
            here = base + (a.window ? depth : row);
        }
        position[tid] = here;
        if (a.window) __hip_atomic_fetch_max(deepest, here, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        if (paths && a.window && depth >= a.window) {
            // rows of the path that lie `back` below this one: those from the window's end on are not seen, up to those of the first positions
            const int last = here < a.sinks ? -1 : here - a.sinks;
            for (int r = row, back = 0; r >= 0;) {
                const uint32_t run = runs[r];
                const int first = (int)(run & 0xffff), from = max(back, a.window), to = min(back + r - first, last);
                if (from <= to) __hip_atomic_fetch_and(mine + (r >> 5), ~bits(r - (to - back), r - (from - back)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                back += r - first + 1;
                r = (int)(run >> 16) - 1;
            }
        }
    }
    __syncthreads();
    t.bottom = a.window ? __builtin_amdgcn_readfirstlane(*deepest) : 0;
    return t;
}
__device__ __forceinline__ int positionOf(const Tree &t, int token) { return t.position[token - t.token0]; }
// Whether a token sees the rows of the tree from `first` on (it may lie before the tree), a bit each.
__device__ __forceinline__ uint32_t seenFrom(const Tree &t, int token, int first) {
    const uint32_t *const mine = t.seen + (token - t.token0) * t.stride;
    const int w = first >> 5;
    const uint32_t lo = (uint32_t)w < (uint32_t)t.words ? mine[w] : 0u, hi = (uint32_t)(w + 1) < (uint32_t)t.words ? mine[w + 1] : 0u;
    return (uint32_t)((((uint64_t)hi << 32) | lo) >> (first & 31));
}

// Which of the 32 positions from `from` on a token at `pos` sees, a bit each: those of the text in front of the tree that are in its window or among the first ones, and the
// tree's (near: there may be some).  In words: where a lane read and compared four at a time, the trees above took 21.3 us, so 16.5 (a chunk of as many rows 12.3); with
// windows of 1024 over up to 4096 positions 35.2 and 31.3; 16 trees of up to 64 rows over up to 8192 positions of int8, 32 heads of 128 over 8, 171 and 159.
__device__ __forceinline__ uint32_t seenBits(const AttentionArgs &a, const Tree &t, const Item &it, int token, int pos, int from, bool near) {
    const auto upTo = [&](int end) {  // the positions before `end`; a last block may pass 2^31
        const int n = (int)((uint32_t)end - (uint32_t)from);
        return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1;
    };
    uint32_t text = pos < 0 ? 0u : upTo(it.w.first);
    if (a.window) text &= ~upTo(max(pos - a.window + 1, 0)) | upTo(a.sinks);
    return near ? text | seenFrom(t, token, (int)((uint32_t)from - (uint32_t)it.w.first)) : text;
}

// ---- one row, key by key ----------------------------------------------------------------------------------------------

// One row by one wave: a lane has the scores of one key of 64, then four of the result's elements (lane + 64 e).  A value is only touched
// where the row sees its position, so what other positions hold, NaN and infinities among it, cannot come in: the tiles below multiply a
// masked value, or the scale of one, by a weight of zero, and hand a row here where that left a NaN.  (A select by the weight would drop
// the NaN of a position that the row sees with a weight too small for 32 bits.)  Adds the `count` (up to 64) positions from `from` on to o, m and l.
// q: D floats of LDS, the row's query.
template <bool PAGED, bool Q8, bool TREE>
__device__ __forceinline__ void attendRow(const AttentionArgs &a, const float *q, const Item &it, const Tree &tree, int token, int pos, int from, int count, float *o, float *m, float *l) {
    const CacheArgs &c = a.c;
    const int lane = threadIdx.x & 63, D = c.D;
    float most = *m, sum = *l;
    const int j = (int)((uint32_t)from + (uint32_t)lane);
    int row = -1;
    bool see = lane < count && sees(windowOf(a), sinksOf(a, pos), pos, j);
    if constexpr (TREE) {
        if (j >= it.w.first) see = lane < count && (seenFrom(tree, token, j - it.w.first) & 1);
    }
    if (see) row = keyRow(a, it, askKey<PAGED>(a, it, j, true));
    float s = -INFINITY, vs = 1.0f;
    if (row >= 0) {
        float dot = 0.0f;
        if constexpr (Q8) {
            const int8_t *k = (const int8_t *)a.key + (int64_t)row * D;
            for (int d = 0; d < D; d += 16) {
                const v4i w = *(const v4i *)(k + d);
#pragma unroll
                for (int i = 0; i < 16; i++) dot = fmaf((float)(int8_t)(w[i >> 2] >> (8 * (i & 3))), q[d + i], dot);
            }
            dot *= a.key_scales[row];
            vs = a.value_scales[row];
        } else {
            const uint16_t *k = (const uint16_t *)a.key + (int64_t)row * D;
            for (int d = 0; d < D; d += 8) {
                const v4i w = *(const v4i *)(k + d);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    dot = fmaf(__uint_as_float((uint32_t)w[i] << 16), q[d + 2 * i], dot);
                    dot = fmaf(__uint_as_float((uint32_t)w[i] & 0xffff0000u), q[d + 2 * i + 1], dot);
                }
            }
        }
        s = dot * (a.scale * kLog2e);
    }
    uint64_t seen = __ballot(row >= 0);
    if (seen == 0) return;
    float high = s;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) high = fmaxf(high, __shfl_xor(high, step));
    const float now = fmaxf(most, high), shift = now == -INFINITY ? 0.0f : now;
    const float down = exp2f(most - shift);  // most <= shift or -inf
    const float p = row >= 0 ? exp2f(s - shift) : 0.0f;
    float part = p;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) part += __shfl_xor(part, step);
    sum = sum * down + part;
    most = now;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] *= down;
    while (seen) {
        const int t = __builtin_ctzll(seen);
        seen &= seen - 1;
        const int64_t r = __builtin_amdgcn_readlane(row, t);
        const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), t));
        const float u = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), t));
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int d = lane + 64 * e;
            if (d >= D) continue;
            float v;
            if constexpr (Q8) v = (float)((const int8_t *)a.value)[r * D + d] * u;
            else v = __uint_as_float((uint32_t)((const uint16_t *)a.value)[r * D + d] << 16);
            o[e] = fmaf(w, v, o[e]);
        }
    }
    *m = most;
    *l = sum;
}

// A row of an item once more, key by key, and its result or partial result stored.  q: LDS of this wave, kMaxHeadDim floats.
template <bool TILE, bool PAGED, bool Q8, bool TREE>
__device__ __forceinline__ void redoRow(const AttentionArgs &a, const AttentionPlan &p, const Item &it, const Span &span, const Tree &tree, int r, float *q) {
    const int lane = threadIdx.x & 63, D = a.c.D;
    const int inSeq = (it.tile << p.rowsLog) + r, token = (int)fastDiv((uint32_t)inSeq, a.g), h = it.head * a.G + inSeq - token * a.G;
    const int64_t at = ((int64_t)(it.w.begin + token) * a.H + h) * D;
    for (int d = lane; d < D; d += 64) q[d] = __uint_as_float((uint32_t)a.query[at + d] << 16);
    __threadfence_block();
    float o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
    int pos = it.w.first + token;
    if constexpr (TREE) pos = positionOf(tree, token);
    for (int b = span.from; b < span.to; b++) {
        const int j = blockStart(p, span, b);
        attendRow<PAGED, Q8, TREE>(a, q, it, tree, token, pos, j, p.keys(), o, &m, &l);
        // Where no element is a number any more, nothing that follows makes it one.  (With no weight above 0 yet the result may still be zeros.)
        bool lost = l != 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) lost &= lane + 64 * e >= D || o[e] != o[e];
        if (__all(lost)) break;
    }
    if (it.slot < 0) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int d = lane + 64 * e;
            if (d < D) a.out[at + d] = bf16Bits(l == 0.0f ? 0.0f : o[e] / l);
        }
    } else {
        const auto slots = slotsOf(a, p);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int d = lane + 64 * e;
            const uint32_t to = TILE ? tileSums(a, it.slot) + (uint32_t)((((r >> 5) * (D >> 3) + (d >> 3)) * 64 + ((d >> 2) & 1) * 32 + (r & 31)) * 4 + (d & 3)) * 4u
                                     : slotRow(a, p, it.slot, r) + (uint32_t)d * 4u;
            if (d < D) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(o[e]), slots, (int)to, 0, kDeviceScope);
        }
        if (lane == 0) put4(slots, TILE ? tileStats(a, it.slot, r) : slotRow(a, p, it.slot, r) + D * 4, m, l, 0.0f, 0.0f);
    }
    __threadfence_block();
}

// ---- small helpers of the tiles ---------------------------------------------------------------------------------------

// What is left of x and y behind their bf16 in `word`, as bf16 again.
__device__ __forceinline__ int restOf(int word, float x, float y) {
    return packBf16(x - __uint_as_float((uint32_t)word << 16), y - __uint_as_float((uint32_t)word & 0xffff0000u));
}

// Four int8 as bf16, which holds them: the upper halves of their floats.
__device__ __forceinline__ v2i wholeBf16(int w) {
    const uint32_t f0 = __float_as_uint((float)(int8_t)w), f1 = __float_as_uint((float)(int8_t)(w >> 8));
    const uint32_t f2 = __float_as_uint((float)(int8_t)(w >> 16)), f3 = __float_as_uint((float)(w >> 24));
    return v2i{(int)__builtin_amdgcn_perm(f1, f0, 0x07060302u), (int)__builtin_amdgcn_perm(f3, f2, 0x07060302u)};
}
__device__ __forceinline__ v8bf wholeBf16x8(int lo, int hi) {
    const v2i a = wholeBf16(lo), b = wholeBf16(hi);
    return __builtin_bit_cast(v8bf, v4i{a[0], a[1], b[0], b[1]});
}

// Four rows of 16 elements, a lane's eight bytes of one of them: the lane gets a column (16 lanes a group).
__device__ __forceinline__ v2i turn16(const int8_t *p) {
    return __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)p));
}
// Eight rows of 16 bytes, likewise.
__device__ __forceinline__ v2i turn8(const int8_t *p) { return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i *)p); }

// Rows of keys and values in LDS are as long as a head; 16 of them at one 16-byte chunk, or 8 of them at four neighbouring ones, must not meet in the banks.
// The chunk of a row is stored at chunk ^ swizzle(row): the row's low two bits move it by whole groups of four chunks, the next two
// within a group.
template <int ROW_BYTES>
__device__ __forceinline__ int swizzle(int row) {
    if constexpr (ROW_BYTES >= 256) return ((row & 3) << 2) | ((row >> 2) & 3);
    else return ((row & 2) << 1) | ((row >> 2) & 3);  // 128 bytes: rows lie in both halves of the banks in turn
}

// The same for the streams' values.  int8 rows are shorter, and eight bytes of 32 rows are read at a time: a chunk of each.
template <int ROW_BYTES, bool Q8>
__device__ __forceinline__ int streamSwizzle(int row) {
    if constexpr (!Q8) return swizzle<ROW_BYTES>(row);
    else return ROW_BYTES >= 256 ? row & 15 : ROW_BYTES == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
}

// Address of chunk `c` ^ swizzle of a row, given that of chunk `own` ^ swizzle where c has none of own's bits set: of a chunk's number the low four bits are
// swizzled, and rows start at multiples of theirs, so that is one XOR with a constant.  `hold` keeps the compiler from making all of them before
// a loop, where they would take registers.
__device__ __forceinline__ int chunkAt(int base, int c) { return (base ^ ((c & 15) << 4)) + ((c >> 4) << 8); }
__device__ __forceinline__ int hold(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// What is taken off a row's scores is set this far (powers of two) above their maximum, so that all is scaled down only where a later one passes
// that.  Above, not at it: weights then never pass 1, and sums of finite values no further than the definition's.  (What has less than 2^-118 of the
// largest weight counts as nothing.)
constexpr float kSlack = 8.0f;

// ---- few rows: keys and values streamed -----------------------------------------------------------------------------------

// A tile of 16 rows (a token's heads, or a few tokens'); each of the four waves has blocks of 32 keys of its own, every fourth, and joins the
// others at the end.  A wave waits for nobody: its keys go straight into the matrix operand's registers, its values through LDS of its own.
// The registers are filled again as soon as their content is used, so a block's 2 x 32 rows are under way while the one before is worked on.
// Bound by memory where there is much to read (a token for each of 16 sequences of up to 32768 positions, 32 heads of 128 over 8, int8, 770 MB: 152 us,
// 5.1 TB/s, what a large copy reaches), else by a chain of loads: starts, table, keys, and what the parts wrote (1024 positions of one head
// of 256: 10 us, of which 2 are the join).
template <int DT, bool EXACT, bool PAGED, bool Q8, bool TREE>
__device__ __forceinline__ void streamItem(const AttentionArgs &a, const AttentionPlan &p, const Item &it) {
    constexpr int KB = 32, STEPS = DT / 32, ROW = DT * (Q8 ? 1 : 2), LOADS = ROW / 64;  // LOADS: 16-byte pieces of a row that one of four lanes has
    constexpr int JOIN = 16 * (DT + 4);  // floats of a wave's result
    extern __shared__ __attribute__((aligned(16))) int8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = lane >> 4, col = lane & 15;
    const CacheArgs &c = a.c;
    const Span span = spanOf<TREE>(a, p, it);
    const int D = c.D, r0 = it.tile * 16;
    const int top = it.w.first + (int)fastDiv((uint32_t)r0, a.g), bottom = it.w.first + (int)fastDiv((uint32_t)(r0 + span.rows - 1), a.g);
    const int inSeq = r0 + min(col, span.rows - 1), token = (int)fastDiv((uint32_t)inSeq, a.g);
    int pos = it.w.first + token;
    float *const scales = (float *)(smem + 4 * KB * ROW) + wave * 2 * KB;

    // Loads are never skipped: a position that is not there is read as row 0, its value taken for zeros and its score for minus infinity; behind D
    // (not EXACT) a piece is the first one, against zeros of the query.
    int row0, row1;      // of the block to be fetched next: keys col and 16 + col
    bool there0, there1; // of the block in the registers
    KeyAsk<PAGED> asked0, asked1;  // of the block behind that
    v4i kreg[2][LOADS], vreg[2][LOADS];
    float sreg = 0.0f;
    auto ask = [&](int b) {
        const int j = blockStart(p, span, b) + col;
        asked0 = askKey<PAGED>(a, it, j, b < span.to);
        asked1 = askKey<PAGED>(a, it, j + 16, b < span.to);
    };
    auto resolve = [&]() {
        row0 = keyRow(a, it, asked0);
        row1 = keyRow(a, it, asked1);
    };
    constexpr int ELEMS = Q8 ? 16 : 8, SIZE = Q8 ? 1 : 2;  // elements of a piece, bytes of an element
    auto fetch = [&](const void *from, v4i(&reg)[2][LOADS]) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int8_t *const at = (const int8_t *)from + ((int64_t)max(k ? row1 : row0, 0) * D + (EXACT ? quarter * ELEMS : 0)) * SIZE;
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const int d = (4 * i + quarter) * ELEMS;
                reg[k][i] = *(const v4i *)(at + (EXACT ? 64 * i : d < D ? d * SIZE : 0));
            }
        }
    };
    ask(span.from + wave);
    auto fetchScales = [&]() {
        if constexpr (Q8) sreg = (lane < 32 ? a.key_scales : a.value_scales)[max((lane & 16) ? row1 : row0, 0)];
    };

    v8bf q[STEPS];
    {
        const int64_t at = ((int64_t)(it.w.begin + token) * a.H + it.head * a.G + inSeq - token * a.G) * D;
#pragma unroll
        for (int t = 0; t < STEPS; t++) {
            // of an int8 row a lane has 16 elements at a time, for two steps
            const int d = Q8 ? 64 * (t >> 1) + 16 * quarter + 8 * (t & 1) : 32 * t + 8 * quarter;
            v4i w = *(const v4i *)(a.query + at + (EXACT || d < D ? d : 0));
            if (!EXACT && d >= D) w = v4i{0, 0, 0, 0};
            q[t] = __builtin_bit_cast(v8bf, w);
        }
    }
    v4f o[DT / 16];
#pragma unroll
    for (int t = 0; t < DT / 16; t++) o[t] = v4f{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    const float scale = a.scale * kLog2e;
    resolve();
    ask(span.from + wave + 4);
    there0 = row0 >= 0;
    there1 = row1 >= 0;
    fetchScales();
    fetch(a.value, vreg);
    fetch(a.key, kreg);
    Tree tree{};
    if constexpr (TREE) {
        tree = plantTree(a, it, smem, r0, span.rows, span.to > span.from && blockStart(p, span, span.to - 1) > it.w.first - KB);  // a block may end at 2^31
        pos = positionOf(tree, token);
    }
    for (int b = span.from + wave; b < span.to; b += 4) {
        const int j0 = blockStart(p, span, b);
        resolve();
        ask(b + 8);
        const uint64_t gone0 = __ballot(!there0), gone1 = __ballot(!there1);
        if (gone0 | gone1) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                if (!there0) vreg[0][i] = v4i{0, 0, 0, 0};
                if (!there1) vreg[1][i] = v4i{0, 0, 0, 0};
            }
        }
        __builtin_amdgcn_wave_barrier();
        const int storeAt = hold(wave * KB * ROW + col * ROW + ((quarter ^ streamSwizzle<ROW, Q8>(col)) << 4));
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            *(v4i *)(smem + chunkAt(storeAt, 4 * i)) = vreg[0][i];
            *(v4i *)(smem + chunkAt(storeAt, 4 * i) + 16 * ROW) = vreg[1][i];
        }
        if constexpr (Q8) scales[lane] = ((lane & 16) ? there1 : there0) ? sreg : 0.0f;  // here, where the load has come back
        __builtin_amdgcn_wave_barrier();
        const bool now0 = row0 >= 0, now1 = row1 >= 0;
        fetchScales();
        fetch(a.value, vreg);
        v4f s[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            s[k] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < STEPS; t++) {
                v8bf kw;
                if constexpr (Q8) kw = (t & 1) ? wholeBf16x8(kreg[k][t >> 1][2], kreg[k][t >> 1][3]) : wholeBf16x8(kreg[k][t >> 1][0], kreg[k][t >> 1][1]);
                else kw = __builtin_bit_cast(v8bf, kreg[k][t]);
                s[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kw, q[t], s[k], 0, 0, 0);
            }
        }
        fetch(a.key, kreg);
        there0 = now0;
        there1 = now1;
        if constexpr (Q8) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const v4f u = *(const v4f *)(scales + 16 * k + 4 * quarter);
#pragma unroll
                for (int i = 0; i < 4; i++) s[k][i] *= u[i];
            }
        }
        const bool whole = (TREE ? tree.all && j0 <= it.w.first - KB : j0 + KB - 1 <= top) && (a.window == 0 || (TREE ? min(bottom, tree.bottom) : bottom) - j0 < a.window || j0 + KB <= a.sinks);
        if (!whole || (gone0 | gone1)) {
            const uint32_t window = windowOf(a);
            const int sinks = sinksOf(a, pos);
            uint32_t seen = 0;  // of the 32 keys from j0 + 4 quarter on
            if constexpr (TREE) seen = seenBits(a, tree, it, token, pos, j0 + 4 * quarter, j0 > it.w.first - KB);
#pragma unroll
            for (int k = 0; k < 2; k++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int key = 4 * quarter + i, j = j0 + 16 * k + key;
                    bool see = sees(window, sinks, pos, j) & !(((k ? gone1 : gone0) >> key) & 1);
                    if constexpr (TREE) see = ((seen >> (16 * k + i)) & 1) & !(((k ? gone1 : gone0) >> key) & 1);
                    s[k][i] = see ? s[k][i] : -INFINITY;
                }
            }
        }
        float high = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        high = maxOverQuarters(high) * scale;
        if (__any(high > m)) {
            const float now = high > m ? high + kSlack : m, down = __builtin_amdgcn_exp2f(m - (now == -INFINITY ? 0.0f : now));
            m = now;
            l *= down;
#pragma unroll
            for (int t = 0; t < DT / 16; t++) o[t] *= down;
        }
        const float shift = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int k = 0; k < 2; k++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[k][i] = __builtin_amdgcn_exp2f(fmaf(s[k][i], scale, -shift));
                l += s[k][i];
            }
        }
        if constexpr (Q8) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const v4f u = *(const v4f *)(scales + 32 + 16 * k + 4 * quarter);
#pragma unroll
                for (int i = 0; i < 4; i++) s[k][i] *= u[i];
            }
        }
        // in two parts, what the first leaves being the second: the matrix units have the time
        v4i high4, low4;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float x = s[i >> 1][2 * (i & 1)], y = s[i >> 1][2 * (i & 1) + 1];
            high4[i] = packBf16(x, y);
            low4[i] = restOf(high4[i], x, y);
        }
        const v8bf weights = __builtin_bit_cast(v8bf, high4), rest = __builtin_bit_cast(v8bf, low4);
        // a lane's part of V: of four rows (quarter) and the four 16 on, eight bytes at a time; of eight rows at once where they are int8
        const int valueRow = Q8 ? 4 * quarter + ((col >> 1) & 3) + 16 * (col >> 3) : 4 * quarter + (col >> 2);
        const int valueAt = hold(wave * KB * ROW + valueRow * ROW + (((Q8 ? 0 : (col & 3) >> 1) ^ streamSwizzle<ROW, Q8>(valueRow)) << 4) + 8 * (col & 1));
#pragma unroll
        for (int t = 0; t < DT / 16; t++) {
            v8bf vw;
            if constexpr (Q8) {
                const v2i w = turn8(smem + chunkAt(valueAt, t));
                vw = wholeBf16x8(w[0], w[1]);
            } else {
                const v2i v0 = turn16(smem + chunkAt(valueAt, 2 * t)), v1 = turn16(smem + chunkAt(valueAt, 2 * t) + 16 * ROW);
                vw = __builtin_bit_cast(v8bf, v4i{v0[0], v0[1], v1[0], v1[1]});
            }
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vw, weights, o[t], 0, 0, 0);
            o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vw, rest, o[t], 0, 0, 0);
        }
    }
    l = sumOverQuarters(l);
    __syncthreads();
    // [wave][row][D + 4]: sums, maximum, sum of weights
    float *const join = (float *)smem;
#pragma unroll
    for (int t = 0; t < DT / 16; t++) *(v4f *)(join + wave * JOIN + col * (DT + 4) + 16 * t + 4 * quarter) = o[t];
    if (quarter == 0) {
        join[wave * JOIN + col * (DT + 4) + DT] = m;
        join[wave * JOIN + col * (DT + 4) + DT + 1] = l;
    }
    __syncthreads();
    const int r = tid >> 4;  // 16 threads a row
    float most = -INFINITY, factor[4], total = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) most = fmaxf(most, join[w * JOIN + r * (DT + 4) + DT]);
#pragma unroll
    for (int w = 0; w < 4; w++) {
        factor[w] = __builtin_amdgcn_exp2f(join[w * JOIN + r * (DT + 4) + DT] - (most == -INFINITY ? 0.0f : most));
        total += factor[w] * join[w * JOIN + r * (DT + 4) + DT + 1];
    }
    v4f sum[DT / 64];
    bool odd = false;
#pragma unroll
    for (int e = 0; e < DT / 64; e++) {
        sum[e] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; w++) sum[e] += factor[w] * *(const v4f *)(join + w * JOIN + r * (DT + 4) + 64 * e + 4 * col);
#pragma unroll
        for (int i = 0; i < 4; i++) odd |= sum[e][i] != sum[e][i];
    }
    // the rows of this wave that have a NaN: 4 wave .. 4 wave + 3, 16 lanes each
    const uint64_t odds = __ballot(odd);
    if (r < span.rows && !((odds >> (16 * (r & 3))) & 0xffff)) {
        const int mine = r0 + r, tok = (int)fastDiv((uint32_t)mine, a.g);
        if (it.slot < 0) {
            const float by = total == 0.0f ? 0.0f : 1.0f / total;
            uint16_t *out = a.out + ((int64_t)(it.w.begin + tok) * a.H + it.head * a.G + mine - tok * a.G) * D;
#pragma unroll
            for (int e = 0; e < DT / 64; e++) {
                if (64 * e + 4 * col < D) *(v2i *)(out + 64 * e + 4 * col) = v2i{packBf16(sum[e][0] * by, sum[e][1] * by), packBf16(sum[e][2] * by, sum[e][3] * by)};
            }
        } else {
            const auto slots = slotsOf(a, p);
            const uint32_t to = slotRow(a, p, it.slot, r);
#pragma unroll
            for (int e = 0; e < DT / 64; e++) {
                if (64 * e + 4 * col < D) put4(slots, to + (64 * e + 4 * col) * 4, sum[e][0], sum[e][1], sum[e][2], sum[e][3]);
            }
            if (col == 0) put4(slots, to + D * 4, most, total, 0.0f, 0.0f);
        }
    }
    __syncthreads();
    for (int k = 0; k < 4; k++) {
        if (__builtin_expect(((odds >> (16 * k)) & 0xffff) && 4 * wave + k < span.rows, 0)) redoRow<false, PAGED, Q8, TREE>(a, p, it, span, tree, 4 * wave + k, (float *)smem + wave * kMaxHeadDim);
    }
    if (it.slot >= 0) {
        __syncthreads();
        joinParts<16, 64, TREE && DT == 256 ? 4 : 1>(a, p, it, span.rows, (float *)smem + 4 * kMaxHeadDim);
    }
}

// ---- tiles of 128 rows ------------------------------------------------------------------------------------------------

// Waves of a SIMD: so many that what a wave keeps over the loop has its registers (int8 on the way to bf16 among it).  In memory a register would be
// waited for with all that is under way.
template <int DT, bool Q8>
constexpr int kTileWaves = DT == 256 ? Q8 ? 1 : 2 : 3;

// Four waves of 32 rows each; keys and values of a block in LDS, two buffers in turn, one barrier a block.  The next block is on its way while
// one is worked on, and the pages of the block behind that are asked for.  A wave's keys and values feed one product each from LDS, which gives
// just what the matrix units take; 64 rows a wave halve that, but leave two waves a SIMD where three hide each other's softmax (8192 tokens,
// 32 heads of 128, a window of 1024: 230 us where 32 rows took 195).  Blocks are as long as three workgroups a CU allow: 32 keys, 64 with heads of 64
// (64 with heads of 128: 214 us for 195).
//
// Bound by the waits of a wave for itself (products, the softmax of their results, products) and by vector instructions next to matrix ones: that
// prompt takes 159 us, 810 TFLOP/s; four chunks of up to 512 tokens over up to 8192 positions 169, 730.  Heads of 256 leave two waves a SIMD and LDS busy with the
// blocks that come (six prompts of up to 2048 tokens: 99 us, 380 TFLOP/s, where the longest tile's blocks alone take nearly all of it).
template <int DT, bool PAGED, bool Q8, bool FINE, bool TREE>
__device__ __forceinline__ void tileItem(const AttentionArgs &a, const AttentionPlan &p) {
    constexpr int KB = DT >= 128 ? 32 : 64, CH = DT / 8, PER = KB * CH / 256, STEP = 256 / CH, ROW = DT * 2;
    extern __shared__ __attribute__((aligned(16))) int8_t smem[];
    float *const scaleRoom = (float *)(smem + 4 * KB * ROW);       // [2][keys, values][KB]
    uint8_t *const flagRoom = (uint8_t *)(scaleRoom + 4 * KB);      // [2][4 waves]: some position of the block has no page
    uint8_t *const absentRoom = flagRoom + 16;                       // [2][KB]: the position has no row
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, col = lane & 31;
    const CacheArgs &c = a.c;
    Item it;
    if (!findItem(a, p, blockIdx.x, &it, smem)) return;
    // single tokens among prompts: a tile would have one wave at work, and that for one row of 32 in its products
    if constexpr (PAGED && DT <= 128) {
        if (goesByStream(a, it.w.count)) {
            AttentionPlan stream = p;
            stream.keysLog = 5;
            it.part <<= p.keysLog - 5;
            return streamItem<DT, false, PAGED, Q8, TREE>(a, stream, it);
        }
    }
    const Span span = spanOf<TREE>(a, p, it);
    const int D = c.D, r0 = it.tile * 128 + wave * 32, rowsHere = min(32, span.rows - wave * 32);  // of this wave; none: <= 0
    const bool active = rowsHere > 0;
    const int top = it.w.first + (int)fastDiv((uint32_t)r0, a.g), bottom = it.w.first + (int)fastDiv((uint32_t)(r0 + max(rowsHere, 1) - 1), a.g);
    // where this lane's row lies; made twice, not kept over the loop
    auto rowAt = [&](int column) {
        const int inSeq = r0 + min(column, max(rowsHere, 1) - 1), token = (int)fastDiv((uint32_t)inSeq, a.g);
        return ((int64_t)(it.w.begin + min(token, it.w.count - 1)) * a.H + it.head * a.G + inSeq - token * a.G) * D;
    };
    const int token = (int)fastDiv((uint32_t)(r0 + min(col, max(rowsHere, 1) - 1)), a.g);
    int pos = it.w.first + token;

    v16f o[DT / 32];
#pragma unroll
    for (int t = 0; t < DT / 32; t++) o[t] = v16f{0};
    float m = -INFINITY, l = 0.0f;
    const float scale = a.scale * kLog2e;

    // this thread's part of a block: chunk `piece` of rows tid / CH + STEP i.  Loads are never skipped: a position that is not there is read
    // as row 0, and the value taken for zeros, its score for minus infinity; behind D a piece is the first one, against zeros of the query.
    const int piece = tid % CH, myRow = tid / CH, pieceAt = piece * 8 < D ? piece * 8 : 0;
    uint32_t gone = 0;  // rows of the block last sent for that are not there, a bit each
    bool unpaged = false;  // some of them, or of those that were fetched, are the sequence's, but have no page
    // bf16: straight into LDS, a wave's 64 pieces of 16 bytes one behind the other, so that a lane's place is given and it takes the
    // piece that belongs there
    const unsigned lds = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) int8_t *)smem) + wave * 1024;
    // Where the rows that one load of a wave brings (64 / CH, at most 8) lie behind one another, their place is a scalar's, and a lane's among them stays the
    // same; in pages of a multiple of 8 positions they do.  Else, and in a block that is not whole, each lane looks its rows up.
    constexpr int TURNS = DT == 256 ? 2 : 1;  // STEP rows on, the swizzle is another one (rows eight apart)
    const int waveRow = wave * (64 / CH);
    const int64_t rowElems = PAGED ? D : (int64_t)c.KVH * D;  // from one position to the next
    const bool together = PAGED ? c.PS % 8 == 0 : rowElems < 1 << 24;
    auto pieceOf = [&](int i) {
        const int mine = piece ^ swizzle<ROW>(myRow + STEP * i);
        return mine * 8 < D ? mine * 8 : 0;
    };
    uint32_t laneOff[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; i++) laneOff[i] = ((uint32_t)(myRow - waveRow) * (uint32_t)rowElems + (uint32_t)pieceOf(i)) * 2;
    uint32_t pages[PER];
    // the pages are asked for a block ahead; by scalar loads, which do not come back in order with the others
    auto askPages = [&](int b) {
        if constexpr (PAGED) {
            const int j0 = blockStart(p, span, max(min(b, span.to - 1), 0));
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const uint32_t at = (uint32_t)max(min(j0 + STEP * i + waveRow, c.capacity - 1), 0);
                pages[i] = ((const __attribute__((address_space(4))) uint32_t *)(uintptr_t)c.pages)[(int64_t)it.seq * c.P + fastDiv(at, c.ps)];
            }
        }
    };
    auto send = [&](int stage, int b) {
        const int j0 = blockStart(p, span, b);
        const unsigned to = lds + stage * 2 * KB * ROW;
        bool whole = together && b < span.to && j0 <= it.w.length - KB;
        if constexpr (PAGED) {
#pragma unroll
            for (int i = 0; i < PER; i++) whole = whole & (pages[i] < (uint32_t)c.NP);
        }
        gone = 0;
        unpaged = false;
        if (whole) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const uint32_t at = (uint32_t)(j0 + STEP * i + waveRow);
                uint32_t first;
                if constexpr (PAGED) first = (pages[i] * (uint32_t)c.KVH + (uint32_t)it.head) * (uint32_t)c.PS + (at - fastDiv(at, c.ps) * c.ps.d);
                else first = (at + (uint32_t)it.w.begin) * (uint32_t)c.KVH + (uint32_t)it.head;
                const uint64_t from = (uint64_t)first * ((uint32_t)D * 2u);
                dmaLoad16((const int8_t *)a.key + from, laneOff[i % TURNS], to + i * 4096);
                dmaLoad16((const int8_t *)a.value + from, laneOff[i % TURNS], to + KB * ROW + i * 4096);
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const KeyAsk<PAGED> asking = askKey<PAGED>(a, it, j0 + myRow + STEP * i, b < span.to);
                const int row = keyRow(a, it, asking);
                gone |= row < 0 ? 1u << i : 0u;
                if constexpr (PAGED) unpaged |= asking.page.in & (row < 0);
                const int64_t from = ((int64_t)max(row, 0) * D + pieceOf(i)) * 2;
                dmaLoad16((const int8_t *)a.key + from, to + i * 4096);
                dmaLoad16((const int8_t *)a.value + from, to + KB * ROW + i * 4096);
            }
        }
    };
    // int8: a thread has 16 elements of rows qRow + Q_STEP i, which become two chunks
    constexpr int Q_CH = DT / 16, Q_PER = KB * Q_CH / 256, Q_STEP = 256 / Q_CH;
    const int qPiece = tid % Q_CH, qRow = tid / Q_CH, qPieceAt = qPiece * 16 < D ? qPiece * 16 : 0;
    auto flag = [&](int stage) {
        const bool some = __any(unpaged);
        if (lane == 0) flagRoom[stage * 4 + wave] = some;
        if ((Q8 ? qPiece : piece) == 0) {
#pragma unroll
            for (int i = 0; i < (Q8 ? Q_PER : PER); i++) absentRoom[stage * KB + (Q8 ? qRow + Q_STEP * i : myRow + STEP * i)] = (gone >> i) & 1;
        }
    };
    auto arrive = [&](int stage) {
        waitVmcnt<0>();
        if (__any(gone != 0)) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if ((gone >> i) & 1) *(v4i *)(smem + stage * 2 * KB * ROW + KB * ROW + i * 4096 + tid * 16) = v4i{0, 0, 0, 0};
            }
        }
        if constexpr (PAGED) flag(stage);
    };
    // int8: through registers, where they become bf16, every lane's rows looked up a block ahead (23 single tokens and a prompt's 777 in one batch, 16 heads of
    // 64 over 4, windows of 2048: 35 us)
    int rows[Q_PER], scaleRow = -1;
    KeyAsk<PAGED> asked[Q_PER], scaleAsked;
    v4i kreg[Q_PER], vreg[Q_PER];
    float sreg = 0.0f;
    bool scaleGone = false;  // of sreg's position
    bool holes = false;  // unpaged, of the rows that were looked up
    auto ask = [&](int b) {
        const int j0 = blockStart(p, span, b);
#pragma unroll
        for (int i = 0; i < Q_PER; i++) asked[i] = askKey<PAGED>(a, it, j0 + qRow + Q_STEP * i, b < span.to);
        if constexpr (Q8) scaleAsked = askKey<PAGED>(a, it, j0 + (tid & (KB - 1)), b < span.to);
    };
    auto resolve = [&]() {
        holes = false;
#pragma unroll
        for (int i = 0; i < Q_PER; i++) {
            rows[i] = keyRow(a, it, asked[i]);
            if constexpr (PAGED) holes |= asked[i].page.in & (rows[i] < 0);
        }
        if constexpr (Q8) scaleRow = keyRow(a, it, scaleAsked);
    };
    auto fetch = [&]() {
        gone = 0;
        unpaged = holes;
#pragma unroll
        for (int i = 0; i < Q_PER; i++) {
            gone |= rows[i] < 0 ? 1u << i : 0u;
            const int64_t from = (int64_t)max(rows[i], 0) * D + qPieceAt;
            kreg[i] = *(const v4i *)((const int8_t *)a.key + from);
            vreg[i] = *(const v4i *)((const int8_t *)a.value + from);
        }
        sreg = (tid & KB ? a.value_scales : a.key_scales)[max(scaleRow, 0)];
        scaleGone = scaleRow < 0;
    };
    auto put = [&](int stage) {
        int8_t *const keys = smem + stage * 2 * KB * ROW, *const values = keys + KB * ROW;
#pragma unroll
        for (int i = 0; i < Q_PER; i++) {
            const int row = qRow + Q_STEP * i;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int where = row * ROW + (((2 * qPiece + c) ^ swizzle<ROW>(row)) << 4);
                *(v8bf *)(keys + where) = wholeBf16x8(kreg[i][2 * c], kreg[i][2 * c + 1]);
                *(v8bf *)(values + where) = wholeBf16x8(vreg[i][2 * c], vreg[i][2 * c + 1]);
            }
        }
        if (tid < 2 * KB) scaleRoom[stage * 2 * KB + tid] = scaleGone ? 0.0f : sreg;
        flag(stage);
    };

    if constexpr (Q8) {
        ask(span.from);
        resolve();
        ask(span.from + 1);
        fetch();
    } else {
        askPages(span.from);
        send(0, span.from);
        askPages(span.from + 1);
    }
    v8bf q[DT / 16];
    const int64_t at = rowAt(col);
#pragma unroll
    for (int t = 0; t < DT / 16; t++) {
        v4i w = *(const v4i *)(a.query + at + (16 * t < D ? 16 * t : 0) + 8 * half);
        if (16 * t >= D) w = v4i{0, 0, 0, 0};
        q[t] = __builtin_bit_cast(v8bf, w);
    }
    Tree tree{};
    if constexpr (TREE) {
        tree = plantTree(a, it, smem, it.tile * 128, span.rows, span.to > span.from && blockStart(p, span, span.to - 1) > it.w.first - KB);
        pos = positionOf(tree, min(token, tree.token0 + (int)fastDiv((uint32_t)(it.tile * 128 + span.rows - 1), a.g) - tree.token0));
    }
    for (int b = span.from, stage = 0; b < span.to; b++, stage ^= 1) {
        if constexpr (Q8) {
            resolve();
            ask(b + 2);
            put(stage);
            fetch();
            __syncthreads();
        } else {
            arrive(stage);
            __syncthreads();  // and everybody is done with the other buffer
            send(stage ^ 1, b + 1);
            askPages(b + 2);
        }
        const int j0 = blockStart(p, span, b);
        if (!active || j0 > bottom) continue;
        const int keyAt = hold(stage * 2 * KB * ROW + col * ROW + ((half ^ swizzle<ROW>(col)) << 4));
        v16f s[KB / 32];
#pragma unroll
        for (int k = 0; k < KB / 32; k++) s[k] = v16f{0};
#pragma unroll
        for (int t = 0; t < DT / 16; t++) {
#pragma unroll
            for (int k = 0; k < KB / 32; k++) {
                const v8bf kw = *(const v8bf *)(smem + chunkAt(keyAt, 2 * t) + k * 32 * ROW);
                s[k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kw, q[t], s[k], 0, 0, 0);
            }
        }
        // reads of LDS run ahead of the products that take them by AHEAD; left alone each is waited for
        constexpr int PRODUCTS = DT / 16 * (KB / 32), AHEAD = 4;
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
        for (int i = 0; i < PRODUCTS - AHEAD; i++) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, AHEAD, 0);
        if constexpr (Q8) {
#pragma unroll
            for (int k = 0; k < KB / 32; k++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const v4f u = *(const v4f *)(scaleRoom + stage * 2 * KB + k * 32 + 8 * i + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; e++) s[k][4 * i + e] *= u[e];
                }
            }
        }
        bool whole = (TREE ? tree.all && j0 <= it.w.first - KB : j0 + KB - 1 <= top) && j0 <= it.w.length - KB && (a.window == 0 || (TREE ? min(bottom, tree.bottom) : bottom) - j0 < a.window || j0 + KB <= a.sinks);
        bool gaps = false;
        if constexpr (PAGED) gaps = __builtin_amdgcn_readfirstlane(*(const int *)(flagRoom + stage * 4)) != 0;
        if (!whole || gaps) {
            const int at = hold(pos), sinks = sinksOf(a, at);
            const uint32_t window = windowOf(a);
#pragma unroll
            for (int k = 0; k < KB / 32; k++) {
                uint32_t seen = 0;  // of the 32 keys from j0 + 32 k + 4 half on
                if constexpr (TREE) seen = seenBits(a, tree, it, token, at, j0 + 32 * k + 4 * half, j0 > it.w.first - KB);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int j = j0 + k * 32 + 8 * i + 4 * half;
                    uint32_t missing = 0;  // a byte a position
                    if constexpr (PAGED) missing = *(const uint32_t *)(absentRoom + stage * KB + k * 32 + 8 * i + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool there = PAGED ? !(missing & (0xffu << (8 * e))) : j + e < it.w.length;
                        bool see = sees(window, sinks, at, j + e);
                        if constexpr (TREE) see = (seen >> (8 * i + e)) & 1;
                        s[k][4 * i + e] = (see & there) ? s[k][4 * i + e] : -INFINITY;
                    }
                }
            }
        }
        float high = s[0][0];
#pragma unroll
        for (int k = 0; k < KB / 32; k++) {
#pragma unroll
            for (int i = 0; i < 16; i++) high = fmaxf(high, s[k][i]);
        }
        high = maxOverHalves(high) * scale;
        if (__any(high > m)) {
            const float now = high > m ? high + kSlack : m, down = __builtin_amdgcn_exp2f(m - (now == -INFINITY ? 0.0f : now));
            m = now;
            l *= down;
#pragma unroll
            for (int t = 0; t < DT / 32; t++) {
#pragma unroll
                for (int i = 0; i < 16; i++) o[t][i] *= down;
            }
        }
        const float shift = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int k = 0; k < KB / 32; k++) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                s[k][i] = __builtin_amdgcn_exp2f(fmaf(s[k][i], scale, -shift));
                l += s[k][i];
            }
        }
        if constexpr (Q8) {
#pragma unroll
            for (int k = 0; k < KB / 32; k++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const v4f u = *(const v4f *)(scaleRoom + stage * 2 * KB + KB + k * 32 + 8 * i + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; e++) s[k][4 * i + e] *= u[e];
                }
            }
        }
        const int valueRow = 4 * half + ((lane & 15) >> 2);
        const int valueAt = hold((stage * 2 + 1) * KB * ROW + valueRow * ROW + (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ swizzle<ROW>(valueRow)) << 4) + (lane & 1) * 8);
#pragma unroll
        for (int k = 0; k < KB / 32; k++) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                v4i w;
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = packBf16(s[k][8 * x + 2 * e], s[k][8 * x + 2 * e + 1]);
                const v8bf weights = __builtin_bit_cast(v8bf, w);
                v4i left{0, 0, 0, 0};
                if constexpr (FINE) {
#pragma unroll
                    for (int e = 0; e < 4; e++) left[e] = restOf(w[e], s[k][8 * x + 2 * e], s[k][8 * x + 2 * e + 1]);
                }
                const v8bf rest = __builtin_bit_cast(v8bf, left);
#pragma unroll
                for (int t = 0; t < DT / 32; t++) {
                    // the rows eight on are swizzled by two chunks more
                    const v2i v0 = turn16(smem + chunkAt(valueAt, 4 * t) + (k * 32 + 16 * x) * ROW);
                    const v2i v1 = turn16(smem + chunkAt(valueAt, (4 * t) ^ 2) + (k * 32 + 16 * x + 8) * ROW);
                    const v8bf vw = __builtin_bit_cast(v8bf, v4i{v0[0], v0[1], v1[0], v1[1]});
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vw, weights, o[t], 0, 0, 0);
                    if constexpr (FINE) o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vw, rest, o[t], 0, 0, 0);
                }
            }
        }
    }
    waitVmcnt<0>();  // the block behind the last one
    __syncthreads();
    l = sumOverHalves(l);
    // a masked value that was no number, or a row that sees one
    bool odd = false;
#pragma unroll
    for (int t = 0; t < DT / 32; t++) {
#pragma unroll
        for (int i = 0; i < 16; i++) odd |= o[t][i] != o[t][i];
    }
    const uint64_t odds = __ballot(odd);
    const uint32_t again = (uint32_t)odds | (uint32_t)(odds >> 32);
    int8_t *const room = smem + wave * 32 * ROW;  // of this wave
    if (it.slot < 0) {
        // by way of LDS, so that what is written lies in whole rows
        const float by = l == 0.0f ? 0.0f : 1.0f / l;
        const int at = col * ROW + half * 8, turn = (col & 7) << 4;
#pragma unroll
        for (int t = 0; t < DT / 32; t++) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                *(v2i *)(room + at + (((4 * t + i) << 4) ^ turn)) = v2i{packBf16(o[t][4 * i] * by, o[t][4 * i + 1] * by), packBf16(o[t][4 * i + 2] * by, o[t][4 * i + 3] * by)};
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < CH / 2; i++) {
            const int r = (64 / CH) * i + lane / CH;
            const v4i w = *(const v4i *)(room + r * ROW + (((lane % CH) ^ (r & 7)) << 4));
            if (r < rowsHere && !((again >> r) & 1) && (lane % CH) * 8 < D) *(v4i *)(a.out + rowAt(r) + (lane % CH) * 8) = w;
        }
        __builtin_amdgcn_wave_barrier();
    } else if (col < rowsHere && !((again >> col) & 1)) {
        const auto slots = slotsOf(a, p);
        const uint32_t to = tileSums(a, it.slot) + (uint32_t)(wave * (D >> 3) * 64 + lane) * 16u;
#pragma unroll
        for (int t = 0; t < DT / 32; t++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (32 * t + 8 * i < D) put4(slots, to + (4 * t + i) * 1024, o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]);
            }
        }
        if (half == 0) put4(slots, tileStats(a, it.slot, wave * 32 + col), m, l, 0.0f, 0.0f);
    }
    for (int r = 0; r < rowsHere; r++) {
        if (__builtin_expect((again >> r) & 1, 0)) redoRow<true, PAGED, Q8, TREE>(a, p, it, span, tree, wave * 32 + r, (float *)room);
    }
    if (it.slot >= 0) joinParts<128, 16, 4>(a, p, it, span.rows, (float *)smem + 4 * kMaxHeadDim);
}

// What a plan has for trees is known to the other kernels when they are compiled: a call of few us waits for each instruction more.
__device__ __forceinline__ void withoutTrees(AttentionArgs *a, AttentionPlan *p) { a->tree_rows = p->manyBlocks = p->shortRun = 0; }

template <int DT, bool PAGED, bool Q8, bool FINE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kTileWaves<DT, Q8>, kTileWaves<DT, Q8>)))
void attention_tiles(AttentionArgs a, AttentionPlan p) {
    withoutTrees(&a, &p);
    tileItem<DT, PAGED, Q8, FINE, false>(a, p);
}

template <int DT, bool Q8, bool FINE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kTileWaves<DT, Q8>, kTileWaves<DT, Q8>)))
void tree_attention_tiles(AttentionArgs a, AttentionPlan p) {
    tileItem<DT, true, Q8, FINE, true>(a, p);
}

template <int DT, bool EXACT, bool PAGED, bool Q8>
__global__ __launch_bounds__(256, DT == 256 && !Q8 ? 1 : 2) void attention_stream(AttentionArgs a, AttentionPlan p) {
    extern __shared__ __attribute__((aligned(16))) int8_t smem[];
    Item it;
    withoutTrees(&a, &p);
    if (findItem(a, p, blockIdx.x, &it, smem)) streamItem<DT, EXACT, PAGED, Q8, false>(a, p, it);
}

template <int DT, bool EXACT, bool Q8>
__global__ __launch_bounds__(256, DT == 256 && !Q8 ? 1 : 2) void tree_attention_stream(AttentionArgs a, AttentionPlan p) {
    extern __shared__ __attribute__((aligned(16))) int8_t smem[];
    Item it;
    if (findItem(a, p, blockIdx.x, &it, smem)) streamItem<DT, EXACT, true, Q8, true>(a, p, it);
}

// ---- launches -------------------------------------------------------------------------------------------------------------

static hipError_t checkAttention(const AttentionArgs &a) {
    const CacheArgs &c = a.c;
    if (c.T < 1 || c.S < 1 || c.KVH < 1 || c.D < 16 || c.D > kMaxHeadDim || c.D % 16 != 0 || a.G < 1 || a.H != a.G * c.KVH) return hipErrorInvalidValue;
    if ((int64_t)c.T * a.H >= (1LL << 31) || a.window < 0 || a.sinks < 0) return hipErrorInvalidValue;
    if (!c.starts || !a.query || !a.out || !a.key || !a.value || !c.lengths != !c.pages || !a.key_scales != !a.value_scales) return hipErrorInvalidValue;
    if (((uintptr_t)a.query | (uintptr_t)a.out | (uintptr_t)a.key | (uintptr_t)a.value | (uintptr_t)a.work) & 15) return hipErrorInvalidValue;
    if (c.pages) {
        if (c.P < 1 || c.NP < 1 || c.PS < 1 || (int64_t)c.P * c.PS != c.capacity || (int64_t)c.NP * c.KVH * c.PS >= (1LL << 31)) return hipErrorInvalidValue;
    } else if (a.key_scales) {
        return hipErrorInvalidValue;
    }
    if (a.parents && (!c.pages || a.tree_rows != treeRows(c.T))) return hipErrorInvalidValue;
    if (a.work_bytes < attentionWorkspaceBytes(c.T, c.S, a.H, c.KVH, c.D, c.pages ? c.capacity : c.T, a.window, a.sinks, a.parents ? a.tree_rows : 0, a.parents && a.key_scales)) return hipErrorInvalidValue;
    return hipSuccess;
}

constexpr size_t streamLds(int DT, bool Q8) {
    const size_t tiles = 4 * 32 * DT * (Q8 ? 1 : 2) + (Q8 ? 4 * 64 * 4 : 0), join = 4 * 16 * (DT + 4) * 4;
    return tiles > join ? tiles : join;
}

template <int DT, bool PAGED, bool Q8>
static hipError_t enqueueAttention(const AttentionArgs &a, const AttentionPlan &p, const LaunchCtx &ctx) {
    if (p.grid > 0x7fffffffLL || p.slots * 4 > (int64_t)kAttentionCounterBytes) return hipErrorInvalidValue;
    const dim3 grid((unsigned)p.grid);
    if (p.tiles) {
        constexpr int KB = DT >= 128 ? 32 : 64;
        constexpr size_t tiles = 4 * KB * DT * 2 + 4 * KB * 4 + 16 + 2 * KB, streams = PAGED && DT <= 128 ? streamLds(DT, Q8) : 0, lds = tiles > streams ? tiles : streams;
        static_assert(lds >= (4 * kMaxHeadDim + 128 * 17 + 1) * 4, "what joins the parts");
        auto enqueue = [&](auto fine) -> hipError_t {
            constexpr bool FINE = decltype(fine)::value;
            if constexpr (PAGED) {
                if (a.parents) {
                    AttentionArgs t = a;
                    t.tree_at = lds;
                    const int bytes = (int)lds + treeBytes(a.tree_rows, 128);
                    auto kernel = tree_attention_tiles<DT, Q8, FINE>;
                    if (ctx.name) {
                        if (hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds + treeBytes(kTreeRows, 128))) return e;
                    }
                    THIP_ENQUEUE(ctx, kernelLabel("tree_attention_tiles", {DT, Q8, FINE}), kernel, grid, dim3(256), bytes, t, p);
                    return hipSuccess;
                }
            }
            auto kernel = attention_tiles<DT, PAGED, Q8, FINE>;
            // asked for the kernel's name, as every executable does once on its device, the launcher configures it there
            if (lds > 64 * 1024 && ctx.name) {
                if (hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds)) return e;
            }
            THIP_ENQUEUE(ctx, kernelLabel("attention_tiles", {DT, PAGED, Q8, FINE}), kernel, grid, dim3(256), lds, a, p);
            return hipSuccess;
        };
        if (hipError_t e = p.fine ? enqueue(std::true_type{}) : enqueue(std::false_type{})) return e;
    } else {
        constexpr size_t lds = streamLds(DT, Q8);
        static_assert(lds >= (4 * kMaxHeadDim + 16 * 65 + 1) * 4, "what joins the parts");
        auto enqueue = [&](auto exact) -> hipError_t {
            constexpr bool EXACT = decltype(exact)::value;
            if constexpr (PAGED) {
                if (a.parents) {
                    AttentionArgs t = a;
                    t.tree_at = lds;
                    const int bytes = (int)lds + treeBytes(a.tree_rows, 16);
                    auto kernel = tree_attention_stream<DT, EXACT, Q8>;
                    if (ctx.name) {
                        if (hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds + treeBytes(kTreeRows, 16))) return e;
                    }
                    THIP_ENQUEUE(ctx, kernelLabel("tree_attention_stream", {DT, EXACT, Q8}), kernel, grid, dim3(256), bytes, t, p);
                    return hipSuccess;
                }
            }
            auto kernel = attention_stream<DT, EXACT, PAGED, Q8>;
            if (lds > 64 * 1024 && ctx.name) {
                if (hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds)) return e;
            }
            THIP_ENQUEUE(ctx, kernelLabel("attention_stream", {DT, EXACT, PAGED, Q8}), kernel, grid, dim3(256), lds, a, p);
            return hipSuccess;
        };
        if (hipError_t e = a.c.D == DT ? enqueue(std::true_type{}) : enqueue(std::false_type{})) return e;
    }
    return ctx.name ? hipSuccess : hipGetLastError();
}

template <bool PAGED, bool Q8>
static hipError_t byHeadDim(const AttentionArgs &a, const AttentionPlan &p, const LaunchCtx &ctx) {
    if (a.c.D <= 64) return enqueueAttention<64, PAGED, Q8>(a, p, ctx);
    if (a.c.D <= 128) return enqueueAttention<128, PAGED, Q8>(a, p, ctx);
    return enqueueAttention<256, PAGED, Q8>(a, p, ctx);
}

hipError_t launchAttention(const AttentionArgs &a, const LaunchCtx &ctx) {
    if (hipError_t e = checkAttention(a)) return e;
    const AttentionPlan p = attentionPlan(a.c.T, a.c.S, a.H, a.c.KVH, a.c.D, a.c.pages ? a.c.capacity : a.c.T, a.window, a.sinks, a.key_scales != nullptr,
                                          a.parents ? a.tree_rows : 0);
    return !a.c.pages ? byHeadDim<false, false>(a, p, ctx) : a.key_scales ? byHeadDim<true, true>(a, p, ctx) : byHeadDim<true, false>(a, p, ctx);
}

}  // namespace thip
