// Which blocks the tiles of trees read and how their runs are cut, by the arithmetic that the kernels use (thip_attention.h), on the host: every position that a row of a
// tile can see lies in the tile's blocks, those are no more than the sequence's count, which parts are made of, and a cut run's parts have all of them; parts and
// workgroups have their places.  Trees whose first rows stand below position 0, of more rows than a tree has, of sequences longer than their tables.
// Arguments: a seed; "short": the count as if it were one block less, which has to be found.  Prints how many tiles were cut.
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <random>
#include <vector>

#include "thip_attention.h"

using namespace thip;

static std::mt19937 rng;
static int64_t pick(int64_t low, int64_t high) {  // even over the logarithm
    const double x = exp(std::uniform_real_distribution<double>(log((double)low), log((double)high + 1))(rng));
    return std::min(high, std::max(low, (int64_t)x));
}

struct Seq {
    int32_t rows, first, length, tiles, blocks, splits;
    bool light;
};

int main(int argc, char **argv) {
    if (argc < 2) return 2;
    rng.seed((unsigned)atoi(argv[1]));
    const bool shorter = argc > 2 && !strcmp(argv[2], "short");
    long cut = 0;
    for (int it = 0; it < 20000; it++) {
        const int64_t S = pick(1, 100), KVH = pick(1, 16), G = pick(1, 16), D = 16 * pick(1, 16), most = pick(1, 900), longest = pick(1, 40000), page = pick(1, 128);
        const int64_t window = rng() % 4 ? rng() % 16 ? pick(1, 5000) : 0x7fffffff : 0, sinks = window && (rng() & 1) ? rng() % 16 ? pick(1, 6000) : 0x7fffffff : 0;
        const bool quantised = rng() & 1;
        std::vector<Seq> seqs((size_t)S);
        int64_t T = 0, top = 1;
        for (Seq &s : seqs) {
            s.rows = (int32_t)(pick(1, most) - (rng() % 5 == 0));
            const int64_t length = rng() % 8 ? pick(1, longest) : rng() % 2 ? 0 : s.rows / 2;  // some of fewer positions than rows
            s.first = (int32_t)(length - s.rows);
            T += s.rows;
            top = std::max(top, length);
        }
        if (T < 1) continue;
        int64_t P = (top - 1) / page + 1;
        if (rng() % 3 == 0) P += pick(1, 50);
        else if (rng() % 4 == 0) P = std::max<int64_t>(1, P / 2);  // sequences pass the end of their tables
        const int64_t capacity = P * page, tree = treeRows(T);
        const AttentionPlan p = attentionPlan(T, S, KVH * G, KVH, D, capacity, window, sinks, quantised, tree);
        float total = 0.0f, full = 0.0f;
        for (Seq &s : seqs) {
            s.length = (int32_t)std::min<int64_t>((int64_t)s.first + s.rows, capacity);
            s.tiles = (int32_t)((s.rows * G + p.rows() - 1) >> p.rowsLog);
            s.blocks = seqBlocks(p, (int32_t)window, (int32_t)sinks, (int32_t)tree, s.first, s.rows, s.length);
            if (shorter && s.blocks > 1) s.blocks--;
            s.light = p.tiles && D <= 128 && s.rows * G <= 16;
            total += (float)s.tiles * (float)s.blocks * (s.light ? 0.25f : 1.0f);
            if (s.rows * G > 16) full += (float)s.tiles;
        }
        const PartBlocks part = p.splits ? partBlocks(p, total, full, (int32_t)KVH) : PartBlocks{0, 0, 0};
        int64_t items = 0, parts = 0;
        for (Seq &s : seqs) {
            s.splits = partsOf(p, s.blocks, s.light ? part.stream : part.tile, s.light ? 0 : part.tileWhole);
            items += (int64_t)s.tiles * s.splits * KVH;
            if (s.splits > 1) parts += (int64_t)s.tiles * s.splits * KVH;
            const int64_t each = s.splits > 1 ? (s.blocks + s.splits - 1) / s.splits : 0, keys = p.keys();
            for (int64_t t = 0; t < s.tiles; t++) {
                const int64_t last = (std::min<int64_t>((t + 1) * p.rows(), s.rows * G) - 1) / G;
                const RowBlocks r = rowBlocks(p, (int32_t)window, (int32_t)sinks, s.first, (int32_t)(s.first + std::min(last, tree - 1)), s.length);
                const auto reads = [&](int64_t position) {
                    const int64_t b = position / keys;
                    return b < r.sinks || (b >= r.window && b - r.window < r.all - r.sinks);
                };
                // a tile's rows stand at positions from the tree's first to its last place; what they can see, at its ends: the text from the first one's window on, the first
                // positions, the tree's places up to the tile's last row
                const int64_t base = s.first, end = std::min<int64_t>(base + std::min(last, tree - 1), s.length - 1);
                std::vector<int64_t> look;
                if (end >= 0) {
                    const int64_t low = window ? std::max<int64_t>(std::max<int64_t>(base, 0) - window + 1, 0) : 0;
                    for (int64_t x : {low, low + 1, std::max<int64_t>(base, 0) - 1, std::max<int64_t>(base, 0), end - 1, end}) {
                        if (x >= low && x <= end) look.push_back(x);
                    }
                    for (int64_t x : {(int64_t)0, sinks / 2, std::min(sinks, base) - 1}) {
                        if (window && x >= 0 && x < sinks && x < base && x <= end) look.push_back(x);
                    }
                }
                for (int64_t x : look) {
                    if (reads(x)) continue;
                    printf("FAIL: position %lld is in no block (rows %d first %d length %d window %lld sinks %lld)\n", (long long)x, s.rows, s.first, s.length, (long long)window, (long long)sinks);
                    return 1;
                }
                if (r.all > s.blocks || (s.splits > 1 && r.all > each * s.splits)) {
                    printf("FAIL: %d blocks, the sequence counts %d, in %d parts of %lld (rows %d first %d length %d window %lld sinks %lld)\n", r.all, s.blocks, s.splits, (long long)each, s.rows,
                           s.first, s.length, (long long)window, (long long)sinks);
                    return 1;
                }
                cut += s.splits > 1;
            }
        }
        if (items > p.grid || parts > p.slots || p.slots * 4 > (int64_t)kAttentionCounterBytes) {
            printf("FAIL: %lld items of %lld, %lld parts of %lld\n", (long long)items, (long long)p.grid, (long long)parts, (long long)p.slots);
            return 1;
        }
    }
    printf("%ld\n", cut);
    return cut > 1000 ? 0 : 1;
}
