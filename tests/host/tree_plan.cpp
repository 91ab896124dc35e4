// How attention of trees shares out its work (thip_attention.h), on the host: whatever a tree's size, its window and the positions before it are, a tile's run of
// blocks is no longer than the plan takes it for, so that the parts of a run that is cut have all of it; parts and workgroups have their places.
// Argument: a seed.  Prints how many tiles were cut.
#include <math.h>
#include <stdio.h>
#include <stdlib.h>

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
    int64_t rows, length;
};

int main(int argc, char **argv) {
    if (argc != 2) return 2;
    rng.seed((unsigned)atoi(argv[1]));
    long cut = 0;
    for (int it = 0; it < 20000; it++) {
        const int64_t S = pick(1, 200), KVH = pick(1, 16), G = pick(1, 16), D = 16 * pick(1, 16), most = pick(1, 700), longest = pick(1, 40000);
        const int64_t window = rng() & 1 ? pick(1, 5000) : 0, sinks = window && (rng() & 1) ? pick(1, 300) : 0, page = pick(1, 128);
        const bool quantised = rng() & 1;
        std::vector<Seq> seqs;
        int64_t T = 0, top = 1;
        for (int64_t s = 0; s < S; s++) {
            seqs.push_back({pick(1, most) - (rng() % 5 == 0), pick(1, longest)});
            T += seqs.back().rows;
            top = std::max(top, seqs.back().length);
        }
        if (T < 1) continue;
        const int64_t P = (top - 1) / page + 1 + (rng() % 3 ? 0 : pick(1, 50)), capacity = P * page, tree = treeRows(T);
        const AttentionPlan p = attentionPlan(T, S, KVH * G, KVH, D, capacity, window, sinks, quantised, tree);
        const uint64_t sized = attentionWorkspaceBytes(T, S, KVH * G, KVH, D, capacity, window, sinks, tree, quantised);
        if (sized != (p.slots ? kAttentionCounterBytes + (uint64_t)p.slots * p.rows() * (D + 4) * 4 : 0)) {
            printf("FAIL: a workspace that the launch does not fit\n");
            return 1;
        }
        float total = 0.0f, full = 0.0f;
        std::vector<int64_t> tiles(S), blocks(S);
        std::vector<bool> light(S);
        for (int64_t s = 0; s < S; s++) {
            const int64_t rows = seqs[s].rows * G;
            tiles[s] = (rows + p.rows() - 1) >> p.rowsLog;
            blocks[s] = (std::min(seqs[s].length, capacity) + p.keys() - 1) >> p.keysLog;
            if (window) blocks[s] = std::min<int64_t>(blocks[s], p.windowBlocks);
            light[s] = p.tiles && D <= 128 && rows <= 16;
            total += (float)tiles[s] * (float)blocks[s] * (light[s] ? 0.25f : 1.0f);
            if (rows > 16) full += (float)tiles[s];
        }
        const PartBlocks part = p.splits ? partBlocks(p, total, full, (int32_t)KVH) : PartBlocks{0, 0, 0};
        int64_t items = 0, parts = 0;
        for (int64_t s = 0; s < S; s++) {
            const int32_t n = partsOf(p, (int32_t)blocks[s], light[s] ? part.stream : part.tile, light[s] ? 0 : part.tileWhole);
            const int64_t each = n > 1 ? (blocks[s] + n - 1) / n : 0;
            items += tiles[s] * n * KVH;
            if (n > 1) parts += tiles[s] * n * KVH;
            const int64_t base = seqs[s].length - seqs[s].rows, length = std::min(seqs[s].length, capacity);
            for (int64_t t = 0; t < tiles[s]; t++) {
                const int64_t last = std::min(t * p.rows() + p.rows(), seqs[s].rows * G) - 1;
                const int64_t bottom = base + std::min(last / G, tree - 1), high = std::max<int64_t>(std::min(bottom + 1, length), 0);
                const int64_t low = window ? std::max<int64_t>(std::max<int64_t>(base, -1) - window + 1, 0) : 0, keys = p.keys();
                const auto to = [&](int64_t end) { return (end + keys - 1) / keys; };
                const int64_t sinkBlocks = to(std::min(std::min(sinks, low), high)), windowBlock = std::max(low / keys, sinkBlocks);
                const int64_t run = sinkBlocks + std::max<int64_t>(to(high) - windowBlock, 0);
                if (n > 1) {
                    cut++;
                    if (run > each * n) {
                        printf("FAIL: %lld blocks in %d parts of %lld (rows %lld length %lld window %lld sinks %lld)\n", (long long)run, n, (long long)each, (long long)seqs[s].rows,
                               (long long)seqs[s].length, (long long)window, (long long)sinks);
                        return 1;
                    }
                }
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
