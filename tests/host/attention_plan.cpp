// How an attention shares out its work (thip_attention.h), on the host: for batches of every size and skew the items that the device makes of it are no more
// than the launch has workgroups, those that are parts no more than the workspace has places, every block of a tile is some part's, and a workspace of what
// attentionWorkspaceBytes says holds the last place.
// Argument: a seed.  Prints how many of the batches were cut.
#include <math.h>
#include <stdio.h>
#include <stdlib.h>

#include <random>
#include <vector>

#include "thip_attention.h"

using namespace thip;

struct Seq {
    int64_t rows, length;
};
static std::mt19937 rng;
static int64_t pick(int64_t low, int64_t high) {  // even over the logarithm
    const double x = exp(std::uniform_real_distribution<double>(log((double)low), log((double)high + 1))(rng));
    return std::min(high, std::max(low, (int64_t)x));
}

struct Made {
    int64_t items = 0, parts = 0, longest = 0;
};

static bool check(const std::vector<Seq> &seqs, int64_t KVH, int64_t G, int64_t D, int64_t capacity, int64_t window, int64_t sinks, bool cached, bool quantised, Made *made) {
    int64_t T = 0;
    for (const Seq &s : seqs) T += s.rows;
    const int64_t S = (int64_t)seqs.size(), H = KVH * G;
    const AttentionPlan p = attentionPlan(T, S, H, KVH, D, capacity, window, sinks, quantised);
    // what the device sums up, lane by lane, in 32 bits
    std::vector<float> total(256, 0.0f), full(256, 0.0f);
    std::vector<int64_t> tiles(S), blocks(S);
    std::vector<bool> light(S);
    for (int64_t s = 0; s < S; s++) {
        const int64_t rows = seqs[s].rows * G;
        tiles[s] = (rows + p.rows() - 1) >> p.rowsLog;
        blocks[s] = (std::min(seqs[s].length, capacity) + p.keys() - 1) >> p.keysLog;
        if (window) blocks[s] = std::min<int64_t>(blocks[s], p.windowBlocks);
        light[s] = p.tiles && cached && D <= 128 && rows <= 16;
        total[s % 256] += (float)tiles[s] * (float)blocks[s] * (light[s] ? 0.25f : 1.0f);
        if (rows > 16) full[s % 256] += (float)tiles[s];
    }
    float allBlocks = 0.0f, allFull = 0.0f;
    for (int i = 0; i < 256; i++) {
        allBlocks += total[i];
        allFull += full[i];
    }
    const PartBlocks part = p.splits ? partBlocks(p, allBlocks, allFull, (int32_t)KVH) : PartBlocks{0, 0, 0};
    *made = Made{};
    for (int64_t s = 0; s < S; s++) {
        const int32_t n = partsOf(p, (int32_t)blocks[s], light[s] ? part.stream : part.tile, light[s] ? 0 : part.tileWhole);
        if (p.splits && !p.tiles && blocks[s] > part.tile && n == 1) return false;  // streams are cut wherever they are longer than a part
        const int64_t each = (blocks[s] + n - 1) / n;
        if (n > 1 && (n > p.maxParts || each * n < blocks[s] || each < 1)) return false;
        made->items += tiles[s] * n * KVH;
        if (n > 1) made->parts += tiles[s] * n * KVH;
        made->longest = std::max(made->longest, each);
    }
    if (made->items > p.grid || made->parts > p.slots) return false;
    const uint64_t bytes = attentionWorkspaceBytes(T, S, H, KVH, D, capacity, window, sinks);
    return p.slots == 0 ? bytes == 0 : (uint64_t)p.slots * 4 <= kAttentionCounterBytes && bytes >= kAttentionCounterBytes + (uint64_t)p.slots * (uint64_t)(p.rows() * (D + 4) * 4);
}

int main(int argc, char **argv) {
    if (argc != 2) return 2;
    rng.seed((unsigned)atoi(argv[1]));
    static const int64_t heads[] = {1, 2, 3, 8, 16}, groups[] = {1, 2, 4, 5, 16}, dims[] = {16, 64, 80, 128, 256};
    int cut = 0;
    for (int i = 0; i < 3000; i++) {
        const int64_t KVH = heads[rng() % 5], G = groups[rng() % 5], D = dims[rng() % 5], S = pick(1, i % 50 == 0 ? 20000 : 400), capacity = pick(16, 1 << 17);
        const int64_t window = rng() % 3 ? 0 : pick(1, 40000), sinks = window ? pick(1, 100) - 1 : 0, most = pick(1, 3000);
        const bool cached = rng() % 4 != 0, quantised = cached && rng() % 2;
        std::vector<Seq> seqs(S);
        const int kind = rng() % 5;  // alike; one long; few rows in some; ragged; none in some
        for (int64_t s = 0; s < S; s++) {
            Seq &q = seqs[s];
            q.rows = kind == 0 ? most : kind == 1 ? 1 : kind == 2 ? (rng() % 2 ? 1 : most) : kind == 3 ? pick(1, most) : (int64_t)(rng() % 2) * most;
            q.length = kind == 0 ? capacity : kind == 1 ? (s == S / 2 ? capacity : std::min<int64_t>(capacity, 100)) : pick(1, capacity + 100);
            q.length = std::max(q.length, q.rows);
        }
        if (S > 2000) {
            for (Seq &q : seqs) q.rows = std::min<int64_t>(q.rows, 3);
        }
        int64_t T = 0;
        for (const Seq &q : seqs) T += q.rows;
        if (T < 1 || T * KVH * G >= (1LL << 31)) continue;
        Made m;
        if (!check(seqs, KVH, G, D, capacity, window, sinks, cached, quantised, &m)) {
            printf("batch %d: S %d T %d KVH %d G %d D %d capacity %d window %d sinks %d kind %d: items %d parts %d\n", i, (int)S, (int)T, (int)KVH, (int)G, (int)D, (int)capacity,
                   (int)window, (int)sinks, kind, (int)m.items, (int)m.parts);
            return 1;
        }
        cut += m.parts > 0;
    }
    // one long run among many short ones is cut, however many there are
    for (int64_t S : {2, 64, 65, 100, 300, 5000}) {
        std::vector<Seq> seqs(S, Seq{1, 200});
        seqs[S / 3].length = 32768;
        Made m;
        if (!check(seqs, 8, 4, 128, 32768, 0, 0, true, false, &m) || m.longest >= 1024) {
            printf("%d sequences: a run of %d blocks in one part\n", (int)S, (int)m.longest);
            return 1;
        }
        for (Seq &q : seqs) q.rows = 40;
        if (S <= 300 && (!check(seqs, 8, 4, 128, 32768, 0, 0, true, false, &m) || (S <= 100 && m.longest >= 1024))) {
            printf("%d sequences of 40 rows: a run of %d blocks in one part\n", (int)S, (int)m.longest);
            return 1;
        }
    }
    printf("%d\n", cut);
    return 0;
}
