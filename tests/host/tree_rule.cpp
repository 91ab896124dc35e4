// By streams or by tiles: of trees that were timed both ways (with sequences of a third to all of the longest's rows and positions) the plan takes none
// by a side that is an eighth slower, and all together by what is at most 2 % above the faster sides' sum.  Prints the two sums.
#include <stdio.h>

#include "thip_attention.h"

struct Timed {
    int64_t rows, sequences, heads, kvHeads, D, capacity, window;
    bool quantised;
    double streams, tiles;  // us
};
static const Timed kTimed[] = {
    {12, 1, 16, 4, 128, 2496, 0, true, 12.8, 38.7},
    {129, 1, 4, 1, 128, 7328, 2275, true, 16.5, 50.4},
    {148, 32, 64, 8, 80, 1128, 512, true, 30.5, 33.9},
    {1714, 20, 32, 8, 80, 768, 0, false, 67.8, 36.4},
    {770, 3, 8, 8, 256, 2928, 0, false, 165.5, 77.1},
    {409, 8, 32, 8, 256, 4336, 0, true, 187.8, 212.3},
    {104, 7, 32, 4, 128, 25600, 0, false, 259.7, 121.4},
    {128, 46, 32, 2, 128, 19968, 0, true, 122.8, 206.2},
    {20, 1, 64, 8, 256, 32768, 0, true, 199.5, 216.1},
    {100, 1, 8, 8, 256, 32768, 0, true, 133.4, 217.5},
    {208, 4, 16, 4, 256, 8192, 0, true, 106.0, 139.1},
    {298, 4, 16, 4, 256, 8192, 0, true, 127.6, 164.7},
    {352, 16, 8, 2, 256, 8192, 0, true, 93.2, 140.7},
    {1084, 16, 8, 2, 256, 4096, 0, true, 125.8, 142.6},
    {1077, 8, 8, 4, 256, 4096, 0, true, 111.8, 132.5},
    {769, 2, 16, 4, 256, 8192, 0, true, 295.7, 284.0},
    {642, 32, 16, 4, 256, 2048, 0, true, 94.5, 113.7},
    {553, 2, 16, 8, 256, 20032, 0, true, 557.4, 436.6},
    {615, 8, 32, 8, 256, 4096, 0, true, 252.6, 231.8},
    {690, 4, 32, 8, 256, 1024, 0, true, 81.2, 90.4},
    {735, 16, 32, 8, 256, 4096, 0, true, 263.1, 244.4},
    {319, 3, 64, 8, 256, 12032, 0, true, 704.9, 541.3},
    {247, 24, 64, 8, 256, 4096, 0, true, 198.9, 221.7},
};

int main() {
    double taken = 0, least = 0;
    bool ok = true;
    for (const Timed &t : kTimed) {
        const thip::AttentionPlan p = thip::attentionPlan(t.rows, t.sequences, t.heads, t.kvHeads, t.D, t.capacity, t.window, 0, t.quantised, thip::treeRows(t.rows));
        const double us = p.tiles ? t.tiles : t.streams, best = t.tiles < t.streams ? t.tiles : t.streams;
        taken += us;
        least += best;
        if (us <= 1.125 * best) continue;
        printf("FAIL: %lld rows of %lld sequences, %lld heads of %lld over %lld: %s take %g us, the others %g\n", (long long)t.rows, (long long)t.sequences, (long long)t.heads, (long long)t.D,
               (long long)t.kvHeads, p.tiles ? "tiles" : "streams", us, best);
        ok = false;
    }
    printf("%.1f %.1f\n", taken, least);
    return ok && taken <= 1.02 * least ? 0 : 1;
}
