// Host-side fuzz of programs of norms, rotary positions, attention of trees and moves in the cache (thip_lm_*), and of their descriptors, meant to be built with
// -fsanitize=address,undefined.  Nothing here touches a GPU.  Operands are sometimes no values, values of other shapes, or share bytes: every call comes back with
// a status, what serialises validates, and so do mutated copies of it (or not).
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <random>
#include <vector>

#include "../../include/thip.h"
#include "../../torq-compiler_amd/csrc/thip_descriptor.h"

static std::mt19937_64 rng;
static int64_t pick(int64_t lo, int64_t hi) { return lo + (int64_t)(rng() % (uint64_t)(hi - lo + 1)); }
static int32_t wild() {
    static const int32_t some[] = {0, -1, INT32_MAX, INT32_MIN, 1, 1 << 30};
    return rng() % 3 ? some[rng() % 6] : (int32_t)rng();
}
static float wildFloat() {
    static const float some[] = {0.0f, -1.0f, INFINITY, NAN, 1e38f, 1e-40f};
    return some[rng() % 6];
}

static bool build(bool insane, std::vector<uint64_t> *words, size_t *size, long *counts) {
    thip_program_t *p = nullptr;
    if (thip_program_create(&p) != THIP_OK) return false;
    std::vector<thip_value_t> values;
    uint32_t bindings = 0;
    const auto binding = [&](std::vector<int64_t> shape, int32_t dtype) {
        thip_value_t v = -1;
        thip_program_binding(p, bindings++, dtype, (int32_t)shape.size(), shape.data(), &v);
        values.push_back(v);
        return v;
    };
    const auto tensor = [&](std::vector<int64_t> shape, int32_t dtype) {
        thip_value_t v = -1;
        thip_program_tensor(p, dtype, (int32_t)shape.size(), shape.data(), &v);
        values.push_back(v);
        return v;
    };
    const auto view = [&](thip_value_t base, std::vector<int64_t> shape, int64_t at) {
        thip_value_t v = -1;
        thip_program_view(p, base, at, (int32_t)shape.size(), shape.data(), &v);
        values.push_back(v);
        return v;
    };
    const auto constant = [&](std::vector<int64_t> shape, int32_t dtype, const void *data, size_t bytes) {
        thip_value_t v = -1;
        thip_program_constant(p, dtype, (int32_t)shape.size(), shape.data(), data, bytes, &v);
        values.push_back(v);
        return v;
    };
    const auto any = [&](thip_value_t v) { return insane && rng() % 12 == 0 ? (rng() & 1 ? wild() : values[rng() % values.size()]) : v; };
    const auto maybe = [&](thip_value_t v) { return rng() % 3 ? v : THIP_NO_VALUE; };

    const int64_t S = pick(1, 9), T = pick(S, S + 60), KVH = pick(1, 3), H = KVH * pick(1, 4), D = 16 * pick(1, 6), page = 8 * pick(1, 8), P = pick(1, 60), NP = pick(2, 40), K = pick(1, 80);
    const bool quantised = rng() & 1;
    const int32_t bf = THIP_DTYPE_BF16, f32 = THIP_DTYPE_F32, i32 = THIP_DTYPE_I32, cacheType = quantised ? THIP_DTYPE_I8 : bf;
    thip_value_t cache[2], scales[2] = {THIP_NO_VALUE, THIP_NO_VALUE};
    for (auto &c : cache) c = binding({NP, KVH, page, D}, cacheType);
    if (quantised) {
        for (auto &s : scales) s = binding({NP, KVH, page}, f32);
    }
    const thip_value_t pages = binding({S, P}, i32), starts = binding({S + 1}, i32), lengths = binding({S}, i32), parents = binding({T}, i32), accepted = binding({S, K}, i32);
    const thip_value_t positions = binding({2, T}, i32);
    std::vector<thip_value_t> queries{binding({T, H, D}, bf), binding({T, H, D}, bf)}, keys{binding({T, KVH, D}, bf), binding({T, KVH, D}, bf)};
    std::vector<thip_value_t> made{tensor({T, H, D}, bf), tensor({T, H, D}, bf)};  // the program's own
    const int64_t N = pick(1, 300);
    const thip_value_t wide = binding({3 * T, N}, bf), stream = binding({T, N}, f32), gates[] = {binding({T, N}, bf), binding({T, 1}, bf), binding({1, N}, bf), binding({1, 1}, bf)};
    std::vector<thip_value_t> rows{view(wide, {T, N}, 0), view(wide, {T, N}, T * N), view(wide, {T, N}, 2 * T * N), tensor({T, N}, bf), stream, tensor({T, N}, f32)};
    const thip_value_t weights[] = {binding({N}, bf), binding({N}, f32), binding({D}, bf)};
    float frequencies[128];
    int32_t axes[128];
    const int64_t pairs = insane ? pick(1, 128) : 8 * pick(1, D / 16);
    for (int i = 0; i < 128; i++) {
        frequencies[i] = insane && rng() % 40 == 0 ? wildFloat() : (float)pick(-16000, 16000) * 1e-3f;
        axes[i] = insane && rng() % 40 == 0 ? wild() : (int32_t)(rng() & 1);
    }
    const thip_value_t freq = constant({pairs}, f32, frequencies, (size_t)pairs * 4), axis = constant({pairs}, i32, axes, (size_t)pairs * 4);
    for (int n = (int)pick(1, 5); n > 0; n--) {
        thip_status_t s = THIP_OK;
        switch (rng() % 5) {
        case 0: {
            const thip_lm_tree_attention_t c{any(rng() % 3 ? queries[1] : made[0]), any(queries[0]), any(cache[0]), any(cache[1]), any(scales[0]), any(scales[1]), any(pages), any(starts), any(lengths),
                                             any(parents), insane && rng() % 9 == 0 ? wildFloat() : 0.125f, rng() & 1 ? (int32_t)pick(0, 90) : 0, insane ? wild() : 3};
            s = thip_lm_tree_attention(p, &c);
            break;
        }
        case 1: {
            const thip_lm_cache_keep_t c{any(cache[0]), any(cache[1]), any(scales[0]), any(scales[1]), any(accepted), any(pages), any(starts), any(lengths)};
            s = thip_lm_cache_keep(p, &c);
            break;
        }
        case 2: {
            const bool alone = rng() % 3 == 0;
            const thip_lm_rotary_t c{any(rng() & 1 ? queries[0] : made[1]), any(alone ? THIP_NO_VALUE : keys[rng() & 1]), any(queries[0]), any(alone ? THIP_NO_VALUE : keys[0]), any(positions), any(freq),
                                     any(maybe(axis)), (int32_t)(rng() & 1)};
            s = thip_lm_rotary(p, &c);
            break;
        }
        case 3: {  // of heads
            const thip_lm_norm_t c{any(made[0]), THIP_NO_VALUE, any(queries[rng() & 1]), THIP_NO_VALUE, any(maybe(weights[2])), THIP_NO_VALUE, any(weights[2]), 1e-6f, 0.0f, 1.0f};
            s = thip_lm_norm(p, &c);
            break;
        }
        default: {
            const bool sums = rng() & 1, norms = !sums || rng() % 4;
            const thip_lm_norm_t c{any(norms ? rows[rng() & 1 ? 1 : 3] : THIP_NO_VALUE), any(sums ? rows[rng() & 1 ? 4 : 5] : THIP_NO_VALUE), any(rows[0]), any(maybe(rows[rng() & 1 ? 2 : 4])),
                                   any(maybe(weights[rng() & 1])), any(maybe(gates[rng() % 4])), any(norms ? weights[rng() & 1] : THIP_NO_VALUE), insane && rng() % 9 == 0 ? wildFloat() : 1e-6f,
                                   insane && rng() % 9 == 0 ? wildFloat() : 1.0f, insane && rng() % 9 == 0 ? wildFloat() : 0.5f};
            s = thip_lm_norm(p, &c);
        }
        }
        counts[s == THIP_OK ? 0 : 1]++;
    }
    void *blob = nullptr;
    const thip_status_t s = thip_program_serialize(p, &blob, size);
    counts[s == THIP_OK ? 2 : 3]++;
    if (s == THIP_OK) {
        words->assign((*size + 7) / 8, 0);
        memcpy(words->data(), blob, *size);
        thip_blob_free(blob);
    }
    thip_program_destroy(p);
    return s == THIP_OK;
}

int main(int argc, char **argv) {
    if (argc != 3) return 2;
    rng.seed((uint64_t)atoi(argv[2]));
    long counts[4] = {0, 0, 0, 0}, kinds[64] = {0}, refused = 0, accepted = 0;
    for (int it = 0; it < atoi(argv[1]); it++) {
        std::vector<uint64_t> blob;
        size_t size = 0;
        if (!build(it % 2 == 1, &blob, &size, counts)) continue;
        if (thip_descriptor_validate(blob.data(), size) != THIP_OK) {
            printf("FAIL: what the emitter wrote does not validate: %s\n", thip_status_message());
            return 1;
        }
        const thip::DescHeader *h = (const thip::DescHeader *)blob.data();
        for (uint32_t i = 0; i < h->op_count; i++) kinds[((const thip::DescOp *)((const uint8_t *)blob.data() + h->ops_offset))[i].kind & 63]++;
        for (int m = 0; m < 40; m++) {
            std::vector<uint64_t> bad = blob;
            uint8_t *bytes = (uint8_t *)bad.data();
            for (int f = (int)pick(1, 3); f > 0; f--) {
                const size_t at = (size_t)pick(0, (int64_t)size - 4) & ~(size_t)3;
                const int32_t v = wild();
                if (rng() & 1) memcpy(bytes + at, &v, 4);
                else bytes[at] ^= (uint8_t)(1u << (rng() % 8));
            }
            (thip_descriptor_validate(bad.data(), size) == THIP_OK ? accepted : refused)++;
        }
    }
    printf("ops taken %ld, refused %ld; programs serialised %ld, refused %ld; records: tree %ld, keep %ld, rotary %ld, norm %ld; mutants refused %ld, accepted %ld\n", counts[0], counts[1], counts[2], counts[3],
           kinds[thip::kKindTreeAttention], kinds[thip::kKindCacheKeep], kinds[thip::kKindRotary], kinds[thip::kKindNorm], refused, accepted);
    for (uint32_t k : {thip::kKindTreeAttention, thip::kKindCacheKeep, thip::kKindRotary, thip::kKindNorm}) {
        if (kinds[k] < 10) return 1;
    }
    return counts[2] > 40 && refused > 0 ? 0 : 1;
}
