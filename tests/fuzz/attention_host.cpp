// Host-side fuzz of programs around a paged cache (thip_lm_*) and of their descriptors, meant to be built with -fsanitize=address,undefined.  Nothing here
// touches a GPU.  Random programs of cache writes, reads, attentions, transposes and matmuls on the same bindings and intermediates, with operands that are
// sometimes no values or values of other shapes: every call comes back with a status, what serialises validates, and so do mutated copies of it (or not).
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

struct Program {
    thip_program_t *p = nullptr;
    uint32_t bindings = 0;
    std::vector<thip_value_t> values;
    thip_value_t keep(thip_value_t v) {
        values.push_back(v);
        return v;
    }
    thip_value_t binding(std::vector<int64_t> shape, int32_t dtype) {
        thip_value_t v = -1;
        thip_program_binding(p, bindings++, dtype, (int32_t)shape.size(), shape.data(), &v);
        return keep(v);
    }
    thip_value_t tensor(std::vector<int64_t> shape) {
        thip_value_t v = -1;
        thip_program_tensor(p, THIP_DTYPE_BF16, (int32_t)shape.size(), shape.data(), &v);
        return keep(v);
    }
    thip_value_t view(thip_value_t base, std::vector<int64_t> shape, int64_t at) {
        thip_value_t v = -1;
        thip_program_view(p, base, at, (int32_t)shape.size(), shape.data(), &v);
        return keep(v);
    }
};

static bool build(bool insane, std::vector<uint64_t> *words, size_t *size, long *counts) {
    Program g;
    if (thip_program_create(&g.p) != THIP_OK) return false;
    const int64_t S = pick(1, 9), T = pick(S, S + 60), KVH = pick(1, 3), H = KVH * pick(1, 4), D = 16 * pick(1, 6), page = 8 * pick(1, 8), P = pick(1, 60), NP = pick(2, 40);
    const bool quantised = rng() & 1;
    const int32_t bf = THIP_DTYPE_BF16, cacheType = quantised ? THIP_DTYPE_I8 : bf;
    thip_value_t cache[2], scales[2] = {THIP_NO_VALUE, THIP_NO_VALUE};
    for (auto &c : cache) c = g.binding({NP, KVH, page, D}, cacheType);
    if (quantised) {
        for (auto &s : scales) s = g.binding({NP, KVH, page}, THIP_DTYPE_F32);
    }
    const thip_value_t pages = g.binding({S, P}, THIP_DTYPE_I32), starts = g.binding({S + 1}, THIP_DTYPE_I32), lengths = g.binding({S}, THIP_DTYPE_I32);
    std::vector<thip_value_t> rows, queries;
    for (int i = 0; i < 2; i++) {
        rows.push_back(g.binding({T, KVH, D}, bf));
        queries.push_back(g.binding({T, H, D}, bf));
        rows.push_back(g.tensor({T, KVH, D}));
        queries.push_back(g.tensor({T, H, D}));
    }
    // rows in the caches' own bytes, and a transposed view of them
    if (!quantised && NP * page >= T) rows.push_back(g.view(cache[0], {T, KVH, D}, 0));
    const int64_t seen = NP * KVH;
    const thip_value_t turnable = quantised ? THIP_NO_VALUE : g.view(cache[0], {seen, page, D}, 0), turned = g.tensor({seen, D, page});
    float zero = 0.0f;
    int64_t one[1] = {1};
    thip_value_t bias = -1;
    thip_program_constant(g.p, THIP_DTYPE_F32, 1, one, &zero, 4, &bias);
    auto any = [&](thip_value_t v) { return insane && rng() % 12 == 0 ? (rng() & 1 ? wild() : g.values[rng() % g.values.size()]) : v; };
    // operands: what is there (bindings, and intermediates once they have been written), no two of an op the same
    std::vector<thip_value_t> made, used;
    auto one_of = [&](const std::vector<thip_value_t> &from, bool read) {
        for (int tries = 0; tries < 50; tries++) {
            const size_t i = rng() % from.size();
            const thip_value_t v = from[i];
            bool no = false;
            for (thip_value_t u : used) no = no || u == v;
            if (read && i % 2 == 1 && i < 4) {
                bool there = false;
                for (thip_value_t u : made) there = there || u == v;
                no = no || !there;
            }
            if (no) continue;
            used.push_back(v);
            if (!read) made.push_back(v);
            return any(v);
        }
        return any(from[0]);
    };
    auto row = [&](bool read) { return one_of(rows, read); };
    auto query = [&](bool read) { return one_of(queries, read); };
    for (int n = (int)pick(1, 4); n > 0; n--) {
        used.clear();
        thip_status_t s = THIP_OK;
        switch (rng() % 6) {
        case 0: {
            thip_lm_cache_write_t c{any(cache[0]), any(cache[1]), any(scales[0]), any(scales[1]), row(true), row(true), any(pages), any(starts), any(lengths)};
            s = thip_lm_cache_write(g.p, &c);
            break;
        }
        case 1: {
            thip_lm_cache_read_t c{row(false), row(false), any(cache[0]), any(cache[1]), any(scales[0]), any(scales[1]), any(pages), any(starts), any(lengths)};
            s = thip_lm_cache_read(g.p, &c);
            break;
        }
        case 2: {
            thip_lm_attention_t c{query(false), query(true), row(true), row(true), THIP_NO_VALUE, THIP_NO_VALUE, THIP_NO_VALUE, any(starts), THIP_NO_VALUE, 0.125f, insane ? wild() : 0, 0};
            s = thip_lm_attention(g.p, &c);
            break;
        }
        case 3: {
            thip_lm_attention_t c{query(false), query(true), any(cache[0]), any(cache[1]), any(scales[0]), any(scales[1]), any(pages), any(starts), any(lengths), 0.125f,
                                  rng() & 1 ? (int32_t)pick(0, 90) : 0, insane ? wild() : 3};
            s = thip_lm_attention(g.p, &c);
            break;
        }
        case 4: {
            if (quantised && !insane) break;
            thip_hl_transpose_t t;
            memset(&t, 0, sizeof(t));
            t.init = any(turned);
            t.input = any(turnable);
            t.rank = 3;
            t.perm[1] = 2;
            t.perm[2] = 1;
            s = thip_hl_transpose(g.p, &t);
            if (rng() % 3 == 0) break;
            if (rng() & 1) {  // between the transpose and its matmul
                thip_lm_cache_write_t c{cache[0], cache[1], scales[0], scales[1], rows[0], rows[2], pages, starts, lengths};
                s = thip_lm_cache_write(g.p, &c);
            }
            [[fallthrough]];
        }
        default: {
            if (quantised && !insane) break;
            thip_hl_matmul_t m;
            memset(&m, 0, sizeof(m));
            m.input1 = g.binding({seen, pick(1, 40), D}, bf);
            m.input2 = any(turned);
            m.init = g.tensor({seen, 1, page});
            m.output_min = (int32_t)0xff800000;
            m.output_max = 0x7f800000;
            m.scale_bias = bias;
            s = thip_hl_matmul(g.p, &m);
        }
        }
        counts[s == THIP_OK ? 0 : 1]++;
    }
    void *blob = nullptr;
    const thip_status_t s = thip_program_serialize(g.p, &blob, size);
    counts[s == THIP_OK ? 2 : 3]++;
    if (s == THIP_OK) {
        words->assign((*size + 7) / 8, 0);
        memcpy(words->data(), blob, *size);
        thip_blob_free(blob);
    }
    thip_program_destroy(g.p);
    return s == THIP_OK;
}

int main(int argc, char **argv) {
    if (argc != 3) return 2;
    rng.seed((uint64_t)atoi(argv[2]));
    long counts[4] = {0, 0, 0, 0}, attentions = 0, refused = 0, accepted = 0;
    for (int it = 0; it < atoi(argv[1]); it++) {
        std::vector<uint64_t> blob;
        size_t size = 0;
        if (!build(it % 2 == 1, &blob, &size, counts)) continue;
        if (thip_descriptor_validate(blob.data(), size) != THIP_OK) {
            printf("FAIL: what the emitter wrote does not validate: %s\n", thip_status_message());
            return 1;
        }
        const thip::DescHeader *h = (const thip::DescHeader *)blob.data();
        for (uint32_t i = 0; i < h->op_count; i++) attentions += ((const thip::DescOp *)((const uint8_t *)blob.data() + h->ops_offset))[i].kind == thip::kKindAttention;
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
    printf("ops taken %ld, refused %ld; programs serialised %ld, refused %ld; attention records %ld; mutants refused %ld, accepted %ld\n", counts[0], counts[1], counts[2], counts[3],
           attentions, refused, accepted);
    return counts[2] > 20 && attentions > 20 && refused > 0 ? 0 : 1;
}
