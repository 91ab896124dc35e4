// Attention of packed rows over themselves or over a paged cache (thip_lm_attention).
//
// o = sum_j w_j v_j / sum_j w_j, w_j = exp(scale (q . k_j) - m), over the positions j that the row sees; one pass over the keys with a
// running maximum m and a running sum, both scaled down where a later key raises m.  Exponents are to base 2, with log2(e) in the scale.
#include "thip_attention.h"
#include "thip_attention_rows.h"
#include "thip_kernels_common.h"

namespace thip {

constexpr float kLog2e = 1.4426950408889634f;

// Whether a row at position p sees position j (0 <= j).
__device__ __forceinline__ bool sees(const AttentionArgs &a, int p, int j) { return j <= p && (a.window == 0 || p - j < a.window || j < a.sinks); }

// Row of the keys (elements / D) that position j of a sequence has; -1: none.
__device__ __forceinline__ int64_t keyRow(const CacheArgs &c, int seq, int begin, int count, int head, int j) {
    if (c.pages) return cacheRow(c, seq, head, j);
    return (uint32_t)j < (uint32_t)count ? (int64_t)(begin + j) * c.KVH + head : -1;
}

// One row by one wave, key by key: a lane has the scores of one key of 64, then four of the result's elements.  A value is only touched where
// the row sees its position, so what other positions hold, NaN and infinity among it, cannot come in.  Leaves in the lanes the elements lane + 64 e of
// sum_j w_j v_j, and the maximum and the sum, of positions [from, to).
// q: D floats of LDS, the row's query.
template <bool Q8>
__device__ void attendRow(const AttentionArgs &a, const float *q, int seq, int begin, int count, int head, int pos, int from, int to, float *o, float *m, float *l) {
    const CacheArgs &c = a.c;
    const int lane = threadIdx.x & 63, D = c.D;
    float most = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = 0.0f;
    for (int base = from; base < to; base += 64) {
        const int j = base + lane;
        int64_t row = -1;
        if (j < to && sees(a, pos, j)) row = keyRow(c, seq, begin, count, head, j);
        float s = -INFINITY, vs = 1.0f;
        if (row >= 0) {
            float dot = 0.0f;
            if constexpr (Q8) {
                const int8_t *k = (const int8_t *)a.key + row * D;
                for (int d = 0; d < D; d += 16) {
                    const v4i w = *(const v4i *)(k + d);
#pragma unroll
                    for (int i = 0; i < 16; i++) dot = fmaf((float)(int8_t)(w[i >> 2] >> (8 * (i & 3))), q[d + i], dot);
                }
                dot *= a.key_scales[row];
                vs = a.value_scales[row];
            } else {
                const uint16_t *k = (const uint16_t *)a.key + row * D;
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
        if (seen == 0) continue;
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
            const int64_t r = ((int64_t)__builtin_amdgcn_readlane((int)(row >> 32), t) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)row, t);
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
    }
    *m = most;
    *l = sum;
}

// A wave a row and query head.
template <bool Q8>
__global__ __launch_bounds__(256) void attention_rows(AttentionArgs a) {
    __shared__ float q[4][kMaxHeadDim];
    const CacheArgs &c = a.c;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    const int row = (int)(item / a.H), h = (int)(item % a.H);
    if (row >= c.T) return;
    const RowPlace p = placeOf(c, c.starts, row);
    if (p.seq < 0) return;
    const uint16_t *query = a.query + ((int64_t)row * a.H + h) * c.D;
    for (int d = lane; d < c.D; d += 64) q[wave][d] = __uint_as_float((uint32_t)query[d] << 16);
    __builtin_amdgcn_wave_barrier();
    __threadfence_block();
    float o[4], m, l;
    const int end = min(p.pos + 1, c.pages ? c.capacity : p.count);
    attendRow<Q8>(a, q[wave], p.seq, p.begin, p.count, h / a.G, p.pos, 0, end, o, &m, &l);
    uint16_t *out = a.out + ((int64_t)row * a.H + h) * c.D;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int d = lane + 64 * e;
        if (d < c.D) out[d] = bf16Bits(l == 0.0f ? 0.0f : o[e] / l);
    }
}

static hipError_t checkAttention(const AttentionArgs &a) {
    const CacheArgs &c = a.c;
    if (c.T < 1 || c.S < 1 || c.KVH < 1 || c.D < 16 || c.D > kMaxHeadDim || c.D % 16 != 0 || a.G < 1 || a.H != a.G * c.KVH) return hipErrorInvalidValue;
    if ((int64_t)c.T * a.H >= (1LL << 31) || a.window < 0 || a.sinks < 0) return hipErrorInvalidValue;
    if (!c.starts || !a.query || !a.out || !a.key || !a.value || !c.lengths != !c.pages || !a.key_scales != !a.value_scales) return hipErrorInvalidValue;
    if (((uintptr_t)a.query | (uintptr_t)a.out | (uintptr_t)a.key | (uintptr_t)a.value) & 15) return hipErrorInvalidValue;
    if (c.pages) {
        if (c.P < 1 || c.NP < 1 || c.PS < 1 || (int64_t)c.P * c.PS != c.capacity || (int64_t)c.NP * c.KVH * c.PS >= (1LL << 31)) return hipErrorInvalidValue;
    } else if (a.key_scales) {
        return hipErrorInvalidValue;
    }
    if (a.work_bytes < attentionWorkspaceBytes(c.T, c.S, a.H, c.KVH, c.D, c.pages ? c.capacity : c.T)) return hipErrorInvalidValue;
    return hipSuccess;
}

hipError_t launchAttention(const AttentionArgs &a, const LaunchCtx &ctx) {
    if (hipError_t e = checkAttention(a)) return e;
    const int64_t items = (int64_t)a.c.T * a.H;
    const dim3 grid((unsigned)((items + 3) / 4));
    if (a.key_scales) THIP_ENQUEUE(ctx, kernelLabel("attention_rows", {1}), attention_rows<true>, grid, dim3(256), 0, a);
    else THIP_ENQUEUE(ctx, kernelLabel("attention_rows", {0}), attention_rows<false>, grid, dim3(256), 0, a);
    return ctx.name ? hipSuccess : hipGetLastError();
}

}  // namespace thip
