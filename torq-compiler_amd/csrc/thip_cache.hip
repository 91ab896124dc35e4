// Rows of keys and values to and from a paged cache (thip_lm_cache_write, thip_lm_cache_read).
#include "thip_attention.h"
#include "thip_attention_rows.h"
#include "thip_kernels_common.h"

namespace thip {

// Starts that a workgroup keeps in LDS; of more sequences each row's is looked up where they lie.
constexpr int kStartsInLds = 1024;

// a = max(max |x|, 2^-100) of a row: below that its elements are next to nothing, and 127 / a and a / 127 stay normal numbers.
__device__ __forceinline__ float rowUnit(uint32_t magnitude) { return fmaxf(__uint_as_float(magnitude << 16), 0x1p-100f); }

// A wave has 2^rowsLog rows (a token's head) next to one another, keys and values: each lane looks up where one of them lies, then the rows go
// by, 64 >> LOG of them at a time, D / 8 pieces of 8 elements, each a lane's, 2^LOG lanes a row (those behind its last piece idle).
// Memory bound; what the work is cut for is that lookups (a chain of four loads: the starts, the length, the table's entry, the row) are few and
// overlap.  With every lane of a row looking up for itself the arithmetic of that took the time (four sequences of 8192 positions with
// eight heads of 128 read from int8, 164 MB: 49 us; so 30, 5.4 TB/s.  Five prompts of 12738 tokens together written as bf16, 104 MB:
// 19 us, 5.5 TB/s; 23 before).
constexpr int kBatch = 4;  // rows of a lane at most, all under way together

// Row of the cache that `row` of the T * KVH has; -1: its page is none; -2: no sequence's.
__device__ __forceinline__ int placeInCache(const CacheRowsArgs &a, const int32_t *starts, int64_t row) {
    if (row >= (int64_t)a.c.T * a.c.KVH) return -2;
    const int token = (int)fastDiv((uint32_t)row, a.kvh);
    const RowPlace p = placeOf(a.c, starts, token);
    return p.seq < 0 ? -2 : cacheRow(a.c, p.seq, (int)((uint32_t)row - (uint32_t)token * a.kvh.d), p.pos);
}

// One row's piece to the cache.  Q8: the largest magnitude is taken on the bits (a bf16's magnitude orders as an integer does, with infinities and
// NaNs above all else) by shuffles among the row's lanes, and each element costs one multiply, one rint and one conversion.
template <bool Q8, int LOG>
__device__ __forceinline__ void putRow(const CacheRowsArgs &a, v4i data, int to, int piece, void *cache, float *scales) {
    if constexpr (Q8) {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = (uint32_t)data[i];
            most = max(most, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
        }
#pragma unroll
        for (int step = 1; step < (1 << LOG); step *= 2) most = max(most, (uint32_t)__shfl_xor((int)most, step));
        if (to < 0 || piece >= a.c.D >> 3) return;
        const bool finite = most < 0x7f80u;
        const float unit = rowUnit(finite ? most : 0u), inverse = 127.0f / unit;
        uint32_t q[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = (uint32_t)data[i];
            const int32_t lo = finite ? (int32_t)rintf(__uint_as_float(w << 16) * inverse) : 0;
            const int32_t hi = finite ? (int32_t)rintf(__uint_as_float(w & 0xffff0000u) * inverse) : 0;
            q[i >> 1] |= (((uint32_t)lo & 0xffu) | (((uint32_t)hi & 0xffu) << 8)) << (16 * (i & 1));
        }
        *(v2i *)((int8_t *)cache + (int64_t)to * a.c.D + piece * 8) = v2i{(int)q[0], (int)q[1]};
        if (piece == 0) scales[to] = finite ? unit / 127.0f : __uint_as_float(0x7fc00000u);
    } else {
        if (to >= 0 && piece < a.c.D >> 3) *(v4i *)((uint16_t *)cache + (int64_t)to * a.c.D + piece * 8) = data;
    }
}

template <bool Q8, int LOG>
__global__ __launch_bounds__(256) void cache_write(CacheRowsArgs a, int rowsLog) {
    __shared__ int32_t held[kStartsInLds + 1];
    constexpr int EACH = 64 >> LOG;
    const int lane = threadIdx.x & 63, piece = lane & ((1 << LOG) - 1), mine = lane >> LOG, steps = (1 << rowsLog) / EACH;
    const int64_t rows = (int64_t)a.c.T * a.c.KVH, first = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) << rowsLog;
    const bool idle = piece >= a.c.D >> 3;
    v4i key[kBatch], value[kBatch];
    // before the chain of lookups is walked, and whatever the row is: a load behind a branch would be waited for behind it
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
        const int64_t row = first + min(u, steps - 1) * EACH + mine, at = (row < rows ? row : rows - 1) * a.c.D + (idle ? 0 : piece * 8);
        key[u] = streamLoad<v4i>(a.key + at);
        value[u] = streamLoad<v4i>(a.value + at);
    }
    if (idle) {
#pragma unroll
        for (int u = 0; u < kBatch; u++) key[u] = value[u] = v4i{0, 0, 0, 0};
    }
    const int32_t *starts = holdStarts(a.c, held, kStartsInLds);
    const int place = lane < 1 << rowsLog ? placeInCache(a, starts, first + lane) : -2;
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
        if (u >= steps) break;
        const int to = __shfl(place, u * EACH + mine);
        putRow<Q8, LOG>(a, key[u], to, piece, a.key_cache, a.key_scales);
        putRow<Q8, LOG>(a, value[u], to, piece, a.value_cache, a.value_scales);
    }
}

// Eight int8 times a scale: products of two numbers that fp32 holds, rounded once to 32 bits and once to bf16, as the definition says.
__device__ __forceinline__ v4i scaledRow(v2i q, float scale) {
    v4i out;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int w = q[i >> 1] >> (16 * (i & 1));
        const float lo = (float)(int8_t)w * scale, hi = (float)(int8_t)(w >> 8) * scale;
        out[i] = __builtin_bit_cast(int, __builtin_convertvector((v2f){lo, hi}, v2bf));
    }
    return out;
}

// The way back.
template <bool Q8, int LOG>
__global__ __launch_bounds__(256) void cache_read(CacheRowsArgs a, int rowsLog) {
    __shared__ int32_t held[kStartsInLds + 1];
    typedef std::conditional_t<Q8, v2i, v4i> Piece;
    constexpr int EACH = 64 >> LOG;
    const int lane = threadIdx.x & 63, piece = lane & ((1 << LOG) - 1), mine = lane >> LOG, steps = (1 << rowsLog) / EACH;
    const int64_t first = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) << rowsLog;
    const bool idle = piece >= a.c.D >> 3;
    const int32_t *starts = holdStarts(a.c, held, kStartsInLds);
    const int place = lane < 1 << rowsLog ? placeInCache(a, starts, first + lane) : -2;
    float keyScale = 0.0f, valueScale = 0.0f;
    if constexpr (Q8) {
        if (place >= 0) {
            keyScale = a.key_scales[place];
            valueScale = a.value_scales[place];
        }
    }
    const Piece *const keys = (const Piece *)a.key_cache + (idle ? 0 : piece), *const values = (const Piece *)a.value_cache + (idle ? 0 : piece);
    Piece key[kBatch], value[kBatch];
    int from[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; u++) {  // whatever the place is, as above
        from[u] = __shfl(place, min(u, steps - 1) * EACH + mine);
        const int64_t at = (int64_t)max(from[u], 0) * (a.c.D >> 3);
        key[u] = streamLoad<Piece>(keys + at);
        value[u] = streamLoad<Piece>(values + at);
    }
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
        if (u >= steps) break;
        const int64_t at = (first + u * EACH + mine) * a.c.D + piece * 8;
        v4i k, v;
        if constexpr (Q8) {
            k = scaledRow(key[u], __shfl(keyScale, u * EACH + mine));
            v = scaledRow(value[u], __shfl(valueScale, u * EACH + mine));
        } else {
            k = key[u];
            v = value[u];
        }
        if (from[u] < 0) k = v = v4i{0, 0, 0, 0};
        if (from[u] < -1 || idle) continue;
        *(v4i *)(a.key + at) = k;
        *(v4i *)(a.value + at) = v;
    }
}

static hipError_t checkRows(const CacheRowsArgs &a) {
    const CacheArgs &c = a.c;
    if (c.T < 1 || c.S < 1 || c.KVH < 1 || c.D < 16 || c.D > kMaxHeadDim || c.D % 16 != 0 || c.P < 1 || c.NP < 1 || c.PS < 1) return hipErrorInvalidValue;
    if ((int64_t)c.T * c.KVH >= (1LL << 31) || (int64_t)c.P * c.PS != c.capacity || (int64_t)c.NP * c.KVH * c.PS >= (1LL << 31)) return hipErrorInvalidValue;
    if (!c.starts || !c.lengths || !c.pages || !a.key || !a.value || !a.key_cache || !a.value_cache || !a.key_scales != !a.value_scales) return hipErrorInvalidValue;
    if (((uintptr_t)a.key | (uintptr_t)a.value | (uintptr_t)a.key_cache | (uintptr_t)a.value_cache) & 15) return hipErrorInvalidValue;
    return hipSuccess;
}

constexpr int64_t kEnoughWaves = 2048;  // two on each SIMD

// Lanes of a row: the smallest power of two that has one for every piece of 8 elements.
static int lanesLog(int D) {
    int log = 1;
    while ((8 << log) < D) log++;
    return log;
}

template <typename F>
static void byLanes(int log, F &&f) {
    switch (log) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 3: f(std::integral_constant<int, 3>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    default: f(std::integral_constant<int, 5>{}); break;
    }
}

static hipError_t enqueueRows(const CacheRowsArgs &a, bool write, const LaunchCtx &ctx) {
    byLanes(lanesLog(a.c.D), [&](auto log) {
        constexpr int LOG = decltype(log)::value;
        // rows of a wave: as many as are under way together while there are enough waves (32 x 1024 positions of one head of 256, read: 8.8 us, with two
        // rows a lane 9.9; two batches a wave: the 104 MB above 22 us for 19)
        const int64_t rows = (int64_t)a.c.T * a.c.KVH;
        int rowsLog = 6 - LOG;
        while (rowsLog < 8 - LOG && rowsLog < 6 && rows >> (rowsLog + 1) >= kEnoughWaves) rowsLog++;
        const dim3 grid((unsigned)(((rows - 1) >> (rowsLog + 2)) + 1));
        const bool q8 = a.key_scales != nullptr;
        const std::string label = kernelLabel(write ? "cache_write" : "cache_read", {q8, LOG});
        if (write && q8) THIP_ENQUEUE(ctx, label, (cache_write<true, LOG>), grid, dim3(256), 0, a, rowsLog);
        else if (write) THIP_ENQUEUE(ctx, label, (cache_write<false, LOG>), grid, dim3(256), 0, a, rowsLog);
        else if (q8) THIP_ENQUEUE(ctx, label, (cache_read<true, LOG>), grid, dim3(256), 0, a, rowsLog);
        else THIP_ENQUEUE(ctx, label, (cache_read<false, LOG>), grid, dim3(256), 0, a, rowsLog);
    });
    return ctx.name ? hipSuccess : hipGetLastError();
}

hipError_t launchCacheWrite(const CacheRowsArgs &a, const LaunchCtx &ctx) {
    if (hipError_t e = checkRows(a)) return e;
    return enqueueRows(a, true, ctx);
}

hipError_t launchCacheRead(const CacheRowsArgs &a, const LaunchCtx &ctx) {
    if (hipError_t e = checkRows(a)) return e;
    return enqueueRows(a, false, ctx);
}

}  // namespace thip
