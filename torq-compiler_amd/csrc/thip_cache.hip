// Rows of keys and values to and from a paged cache (thip_lm_cache_write, thip_lm_cache_read).
#include "thip_attention.h"
#include "thip_attention_rows.h"
#include "thip_kernels_common.h"

namespace thip {

// Starts that a workgroup keeps in LDS; of more sequences each row's is looked up where they lie.
constexpr int kStartsInLds = 1024;

// a = max(max |x|, 2^-100) of a row: below that its elements are next to nothing, and 127 / a and a / 127 stay normal numbers.
__device__ __forceinline__ float rowUnit(uint32_t magnitude) { return fmaxf(__uint_as_float(magnitude << 16), 0x1p-100f); }

// A row is D / 8 pieces of 8 elements, each a lane's, 2^LOG lanes a row (those behind its last piece idle); a thread has U rows of
// the T * KVH, a workgroup's 256 >> LOG rows apart.  Memory bound: what a thread waits for is a chain of four (its
// sequence's start, the table's entry, the row, and for a write nothing more), so the rows of a thread overlap and their data
// is asked for before the chain is walked.
//
// Q8: the largest magnitude is taken on the bits (a bf16's magnitude orders as an integer does, with infinities and NaNs above all else)
// by shuffles among the row's lanes, and each element costs one multiply, one rint and one conversion.
template <bool Q8, int LOG, int U>
__global__ __launch_bounds__(256) void cache_write(CacheRowsArgs a) {
    __shared__ int32_t held[kStartsInLds + 1];
    const bool values = blockIdx.y != 0;
    const int piece = threadIdx.x & ((1 << LOG) - 1), pieces = a.c.D >> 3;
    const int64_t rows = (int64_t)a.c.T * a.c.KVH, first = (int64_t)blockIdx.x * (256 >> LOG) * U + (threadIdx.x >> LOG);
    const uint16_t *src = values ? a.value : a.key;
    v4i data[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t row = first + (int64_t)u * (256 >> LOG);
        data[u] = v4i{0, 0, 0, 0};
        if (row < rows && piece < pieces) data[u] = streamLoad<v4i>(src + row * a.c.D + piece * 8);
    }
    const int32_t *starts = holdStarts(a.c, held, kStartsInLds);
    int to[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t row = first + (int64_t)u * (256 >> LOG);
        to[u] = -1;
        if (row < rows) {
            const int token = (int)fastDiv((uint32_t)row, a.kvh);
            const RowPlace p = placeOf(a.c, starts, token);
            if (p.seq >= 0) to[u] = cacheRow(a.c, p.seq, (int)((uint32_t)row - (uint32_t)token * a.kvh.d), p.pos);
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        if constexpr (Q8) {
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t w = (uint32_t)data[u][i];
                most = max(most, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
            }
#pragma unroll
            for (int step = 1; step < (1 << LOG); step *= 2) most = max(most, (uint32_t)__shfl_xor((int)most, step));
            if (to[u] < 0 || piece >= pieces) continue;
            const bool finite = most < 0x7f80u;
            const float unit = rowUnit(finite ? most : 0u), inverse = 127.0f / unit;
            uint32_t q[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t w = (uint32_t)data[u][i];
                const int32_t lo = finite ? (int32_t)rintf(__uint_as_float(w << 16) * inverse) : 0;
                const int32_t hi = finite ? (int32_t)rintf(__uint_as_float(w & 0xffff0000u) * inverse) : 0;
                q[i >> 1] |= (((uint32_t)lo & 0xffu) | (((uint32_t)hi & 0xffu) << 8)) << (16 * (i & 1));
            }
            int8_t *cache = (int8_t *)(values ? a.value_cache : a.key_cache) + (int64_t)to[u] * a.c.D + piece * 8;
            *(v2i *)cache = v2i{(int)q[0], (int)q[1]};
            if (piece == 0) (values ? a.value_scales : a.key_scales)[to[u]] = finite ? unit / 127.0f : __uint_as_float(0x7fc00000u);
        } else {
            if (to[u] < 0 || piece >= pieces) continue;
            uint16_t *cache = (uint16_t *)(values ? a.value_cache : a.key_cache) + (int64_t)to[u] * a.c.D + piece * 8;
            *(v4i *)cache = data[u];
        }
    }
}

// The way back.  A piece of 8 elements of the row that is written is a lane's; values from int8 are products of two numbers that
// fp32 holds, rounded once to 32 bits and once to bf16, as the definition says.
template <bool Q8, int LOG, int U>
__global__ __launch_bounds__(256) void cache_read(CacheRowsArgs a) {
    __shared__ int32_t held[kStartsInLds + 1];
    const bool values = blockIdx.y != 0;
    const int piece = threadIdx.x & ((1 << LOG) - 1), pieces = a.c.D >> 3;
    const int64_t rows = (int64_t)a.c.T * a.c.KVH, first = (int64_t)blockIdx.x * (256 >> LOG) * U + (threadIdx.x >> LOG);
    uint16_t *dst = values ? a.value : a.key;
    const int32_t *starts = holdStarts(a.c, held, kStartsInLds);
    int from[U];
    bool there[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t row = first + (int64_t)u * (256 >> LOG);
        from[u] = -1;
        there[u] = false;
        if (row < rows && piece < pieces) {
            const int token = (int)fastDiv((uint32_t)row, a.kvh);
            const RowPlace p = placeOf(a.c, starts, token);
            there[u] = p.seq >= 0;
            if (there[u]) from[u] = cacheRow(a.c, p.seq, (int)((uint32_t)row - (uint32_t)token * a.kvh.d), p.pos);
        }
    }
    if constexpr (Q8) {
        v2i q[U];
        float scale[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            q[u] = v2i{0, 0};
            scale[u] = 0.0f;
            if (from[u] < 0) continue;
            q[u] = streamLoad<v2i>((const int8_t *)(values ? a.value_cache : a.key_cache) + (int64_t)from[u] * a.c.D + piece * 8);
            scale[u] = (values ? a.value_scales : a.key_scales)[from[u]];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (!there[u]) continue;
            v4i out;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int w = q[u][i >> 1] >> (16 * (i & 1));
                const float lo = (float)(int8_t)w * scale[u], hi = (float)(int8_t)(w >> 8) * scale[u];
                out[i] = __builtin_bit_cast(int, __builtin_convertvector((v2f){lo, hi}, v2bf));
            }
            streamStore(dst + (first + (int64_t)u * (256 >> LOG)) * a.c.D + piece * 8, out);
        }
    } else {
        v4i data[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            data[u] = v4i{0, 0, 0, 0};
            if (from[u] >= 0) data[u] = streamLoad<v4i>((const uint16_t *)(values ? a.value_cache : a.key_cache) + (int64_t)from[u] * a.c.D + piece * 8);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (there[u]) streamStore(dst + (first + (int64_t)u * (256 >> LOG)) * a.c.D + piece * 8, data[u]);
        }
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

// Lanes of a row: the smallest power of two that has one for every piece of 8 elements.
static int lanesLog(int D) {
    int log = 1;
    while ((8 << log) < D) log++;
    return log;
}

template <int U, typename F>
static void byLanes(int log, F &&f) {
    switch (log) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 3: f(std::integral_constant<int, 3>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    default: f(std::integral_constant<int, 5>{}); break;
    }
}

template <int U>
static void enqueueRows(const CacheRowsArgs &a, bool write, const LaunchCtx &ctx) {
    byLanes<U>(lanesLog(a.c.D), [&](auto log) {
        constexpr int LOG = decltype(log)::value;
        const int64_t rows = (int64_t)a.c.T * a.c.KVH, perBlock = (int64_t)(256 >> LOG) * U;
        const dim3 grid((unsigned)((rows + perBlock - 1) / perBlock), 2);
        const bool q8 = a.key_scales != nullptr;
        const std::string label = kernelLabel(write ? "cache_write" : "cache_read", {q8, LOG, U});
        if (write && q8) THIP_ENQUEUE(ctx, label, (cache_write<true, LOG, U>), grid, dim3(256), 0, a);
        else if (write) THIP_ENQUEUE(ctx, label, (cache_write<false, LOG, U>), grid, dim3(256), 0, a);
        else if (q8) THIP_ENQUEUE(ctx, label, (cache_read<true, LOG, U>), grid, dim3(256), 0, a);
        else THIP_ENQUEUE(ctx, label, (cache_read<false, LOG, U>), grid, dim3(256), 0, a);
    });
}

hipError_t launchCacheWrite(const CacheRowsArgs &a, const LaunchCtx &ctx) {
    if (hipError_t e = checkRows(a)) return e;
    enqueueRows<1>(a, true, ctx);
    return ctx.name ? hipSuccess : hipGetLastError();
}

hipError_t launchCacheRead(const CacheRowsArgs &a, const LaunchCtx &ctx) {
    if (hipError_t e = checkRows(a)) return e;
    enqueueRows<1>(a, false, ctx);
    return ctx.name ? hipSuccess : hipGetLastError();
}

}  // namespace thip
