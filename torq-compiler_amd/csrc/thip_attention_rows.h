// Device side of the packed rows and of the paged cache: whose a row is, at which position it stands, and where a position lies.
#pragma once

#include "thip_attention.h"
#include "thip_kernels_common.h"

namespace thip {

struct RowPlace {
    int seq;    // -1: no sequence's
    int begin;  // its first row
    int count;  // its rows
    int pos;    // the row's position
};

// Rows [begin, begin + count) of sequence s; kept inside the tensors whatever row_starts holds.
__device__ __forceinline__ void rowsOf(const CacheArgs &c, const int32_t *starts, int s, int *begin, int *count) {
    const int b = min(max(starts[s], 0), c.T), e = min(max(starts[s + 1], b), c.T);
    *begin = b;
    *count = e - b;
}

// The position of a sequence's row 0 (rows stand behind one another).
__device__ __forceinline__ int firstPosition(const CacheArgs &c, int s, int count) { return c.lengths ? max(c.lengths[s], 0) - count : 0; }

// The last sequence that starts at or before the row (those without rows start where the next one does), if the row is one of its.
__device__ __forceinline__ RowPlace placeOf(const CacheArgs &c, const int32_t *starts, int row) {
    int lo = 0, hi = c.S;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= row) lo = mid;
        else hi = mid;
    }
    RowPlace p{-1, 0, 0, 0};
    rowsOf(c, starts, lo, &p.begin, &p.count);
    if (row < p.begin || row >= p.begin + p.count) return p;
    p.seq = lo;
    p.pos = firstPosition(c, lo, p.count) + (row - p.begin);
    return p;
}

// Where a position lies: the table's entry is asked for, and the row of the cache that it makes (-1: none) is taken when that has come.
// Without branches; a position that is none is asked for as the first.
struct PageAsk {
    uint32_t page, slot;
    bool in;
};
__device__ __forceinline__ PageAsk askPage(const CacheArgs &c, int seq, int pos, int length) {
    PageAsk q;
    q.in = ((uint32_t)pos < (uint32_t)c.capacity) & (pos < length);
    const uint32_t p = q.in ? (uint32_t)pos : 0u, entry = fastDiv(p, c.ps);
    q.slot = p - entry * c.ps.d;
    q.page = (uint32_t)c.pages[(int64_t)seq * c.P + entry];
    return q;
}
__device__ __forceinline__ int rowOf(const CacheArgs &c, const PageAsk &q, int head) {
    return (q.in & (q.page < (uint32_t)c.NP)) ? (int)((q.page * (uint32_t)c.KVH + (uint32_t)head) * (uint32_t)c.PS + q.slot) : -1;
}
__device__ __forceinline__ int cacheRow(const CacheArgs &c, int seq, int head, int pos) { return rowOf(c, askPage(c, seq, pos, 0x7fffffff), head); }

// The starts in LDS, where they fit `most` sequences; every thread of the workgroup calls it.
__device__ __forceinline__ const int32_t *holdStarts(const CacheArgs &c, int32_t *held, int most) {
    if (c.S > most) return c.starts;
    for (int i = threadIdx.x; i <= c.S; i += blockDim.x) held[i] = c.starts[i];
    __syncthreads();
    return held;
}

}  // namespace thip
