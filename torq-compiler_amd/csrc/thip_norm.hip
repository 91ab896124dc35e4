// The norms behind a block and before the next one, and the residual between them (thip_lm_norm).
//
// h = r + s g u, u = x or x c(x) (p + o); out = h c(h) (w + o), c(x) = 1 / sqrt(mean(x^2) + eps).  One pass: a row lies in the registers of its lanes, in
// pieces of eight elements that are neighbours, so each operand is read once and each result written once.  Bound by memory.
#include "thip_layer.h"
#include "thip_kernels_common.h"
#include "thip_lanes.h"

namespace thip {

// Eight elements from `at` on, the first `count` of them where there are fewer, zeros behind these.  Rows of odd lengths start anywhere: loads of 16
// bytes at any alignment.
__device__ __forceinline__ void unpackBf16(v4i w, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float((uint32_t)w[i] << 16);
        x[2 * i + 1] = __uint_as_float((uint32_t)w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void loadPiece(const void *from, int64_t at, int bytes, int count, float (&x)[8]) {
    if (bytes == 2) {
        const uint16_t *p = (const uint16_t *)from + at;
        if (count >= 8) {
            unpackBf16(((const UnalignedV4 *)p)->v, x);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = i < count ? __uint_as_float((uint32_t)p[i] << 16) : 0.0f;
        }
    } else {
        const float *p = (const float *)from + at;
        if (count >= 8) {
            const v4i lo = ((const UnalignedV4 *)p)->v, hi = ((const UnalignedV4 *)(p + 4))->v;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[i] = __uint_as_float((uint32_t)lo[i]);
                x[4 + i] = __uint_as_float((uint32_t)hi[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = i < count ? p[i] : 0.0f;
        }
    }
}
__device__ __forceinline__ void storePiece(void *to, int64_t at, int bytes, int count, const float (&x)[8]) {
    if (bytes == 2) {
        uint16_t *p = (uint16_t *)to + at;
        const v4i w{packBf16(x[0], x[1]), packBf16(x[2], x[3]), packBf16(x[4], x[5]), packBf16(x[6], x[7])};
        if (count >= 8) {
            ((UnalignedV4 *)p)->v = w;
        } else {
#pragma unroll
            for (int i = 0; i < 7; i++) {
                if (i < count) p[i] = (uint16_t)((uint32_t)w[i >> 1] >> (16 * (i & 1)));
            }
        }
    } else {
        float *p = (float *)to + at;
        if (count >= 8) {
            ((UnalignedV4 *)p)->v = v4i{(int)__float_as_uint(x[0]), (int)__float_as_uint(x[1]), (int)__float_as_uint(x[2]), (int)__float_as_uint(x[3])};
            ((UnalignedV4 *)(p + 4))->v = v4i{(int)__float_as_uint(x[4]), (int)__float_as_uint(x[5]), (int)__float_as_uint(x[6]), (int)__float_as_uint(x[7])};
        } else {
#pragma unroll
            for (int i = 0; i < 7; i++) {
                if (i < count) p[i] = x[i];
            }
        }
    }
}

// Sum over the LANES lanes of a row, the same in each.  room: LDS, a float for each wave, used once.
template <int LANES>
__device__ __forceinline__ float rowSum(float v, float *room) {
    v = overLanes<16>(v, [](float x, float y) { return x + y; });
    if constexpr (LANES >= 32) v = sumOverSixteens(v);
    if constexpr (LANES >= 64) v = sumOverHalves(v);
    if constexpr (LANES > 64) {
        if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = v;
        __syncthreads();
        v = room[0];
#pragma unroll
        for (int w = 1; w < LANES / 64; w++) v += room[w];
    }
    return v;
}

// x / sqrt(mean(x^2) + eps) = (x by) inverse.  by is 1 but where the squares would leave 32 bits: then they are taken of scaled values.
struct RowScale {
    float by, inverse;
};
template <int LANES, int EACH>
__device__ __forceinline__ RowScale scaleOf(const float (&x)[EACH][8], int N, float eps, float *room) {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < EACH; e++) {
#pragma unroll
        for (int i = 0; i < 8; i++) sum = fmaf(x[e][i], x[e][i], sum);
    }
    float mean = rowSum<LANES>(sum, room) / (float)N + eps, by = 1.0f;
    const bool odd = !(mean >= 0x1p-100f && mean <= 0x1p120f);
    if (__any(odd)) {  // rows of more than a wave: their waves have the same mean
        by = !odd ? 1.0f : mean > 1.0f ? 0x1p-100f : 0x1p100f;
        sum = 0.0f;
#pragma unroll
        for (int e = 0; e < EACH; e++) {
#pragma unroll
            for (int i = 0; i < 8; i++) sum = fmaf(x[e][i] * by, x[e][i] * by, sum);
        }
        mean = rowSum<LANES>(sum, room + 16) / (float)N + eps * by * by;
    }
    return {by, __builtin_amdgcn_rsqf(mean)};
}

// LANES lanes a row, EACH pieces a lane: LANES apart, so that what a wave loads lies together.
template <int LANES, int EACH>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void norm(NormArgs a) {
    constexpr int ROWS = LANES > 256 ? 1 : 256 / LANES;
    __shared__ float room[LANES > 64 ? 64 : 1];
    const int lane = threadIdx.x % LANES;
    int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
    const bool idle = row >= a.rows;  // takes part in the sums of its wave, and stores nothing
    if (idle) row = a.rows - 1;
    const int64_t begin = row * a.N;
    float x[EACH][8];
    int count[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int column = (lane + LANES * e) * 8;
        count[e] = min(a.N - column, 8);
        loadPiece(a.input, begin + column, 2, count[e], x[e]);
    }
    if (a.post_weight) {
        const RowScale s = scaleOf<LANES, EACH>(x, a.N, a.eps, room);
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            float w[8];
            loadPiece(a.post_weight, (lane + LANES * e) * 8, a.post_bytes, count[e], w);
#pragma unroll
            for (int i = 0; i < 8; i++) x[e][i] = x[e][i] * s.by * s.inverse * (w[i] + a.offset);
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int column = (lane + LANES * e) * 8;
        if (a.gate) {
            float g[8];
            const int64_t at = row * a.gate_row;
            if (a.gate_column) {
                loadPiece(a.gate, at + column, 2, count[e], g);
            } else {
                const float one = __uint_as_float((uint32_t)a.gate[at] << 16);
#pragma unroll
                for (int i = 0; i < 8; i++) g[i] = one;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) x[e][i] *= g[i];
        }
        float r[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (a.residual) loadPiece(a.residual, begin + column, a.residual_bytes, count[e], r);
#pragma unroll
        for (int i = 0; i < 8; i++) x[e][i] = i < count[e] ? fmaf(x[e][i], a.scale, r[i]) : 0.0f;
        if (a.sum && !idle) storePiece(a.sum, begin + column, a.sum_bytes, count[e], x[e]);
    }
    if (!a.out) return;
    const RowScale s = scaleOf<LANES, EACH>(x, a.N, a.eps, room + 32);
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int column = (lane + LANES * e) * 8;
        float w[8];
        loadPiece(a.weight, column, a.weight_bytes, count[e], w);
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = x[e][i] * s.by * s.inverse * (w[i] + a.offset);
        if (!idle) storePiece(a.out, begin + column, 2, count[e], w);
    }
}

hipError_t launchNorm(const NormArgs &a, const LaunchCtx &ctx) {
    if (a.rows < 1 || a.N < 1 || a.N > kMaxNormRow || !a.input || (!a.sum && !a.out) || !a.out != !a.weight) return hipErrorInvalidValue;
    const auto size = [](const void *p, int bytes) { return !p || bytes == 2 || bytes == 4; };
    if (!size(a.residual, a.residual_bytes) || !size(a.sum, a.sum_bytes) || !size(a.weight, a.weight_bytes) || !size(a.post_weight, a.post_bytes)) return hipErrorInvalidValue;
    const auto enqueue = [&](auto lanes, auto each) {
        constexpr int LANES = decltype(lanes)::value, EACH = decltype(each)::value, THREADS = LANES > 256 ? LANES : 256, ROWS = THREADS / LANES;
        const dim3 grid((unsigned)(((int64_t)a.rows - 1) / ROWS + 1));
        THIP_ENQUEUE(ctx, kernelLabel("norm", {LANES, EACH}), (norm<LANES, EACH>), grid, dim3(THREADS), 0, a);
    };
    using std::integral_constant;
    const int pieces = (a.N - 1) / 8 + 1;
    if (pieces <= 16) enqueue(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (pieces <= 32) enqueue(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    else if (pieces <= 64) enqueue(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (pieces <= 256) enqueue(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (pieces <= 512) enqueue(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else if (pieces <= 1024) enqueue(integral_constant<int, 256>{}, integral_constant<int, 4>{});
    else if (pieces <= 2048) enqueue(integral_constant<int, 256>{}, integral_constant<int, 8>{});
    else enqueue(integral_constant<int, 1024>{}, integral_constant<int, 8>{});
    return ctx.name ? hipSuccess : hipGetLastError();
}

}  // namespace thip
