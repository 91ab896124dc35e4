// Rotary positions of a query's and a key's heads (thip_lm_rotary).
//
// (a, b) -> (a cos t - b sin t, b cos t + a sin t), t the position times the pair's step.  A workgroup has a few tokens: their sines and cosines once, in LDS, then
// all of their heads by them, 16 elements a thread at a time.  Bound by memory (8192 tokens, 40 heads of 128, 168 MB: 32.9 us, 5.1 TB/s), of few tokens by the launch
// (16 tokens of 5 heads of 256: 2.3 us, with the first elements fetched behind the angles 3.9).
#include "thip_layer.h"
#include "thip_kernels_common.h"
#include "thip_lanes.h"

namespace thip {

constexpr int kMaxTokens = 8;  // of a workgroup
constexpr int kMaxPairs = 128;

// Cosine and sine of `turn` / 2^32 turns.  The nearest quarter is taken off in whole numbers; what is left is within 45 degrees, where the series, to the powers
// kept here, are off by 2.5e-8 (cosine: x^10 / 10!) and 2e-9.
__device__ __forceinline__ v2f cosSin(uint32_t turn) {
    const uint32_t quarter = (turn + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(turn - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
    const float xx = x * x;
    float s = fmaf(xx, 2.7557319e-6f, -1.9841270e-4f);  // 1 / 9!, -1 / 7!
    s = fmaf(xx, s, 8.3333333e-3f);
    s = fmaf(xx, s, -1.6666667e-1f);
    s = fmaf(xx * x, s, x);
    float c = fmaf(xx, 2.4801587e-5f, -1.3888889e-3f);  // 1 / 8!, -1 / 6!
    c = fmaf(xx, c, 4.1666667e-2f);
    c = fmaf(xx, c, -0.5f);
    c = fmaf(xx, c, 1.0f);
    const float cc = quarter & 1 ? s : c, ss = quarter & 1 ? c : s;
    return v2f{(quarter == 1 || quarter == 2) ? -cc : cc, quarter & 2 ? -ss : ss};
}

template <bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary(RotaryArgs a, int tokens, int pieces, FastDiv byPieces, FastDiv byHeads, FastDiv byPairs) {
    __shared__ float cosines[kMaxTokens * kMaxPairs], sines[kMaxTokens * kMaxPairs];
    const int first = (int)blockIdx.x * tokens, here = min(tokens, a.T - first), heads = a.H + a.KVH, turned = a.pairs >> 3, all = here * heads * pieces;
    // A piece: 16 elements of a head, eight pairs, or those behind the pairs as they are.
    struct Held {
        v4i x, y;
        uint16_t *x_to, *y_to;
        int angle;  // of its first pair in LDS; -1: none
    };
    auto fetch = [&](int i) {
        Held h;
        const int row = (int)fastDiv((uint32_t)i, byPieces), piece = i - row * pieces, token = (int)fastDiv((uint32_t)row, byHeads), head = row - token * heads;
        const bool isKey = head >= a.H, turns = piece < turned;
        const int64_t at = (isKey ? (int64_t)(first + token) * a.KVH + head - a.H : (int64_t)(first + token) * a.H + head) * a.D;
        const int lo = INTERLEAVED || !turns ? 16 * piece : 8 * piece, hi = INTERLEAVED || !turns ? lo + 8 : a.pairs + 8 * piece;
        const uint16_t *const from = (isKey ? a.key : a.query) + at;
        h.x = *(const v4i *)(from + lo);
        h.y = *(const v4i *)(from + hi);
        h.x_to = (isKey ? a.key_out : a.query_out) + at + lo;
        h.y_to = h.x_to + (hi - lo);
        h.angle = turns ? token * a.pairs + 8 * piece : -1;
        return h;
    };
    // the first pieces are on their way while the angles are made, each next one while one is turned
    Held next;
    if ((int)threadIdx.x < all) next = fetch(threadIdx.x);
    for (int i = threadIdx.x; i < here * a.pairs; i += 256) {
        const int token = (int)fastDiv((uint32_t)i, byPairs), pair = i - token * a.pairs;
        const RotaryTurn t = a.turns[pair];
        const v2f cs = cosSin((uint32_t)(((uint64_t)(int64_t)a.positions[(int64_t)t.axis * a.T + first + token] * t.step) >> 32));
        cosines[i] = cs[0];
        sines[i] = cs[1];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < all; i += 256) {
        Held h = next;
        if (i + 256 < all) next = fetch(i + 256);
        if (h.angle >= 0) {
            const float *const c = cosines + h.angle, *const s = sines + h.angle;
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const uint32_t w = (uint32_t)(k < 4 ? h.x[k] : h.y[k - 4]);
                    const float p = __uint_as_float(w << 16), q = __uint_as_float(w & 0xffff0000u);
                    (k < 4 ? h.x : h.y)[k & 3] = packBf16(p * c[k] - q * s[k], q * c[k] + p * s[k]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float p0 = __uint_as_float((uint32_t)h.x[k] << 16), p1 = __uint_as_float((uint32_t)h.x[k] & 0xffff0000u);
                    const float q0 = __uint_as_float((uint32_t)h.y[k] << 16), q1 = __uint_as_float((uint32_t)h.y[k] & 0xffff0000u);
                    h.x[k] = packBf16(p0 * c[2 * k] - q0 * s[2 * k], p1 * c[2 * k + 1] - q1 * s[2 * k + 1]);
                    h.y[k] = packBf16(q0 * c[2 * k] + p0 * s[2 * k], q1 * c[2 * k + 1] + p1 * s[2 * k + 1]);
                }
            }
        }
        *(v4i *)h.x_to = h.x;
        *(v4i *)h.y_to = h.y;
    }
}

hipError_t launchRotary(const RotaryArgs &a, const LaunchCtx &ctx) {
    if (a.T < 1 || a.H < 1 || a.KVH < 0 || a.D < 16 || a.D > 2 * kMaxPairs || a.D % 16 != 0 || a.pairs < 8 || a.pairs % 8 != 0 || 2 * a.pairs > a.D) return hipErrorInvalidValue;
    if (a.T >= 1 << 27 || (int64_t)a.T * a.H >= (1LL << 31) || (int64_t)a.T * a.KVH >= (1LL << 31) || (int64_t)(a.H + a.KVH) * a.D >= (1LL << 26)) return hipErrorInvalidValue;
    if (!a.query || !a.query_out || !a.positions || !a.turns || (a.KVH > 0) != (a.key != nullptr) || !a.key != !a.key_out) return hipErrorInvalidValue;
    if (((uintptr_t)a.query | (uintptr_t)a.key | (uintptr_t)a.query_out | (uintptr_t)a.key_out) & 15) return hipErrorInvalidValue;
    const bool inPlace = a.query == a.query_out && a.key == a.key_out;
    const int pieces = inPlace ? a.pairs / 8 : a.D / 16, heads = a.H + a.KVH;
    // A workgroup has about four pieces a thread where there are tokens for 512 of them (8192 tokens, 40 heads of 128: 32.9 us; two a thread 33.8, eight 35.5),
    // else fewer (777 tokens, 32 heads of 80: 3.5 us by 389 workgroups, 3.9 by 195).
    int tokens = 1024 / (pieces * heads);
    const int share = (a.T - 1) / 512 + 1;
    tokens = tokens < share ? tokens : share;
    tokens = tokens < 1 ? 1 : tokens > kMaxTokens ? kMaxTokens : tokens;
    const dim3 grid((unsigned)((a.T - 1) / tokens + 1));
    const FastDiv byPieces = makeFastDiv((uint32_t)pieces), byHeads = makeFastDiv((uint32_t)heads), byPairs = makeFastDiv((uint32_t)a.pairs);
    if (a.interleaved) THIP_ENQUEUE(ctx, kernelLabel("rotary", {1}), rotary<true>, grid, dim3(256), 0, a, tokens, pieces, byPieces, byHeads, byPairs);
    else THIP_ENQUEUE(ctx, kernelLabel("rotary", {0}), rotary<false>, grid, dim3(256), 0, a, tokens, pieces, byPieces, byHeads, byPairs);
    return ctx.name ? hipSuccess : hipGetLastError();
}

}  // namespace thip
