// The norms behind a block and before the next one, and the residual between them (thip_lm_norm).
//
// h = r + s g u, u = x or x c(x) (p + o); out = h c(h) (w + o), c(x) = 1 / sqrt(mean(x^2) + eps).  One pass: a row lies in the registers of its lanes, in
// pieces of eight elements that are neighbours, so each operand is read once and each result written once.  Bound by memory (4096 rows of 4096, the residual in 32
// bits, 201 MB: 40 us, 5.1 TB/s), or, of few rows, by the launch and the chain from the loads over the sums to the stores (8 rows of 1152: 2.9 us).  Of the longest rows
// a lane's part does not quite fit: above 16384 elements, where an operand has 32 bits or the length is no multiple of 8, 6 to 42 of its registers lie in memory, above 8192
// with both of these 10 (100 rows, a residual and both norms: of 32768 10.0 us, of 30001 14.7; with the residual in 32 bits 22.2 and 24.7).
#include "thip_layer.h"
#include "thip_kernels_common.h"
#include "thip_lanes.h"

namespace thip {

// How rows are cut into pieces: all of them whole; or the last one not, which then is the row's last eight elements, loaded in one as the others are, of which
// the first count nothing (taken one by one where the row ends, each operand's with a wait, 8 rows of 1001 took 5.9 us, so 3.3); or a row of less than eight.
enum RowKind { kWholeRows, kRaggedRows, kShortRows };

// Eight elements as they lie in memory: in `lo`, those of 32 bits in `hi` too.  Rows of odd lengths start anywhere: 16 bytes at any alignment.
struct Piece {
    v4i lo, hi;
};
template <RowKind KIND>
__device__ __forceinline__ Piece fetch(const void *row, int column, int N, int bytes) {
    Piece r{v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}};
    if (column >= N) return r;
    if constexpr (KIND == kShortRows) {
#pragma unroll
        for (int i = 0; i < 7; i++) {
            if (i >= N) continue;
            if (bytes == 2) r.lo[i >> 1] |= (int)((uint32_t)((const uint16_t *)row)[i] << (16 * (i & 1)));
            else (i < 4 ? r.lo : r.hi)[i & 3] = ((const int *)row)[i];
        }
    } else {
        const int8_t *const p = (const int8_t *)row + (int64_t)(KIND == kWholeRows ? column : min(column, N - 8)) * bytes;
        r.lo = ((const UnalignedV4 *)p)->v;
        if (bytes == 4) r.hi = ((const UnalignedV4 *)(p + 16))->v;
    }
    return r;
}
__device__ __forceinline__ void unpack(const Piece &r, int bytes, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t w = (uint32_t)r.lo[i >> 1], half = i & 1 ? w & 0xffff0000u : w << 16;
        x[i] = __uint_as_float(bytes == 2 ? half : (uint32_t)(i < 4 ? r.lo[i & 3] : r.hi[i & 3]));
    }
}
// Which of a piece's elements are its own: [from, to).
template <RowKind KIND>
struct Own {
    int from, to;
    __device__ __forceinline__ Own(int column, int N) {
        from = KIND == kRaggedRows ? max(column + 8 - N, 0) : 0;
        to = column >= N ? 0 : KIND == kShortRows ? N : 8;
    }
    __device__ __forceinline__ bool all() const { return from == 0 && to == 8; }
    __device__ __forceinline__ bool has(int i) const { return (KIND != kRaggedRows || i >= from) && i < to; }
};
template <RowKind KIND>
__device__ __forceinline__ void store(void *row, int column, const Own<KIND> &own, int bytes, const float (&x)[8]) {
    int8_t *const p = (int8_t *)row + (int64_t)(column - own.from) * bytes;
    if (bytes == 2) {
        const v4i w{packBf16(x[0], x[1]), packBf16(x[2], x[3]), packBf16(x[4], x[5]), packBf16(x[6], x[7])};
        if (own.all()) {
            ((UnalignedV4 *)p)->v = w;
        } else if constexpr (KIND != kWholeRows) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (own.has(i)) ((uint16_t *)p)[i] = (uint16_t)((uint32_t)w[i >> 1] >> (16 * (i & 1)));
            }
        }
    } else if (own.all()) {
        ((UnalignedV4 *)p)->v = v4i{(int)__float_as_uint(x[0]), (int)__float_as_uint(x[1]), (int)__float_as_uint(x[2]), (int)__float_as_uint(x[3])};
        ((UnalignedV4 *)(p + 16))->v = v4i{(int)__float_as_uint(x[4]), (int)__float_as_uint(x[5]), (int)__float_as_uint(x[6]), (int)__float_as_uint(x[7])};
    } else if constexpr (KIND != kWholeRows) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (own.has(i)) ((float *)p)[i] = x[i];
        }
    }
}
template <RowKind KIND>
__device__ __forceinline__ void clearOthers(const Own<KIND> &own, float (&x)[8]) {
    if (KIND == kWholeRows && own.all()) return;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = own.has(i) ? x[i] : 0.0f;
}

// Sum over the LANES lanes of a row, the same in each; a row of more than a wave has its workgroup to itself.  room: LDS, a float for each wave, used once.
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

// 1 / sqrt(mean(x^2) + eps).  Where the squares would leave 32 bits, they are taken of x by a power of two.  Small x becomes that, and the factor is that of this: what small x
// is can pass 32 bits.  Large x stays, as its small elements would leave 32 bits by it, and the factor is scaled back (2^-128 at least, of which 32 bits hold 21).
template <int LANES, int EACH>
__device__ __forceinline__ float factorOf(float (&x)[EACH][8], float count, float eps, float *room) {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < EACH; e++) {
#pragma unroll
        for (int i = 0; i < 8; i++) sum = fmaf(x[e][i], x[e][i], sum);
    }
    float mean = rowSum<LANES>(sum, room) / count + eps;
    const bool odd = !(mean >= 0x1p-100f && mean <= 0x1p120f);
    float back = 1.0f;
    if (__builtin_expect(__any(odd), 0)) {  // the waves of a row have the same mean; factors of 1, as a selection takes registers (256 lanes of two pieces: 131, so 125)
        const bool large = odd && mean > 1.0f;
        const float up = odd && !large ? 0x1p100f : 1.0f;
        back = large ? 0x1p-100f : 1.0f;
        sum = 0.0f;
#pragma unroll
        for (int e = 0; e < EACH; e++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[e][i] *= up;
                const float y = x[e][i] * back;
                sum = fmaf(y, y, sum);
            }
        }
        mean = rowSum<LANES>(sum, room + 16) / count + eps * up * up * back * back;
    }
    return __builtin_amdgcn_rsqf(mean) * back;
}

// LANES lanes a row, EACH pieces a lane: LANES apart, so that what a wave loads lies together.  All operands are asked for at once while registers last.
// WIDE: some operand is of 32 bits.  The others' code has none of that: a short launch waits for its instructions too (8 rows of 1152: 3.2 us by the wide code, 2.9 by the
// other; 777 of 2305 9.1 and 6.7).
template <int LANES, int EACH, RowKind KIND, bool WIDE>
__global__ __launch_bounds__(LANES > 64 ? LANES : 256) void norm(NormArgs a, int turns) {
    if constexpr (!WIDE) a.residual_bytes = a.sum_bytes = a.weight_bytes = a.post_bytes = 2;
    constexpr int ROWS = LANES > 64 ? 1 : 256 / LANES;
    constexpr bool AHEAD = EACH <= 3, ROW_AHEAD = AHEAD || !WIDE;
    __shared__ float room[LANES > 64 ? 64 : 1];
    const int lane = threadIdx.x % LANES;
    const float elements = (float)a.N;
    auto columnOf = [&](int e) { return (lane + LANES * e) * 8; };
    auto ownOf = [&](int e) { return Own<KIND>(columnOf(e), a.N); };
    auto part = [&](const void *from, int64_t at, int e, int bytes) { return fetch<KIND>((const int8_t *)from + at * bytes, columnOf(e), a.N, bytes); };
    Piece post[EACH], weight[EACH];
    for (int t = 0; t < turns; t++) {
        int64_t row = (((int64_t)t * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * ROWS + threadIdx.x / LANES;
        const bool idle = row >= a.rows;  // takes part in the sums of its wave, and stores nothing
        if (idle) row = a.rows - 1;
        const int64_t begin = row * a.N;
        Piece in[EACH], residual[EACH], gate[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) in[e] = part(a.input, begin, e, 2);
        float rowGate = 1.0f;
        if (a.gate && !a.gate_column) rowGate = __uint_as_float((uint32_t)a.gate[row * a.gate_row] << 16);
        auto fetchRow = [&](int e) {
            if (a.residual) residual[e] = part(a.residual, begin, e, a.residual_bytes);
            if (a.gate && a.gate_column) gate[e] = part(a.gate, row * a.gate_row, e, 2);
        };
        if constexpr (ROW_AHEAD) {
#pragma unroll
            for (int e = 0; e < EACH; e++) fetchRow(e);
        }
        if (AHEAD && t == 0) {
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                if (a.post_weight) post[e] = part(a.post_weight, 0, e, a.post_bytes);
                if (a.out) weight[e] = part(a.weight, 0, e, a.weight_bytes);
            }
        }
        float x[EACH][8];
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            unpack(in[e], 2, x[e]);
            clearOthers(ownOf(e), x[e]);
        }
        if (a.post_weight) {
            const float factor = factorOf<LANES, EACH>(x, elements, a.eps, room);
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                float w[8];
                if constexpr (!AHEAD) post[e] = part(a.post_weight, 0, e, a.post_bytes);
                unpack(post[e], a.post_bytes, w);
#pragma unroll
                for (int i = 0; i < 8; i++) x[e][i] = x[e][i] * factor * (w[i] + a.offset);
            }
        }
        if (a.residual || a.gate || a.post_weight || a.scale != 1.0f) {
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                float r[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if constexpr (!ROW_AHEAD) fetchRow(e);
                if (a.gate) {
                    float g[8];
                    if (a.gate_column) unpack(gate[e], 2, g);
#pragma unroll
                    for (int i = 0; i < 8; i++) x[e][i] *= a.gate_column ? g[i] : rowGate;
                }
                if (a.residual) unpack(residual[e], a.residual_bytes, r);
#pragma unroll
                for (int i = 0; i < 8; i++) x[e][i] = fmaf(x[e][i], a.scale, r[i]);
                clearOthers(ownOf(e), x[e]);
            }
        }
        if (a.sum && !idle) {
#pragma unroll
            for (int e = 0; e < EACH; e++) store<KIND>((int8_t *)a.sum + begin * a.sum_bytes, columnOf(e), ownOf(e), a.sum_bytes, x[e]);
        }
        if (!a.out) continue;
        const float factor = factorOf<LANES, EACH>(x, elements, a.eps, room + 32);
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            float w[8];
            if constexpr (!AHEAD) weight[e] = part(a.weight, 0, e, a.weight_bytes);
            unpack(weight[e], a.weight_bytes, w);
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = x[e][i] * factor * (w[i] + a.offset);
            if (!idle) store<KIND>(a.out + begin, columnOf(e), ownOf(e), 2, w);
        }
    }
}

hipError_t launchNorm(const NormArgs &a, const LaunchCtx &ctx) {
    if (a.rows < 1 || a.N < 1 || a.N > kMaxNormRow || !a.input || (!a.sum && !a.out) || !a.out != !a.weight) return hipErrorInvalidValue;
    const auto size = [](const void *p, int bytes) { return !p || bytes == 2 || bytes == 4; };
    if (!size(a.residual, a.residual_bytes) || !size(a.sum, a.sum_bytes) || !size(a.weight, a.weight_bytes) || !size(a.post_weight, a.post_bytes)) return hipErrorInvalidValue;
    bool fits = true;
    const auto enqueueWidth = [&](auto lanes, auto each, auto kind, auto wideCode) {
        constexpr int LANES = decltype(lanes)::value, EACH = decltype(each)::value, THREADS = LANES > 64 ? LANES : 256, ROWS = THREADS / LANES;
        constexpr RowKind KIND = decltype(kind)::value;
        constexpr bool WIDE = decltype(wideCode)::value;
        // rows of a wave at most go by several a workgroup, with the weights in its registers, where there would be more than 4096 workgroups (131072 rows of 128
        // 12.5 us, a workgroup for each of its rows 13.3, 2048 workgroups 12.9).  A long row has a workgroup, and
        // many of them a grid of two dimensions, as one holds 2^32 threads.
        const int64_t groups = ((int64_t)a.rows - 1) / ROWS + 1;
        const int turns = LANES > 64 ? 1 : (int)((groups - 1) / 4096 + 1);
        const int64_t blocks = (groups - 1) / turns + 1, high = (blocks - 1) / 32768 + 1;
        fits = high <= 65535;
        if (!fits) return;
        const dim3 grid((unsigned)((blocks - 1) / high + 1), (unsigned)high);
        THIP_ENQUEUE(ctx, kernelLabel("norm", {LANES, EACH, KIND, WIDE}), (norm<LANES, EACH, KIND, WIDE>), grid, dim3(THREADS), 0, a, turns);
    };
    using std::integral_constant;
    const bool wideRows = (a.residual && a.residual_bytes == 4) || (a.sum && a.sum_bytes == 4) || (a.weight && a.weight_bytes == 4) || (a.post_weight && a.post_bytes == 4);
    const auto enqueueKind = [&](auto lanes, auto each, auto kind) {
        if (wideRows) enqueueWidth(lanes, each, kind, std::true_type{});
        else enqueueWidth(lanes, each, kind, std::false_type{});
    };
    const auto enqueue = [&](auto lanes, auto each) {
        if (a.N % 8 == 0) enqueueKind(lanes, each, integral_constant<RowKind, kWholeRows>{});
        else enqueueKind(lanes, each, integral_constant<RowKind, kRaggedRows>{});
    };
    const int pieces = (a.N - 1) / 8 + 1;
    // Lanes that are a row's, and pieces of each (us).  Few rows want many lanes: 8 rows of 1152 by 256 lanes of one piece 3.2, by 64 of three 4.9; 8 of 4096 by 512
    // of one 3.5, by 256 of two 3.9.  Many want few idle ones and no barrier: 8192 of 1152 by 64 of three 16.9, by 256 of one 19.7; 16384 of 1024 by 64 of
    // two 23.6, by 128 of one 24.8; 777 of 2305 by 256 of two 6.7, by 512 of one 7.2.
    const bool many = a.rows >= 2048;
    if (a.N < 8) enqueueKind(integral_constant<int, 16>{}, integral_constant<int, 1>{}, integral_constant<RowKind, kShortRows>{});
    else if (pieces <= 16) enqueue(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (pieces <= 32) enqueue(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    else if (pieces <= 64) enqueue(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (pieces <= 128 && many) enqueue(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (pieces <= 192 && many) enqueue(integral_constant<int, 64>{}, integral_constant<int, 3>{});
    else if (pieces <= 128) enqueue(integral_constant<int, 128>{}, integral_constant<int, 1>{});
    else if (pieces <= 256) enqueue(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (pieces <= 512 && a.rows > 512) enqueue(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else if (pieces <= 512) enqueue(integral_constant<int, 512>{}, integral_constant<int, 1>{});
    else if (pieces <= 1024) enqueue(integral_constant<int, 512>{}, integral_constant<int, 2>{});
    else if (pieces <= 2048) enqueue(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
    else enqueue(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
    if (!fits) return hipErrorInvalidValue;
    return ctx.name ? hipSuccess : hipGetLastError();
}

}  // namespace thip
