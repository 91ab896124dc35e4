// What a decoder's layer has around its linears and its attention: arguments of the launches of norms and rotary positions.
#pragma once

#include "thip_descriptor.h"
#include "thip_kernels.h"

namespace thip {

constexpr int kMaxNormRow = 32768;       // elements of a row
constexpr float kMaxRotaryStep = 16.0f;  // radians a position

struct NormArgs {
    const uint16_t *input;                // [rows][N]
    const void *residual;                 // null: 0
    const uint16_t *gate;                 // null: 1
    const void *post_weight, *weight;     // null: no norm of the input; of the sum
    void *sum;                            // null: not stored
    uint16_t *out;                        // null: not made
    int32_t rows, N;
    int32_t residual_bytes, sum_bytes, weight_bytes, post_bytes;  // of an element
    int32_t gate_row, gate_column;        // elements of gate from one row, one column to the next
    float eps, offset, scale;
};
hipError_t launchNorm(const NormArgs &a, const LaunchCtx &ctx);

struct RotaryArgs {
    const uint16_t *query, *key;          // [T][H][D], [T][KVH][D]; KVH 0: no key
    uint16_t *query_out, *key_out;
    const int32_t *positions;             // [axes][T]
    const RotaryTurn *turns;              // [pairs]
    int32_t T, H, KVH, D, pairs, interleaved;
};
hipError_t launchRotary(const RotaryArgs &a, const LaunchCtx &ctx);

}  // namespace thip
