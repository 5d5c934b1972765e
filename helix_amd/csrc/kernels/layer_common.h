// layer_common.h -- device helpers of the layer operators.
//
// Storage types are float, _Float16 and __bf16: widened to fp32 when they are
// loaded, rounded to nearest even once when they are stored.
#ifndef HELIX_LAYER_COMMON_H
#define HELIX_LAYER_COMMON_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "helix_common.h"
#include "layer_params.h"

// The sum, or largest, over the 64 lanes of a wave; every lane has it.
HELIX_DEV float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}
HELIX_DEV float wave_max(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}

// Exponent byte of the least power of two s >= 2^-126 with top <= 448 s. With
// top = 1.m 2^E and 448 = 1.75 2^8 that is 2^(E - 8), or the next where 1.m >
// 1.75: adding 0x1fffff to the bits carries into the exponent just there. top is
// no NaN; infinity gives 2^120.
HELIX_DEV int block_exponent(float top) {
    const int e = (int)((as_u32(top) + 0x1fffffu) >> 23) - 8;
    return e < 1 ? 1 : e;
}
// 2^(127 - e), the reciprocal of the scale of exponent byte e (1 .. 247).
HELIX_DEV float exponent_recip(int e) { return as_f32((unsigned)(254 - e) << 23); }

// sigmoid(g) and 1 - sigmoid(g), both to full relative precision: with
// u = exp(-|g|) they are 1 / (1 + u) and u / (1 + u), in the order that g's sign
// says. u underflows to 0 where the smaller one does; g = +-inf gives 1 and 0.
HELIX_DEV void gate(float g, float& open, float& shut) {
    const float u = expf(-fabsf(g));
    const float r = 1.0f / (1.0f + u);
    const float s = u * r;
    open = g >= 0.0f ? r : s;
    shut = g >= 0.0f ? s : r;
    if (g != g) open = shut = g;
}

#endif
