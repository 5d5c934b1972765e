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

// sigmoid(g) and 1 - sigmoid(g), each to a few fp32 roundings of itself: with
// u = exp(-|g|) they are 1 / (1 + u) and u / (1 + u), in the order that g's sign
// says. u is 2^t by the hardware's exponential, t = -|g| log2(e) rounded, times
// 2^(what t's rounding left out) as 1 + that times ln 2. Past 150, where u is 0 in
// fp32, |g| counts as 150 (infinities too); a NaN stays one.
HELIX_DEV void gate(float g, float& open, float& shut) {
    constexpr float kLog2e = 1.44269504f, kRest = 1.92596299e-8f, kLn2 = 0.693147181f;
    const float x = fabsf(g) > 150.0f ? 150.0f : fabsf(g);
    const float t = -x * kLog2e;
    const float rest = fmaf(-x, kRest, fmaf(-x, kLog2e, -t));
    float u = __builtin_amdgcn_exp2f(t);
    u = fmaf(u, rest * kLn2, u);
    const float r = __builtin_amdgcn_rcpf(1.0f + u);
    const float s = u * r;
    open = g < 0.0f ? s : r;
    shut = g < 0.0f ? r : s;
}

// Four neighbouring elements as they are stored: two registers of 16-bit types,
// four of fp32.
template <typename T> struct Raw4 { typedef u32x2 type; };
template <> struct Raw4<float> { typedef u32x4 type; };
// A pair of elements with these bits.
template <typename T>
constexpr unsigned inf_bits = __is_same(T, float) ? 0x7f800000u : __is_same(T, _Float16) ? 0x7c007c00u : 0x7f807f80u;

template <typename T>
HELIX_DEV void widen4(typename Raw4<T>::type w, float (&o)[4]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = as_f32(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const unsigned x = w[i];
            o[2 * i] = io_f32<T>((unsigned short)(x & 0xffffu));
            o[2 * i + 1] = io_f32<T>((unsigned short)(x >> 16));
        }
    }
}
template <typename T>
HELIX_DEV unsigned narrow2(float a, float b) {
    typedef T pair __attribute__((ext_vector_type(2)));
    const pair v = {(T)a, (T)b};
    return __builtin_bit_cast(unsigned, v);
}
template <typename T>
HELIX_DEV typename Raw4<T>::type narrow4(const float (&v)[4]) {
    if constexpr (sizeof(T) == 4) return u32x4{as_u32(v[0]), as_u32(v[1]), as_u32(v[2]), as_u32(v[3])};
    else return u32x2{narrow2<T>(v[0], v[1]), narrow2<T>(v[2], v[3])};
}

// Four elements at byte offset voff of a resource: one access where VEC, else the
// first `own` of them one by one. What is out of the resource's range reads as 0
// and is not written.
template <typename T, bool VEC>
HELIX_DEV typename Raw4<T>::type buf_load4(helix_rsrc r, int voff, int own) {
    typename Raw4<T>::type w;
    if constexpr (VEC) {
        if constexpr (sizeof(T) == 4) w = __builtin_amdgcn_raw_buffer_load_b128(r, voff, 0, 0);
        else w = __builtin_amdgcn_raw_buffer_load_b64(r, voff, 0, 0);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = __builtin_amdgcn_raw_buffer_load_b32(r, i < own ? voff + 4 * i : (int)0x80000000, 0, 0);
    } else {
        unsigned e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            e[i] = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(r, i < own ? voff + 2 * i : (int)0x80000000, 0, 0);
        w[0] = e[0] | e[1] << 16;
        w[1] = e[2] | e[3] << 16;
    }
    return w;
}
template <typename T, bool VEC, int AUX = 0>
HELIX_DEV void buf_store4(helix_rsrc r, const float (&v)[4], int voff, int own) {
    if constexpr (VEC) {
        if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b128(narrow4<T>(v), r, voff, 0, AUX);
        else __builtin_amdgcn_raw_buffer_store_b64(narrow4<T>(v), r, voff, 0, AUX);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) io_store<T, AUX>(r, v[i], i < own ? voff + (int)sizeof(T) * i : (int)0x80000000, 0);
    }
}

// Eight neighbouring elements as they are stored, at byte offset voff.
template <typename T> struct Raw8 { u32x4 w[sizeof(T) / 2]; };
template <typename T>
HELIX_DEV Raw8<T> buf_load8(helix_rsrc r, int voff) {
    Raw8<T> o;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) o.w[i] = __builtin_amdgcn_raw_buffer_load_b128(r, voff + 16 * i, 0, 0);
    return o;
}
template <typename T>
HELIX_DEV float at8(const Raw8<T>& v, int i) {
    if constexpr (sizeof(T) == 4) {
        return as_f32(v.w[i >> 2][i & 3]);
    } else {
        const unsigned x = v.w[0][i >> 1];
        return io_f32<T>((unsigned short)(i & 1 ? x >> 16 : x & 0xffffu));
    }
}
template <typename T>
HELIX_DEV void buf_store8(helix_rsrc r, const float (&v)[8], int voff) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            __builtin_amdgcn_raw_buffer_store_b128(
                u32x4{as_u32(v[4 * i]), as_u32(v[4 * i + 1]), as_u32(v[4 * i + 2]), as_u32(v[4 * i + 3])}, r, voff + 16 * i, 0, 0);
    } else {
        __builtin_amdgcn_raw_buffer_store_b128(
            u32x4{narrow2<T>(v[0], v[1]), narrow2<T>(v[2], v[3]), narrow2<T>(v[4], v[5]), narrow2<T>(v[6], v[7])}, r, voff, 0, 0);
    }
}

// The largest over each sixteen lanes, by moves within a row of lanes; all have it.
template <int CTRL>
HELIX_DEV float max_dpp(float v) {
    return fmaxf(v, as_f32((unsigned)__builtin_amdgcn_update_dpp(0, (int)as_u32(v), CTRL, 0xf, 0xf, true)));
}
HELIX_DEV float row16_max(float v) {
    v = max_dpp<0xb1>(v);    // lane ^ 1
    v = max_dpp<0x4e>(v);    // lane ^ 2
    v = max_dpp<0x141>(v);   // mirrored in eight
    return max_dpp<0x140>(v);   // mirrored in sixteen
}

#endif
