// rms_norm.hip -- root-mean-square norm with the residual's addition, into the
// storage type or 8 bits with scales, and its backward pass (helix_layer.h).
#include "layer_common.h"

namespace {

constexpr int NORM_THREADS = 256;

// Sum over a workgroup; every thread has it. red: one float per wave.
HELIX_DEV float group_sum(float v, float* red) {
    v = wave_sum(v);
    if (lane_id() == 0) red[wave_id()] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < NORM_THREADS / 64; ++w) s += red[w];
    return s;
}

template <typename T>
HELIX_DEV float weight_at(const void* w, int w_f32, int c) {
    return w_f32 ? static_cast<const float*>(w)[c] : (float)static_cast<const T*>(w)[c];
}

// One workgroup per row, which is read twice (the second time from the caches).
// A wave handles a block of 128 channels, lane l its channels l and l + 64.
template <typename T>
__device__ void norm_row(const HelixNormParams& p) {
    __shared__ float red[NORM_THREADS / 64];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
    const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.ld_residual : nullptr;
    auto at = [&](int c) { return (float)x[c] + (r ? (float)r[c] : 0.0f); };
    float rstd = 1.0f;
    if (p.weight) {
        float ss = 0.0f;
        for (int c = threadIdx.x; c < p.dim; c += NORM_THREADS) {
            const float v = at(c);
            ss += v * v;
        }
        rstd = 1.0f / sqrtf(group_sum(ss, red) / (float)p.dim + p.eps);
        if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
    }
    for (int b = wave_id(); b * HELIX_BLOCK < p.dim; b += NORM_THREADS / 64) {
        float out[2];
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int c = b * HELIX_BLOCK + 64 * e + lane_id();
            out[e] = 0.0f;
            if (c < p.dim) {
                const float v = at(c);
                if (p.h) static_cast<T*>(p.h)[row * p.ld_h + c] = (T)v;
                out[e] = p.weight ? v * rstd * weight_at<T>(p.weight, p.w_f32, c) : v;
                if (p.y) static_cast<T*>(p.y)[row * p.ld_y + c] = (T)out[e];
            }
            top = fmaxf(top, fabsf(out[e]));
        }
        if (p.y) continue;
        const int ex = block_exponent(wave_max(top));
        const float inv = exponent_recip(ex);
        if (lane_id() == 0) p.scale[row * p.ld_scale + b] = (uint8_t)ex;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int c = b * HELIX_BLOCK + 64 * e + lane_id();
            if (c < p.dim) p.q[row * p.ld_q + c] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(out[e] * inv, 0.0f, 0, false);
        }
    }
}

// dx: one workgroup per row, read twice.
template <typename T>
__device__ void norm_bwd_row(const HelixNormBwdParams& p) {
    __shared__ float red[NORM_THREADS / 64];
    const long long row = blockIdx.x;
    const T* dy = static_cast<const T*>(p.dy) + row * p.ld_dy;
    const T* h = static_cast<const T*>(p.h) + row * p.ld_h;
    const T* dh = p.dh ? static_cast<const T*>(p.dh) + row * p.ld_dh : nullptr;
    T* dx = static_cast<T*>(p.dx) + row * p.ld_dx;
    const float rstd = p.rstd[row];
    float dot = 0.0f;
    for (int c = threadIdx.x; c < p.dim; c += NORM_THREADS)
        dot += (float)dy[c] * weight_at<T>(p.weight, p.w_f32, c) * ((float)h[c] * rstd);
    const float mean = group_sum(dot, red) / (float)p.dim;
    for (int c = threadIdx.x; c < p.dim; c += NORM_THREADS) {
        const float n = (float)h[c] * rstd;
        const float g = rstd * ((float)dy[c] * weight_at<T>(p.weight, p.w_f32, c) - n * mean);
        dx[c] = (T)(g + (dh ? (float)dh[c] : 0.0f));
    }
}

// dweight: the sum of a part's rows, one thread per channel; then the parts'.
template <typename T>
__device__ void norm_dw_part(const HelixNormBwdParams& p) {
    const int c = blockIdx.x * NORM_THREADS + threadIdx.x;
    if (c >= p.dim) return;
    const long long lo = blockIdx.y * p.part_rows, hi = min(p.rows, lo + p.part_rows);
    float s = 0.0f;
    for (long long row = lo; row < hi; ++row)
        s += (float)static_cast<const T*>(p.dy)[row * p.ld_dy + c] *
             ((float)static_cast<const T*>(p.h)[row * p.ld_h + c] * p.rstd[row]);
    p.part[(long long)blockIdx.y * p.dim + c] = s;
}

}  // namespace

extern "C" __global__ __launch_bounds__(NORM_THREADS) void helix_norm_dw(HelixNormBwdParams p) {
    const int c = blockIdx.x * NORM_THREADS + threadIdx.x;
    if (c >= p.dim) return;
    float s = 0.0f;
    for (int i = 0; i < p.parts; ++i) s += p.part[(long long)i * p.dim + c];
    p.dweight[c] = s;
}

#define NORM_KERNELS(TAG, T)                                                                                  \
    extern "C" __global__ __launch_bounds__(NORM_THREADS) void helix_norm_##TAG(HelixNormParams p) {         \
        norm_row<T>(p);                                                                                       \
    }                                                                                                         \
    extern "C" __global__ __launch_bounds__(NORM_THREADS) void helix_norm_bwd_##TAG(HelixNormBwdParams p) {  \
        norm_bwd_row<T>(p);                                                                                   \
    }                                                                                                         \
    extern "C" __global__ __launch_bounds__(NORM_THREADS) void helix_norm_dw_part_##TAG(HelixNormBwdParams p) { \
        norm_dw_part<T>(p);                                                                                   \
    }
NORM_KERNELS(f32, float)
NORM_KERNELS(f16, _Float16)
NORM_KERNELS(bf16, __bf16)
