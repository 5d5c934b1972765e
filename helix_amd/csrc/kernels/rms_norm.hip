// rms_norm.hip -- root-mean-square norm with the residual's addition, into the
// storage type or 8 bits with scales, and its backward pass (helix_layer.h).
//
// Memory binds all of it, so every tensor is read and written once: a row stays in
// registers between its sum and its outputs. A lane holds eight neighbouring channels
// of every chunk of 512 (16-byte accesses; sixteen lanes are a block of 128), and a row
// is a wave's (W = 1: no barrier) or a workgroup's of four waves (W = 4), which divide
// the registers of a wide row, or of one of few.
// Accesses past a row's end are out of the resource's range: they read zeros, which add
// nothing to a sum or a largest magnitude, and write nothing.
//
// Rows start anywhere (8192 x 1001 in bf16 12.7 us, 8192 x 1024 10.9; 2871 x 5183 of
// f32 27, element by element 38). Those wider than what registers hold, 16384, go
// through the forms below that read a row twice, element by element, for widths that no
// layer here has: 512 rows of bf16 of 16384 take 7.3 us forward and 22 back, of 16896 38
// and 58, of 32768 94 and 108 (0.7 and 0.9 TB/s).
//
// 8192 x 2048 of bf16 with a residual into 8 bits: 21 us, 118 MB at 5.6 TB/s; 2871 x 5184
// of f32 21 us, 5.7 TB/s; backward of 32768 x 2560 of bf16 138 us, 4.9 TB/s, where a copy
// of 4 GiB reaches 4.65 (tensors that fit in the 256 MiB of cache go faster than those
// that do not).
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

// A row's resource: `dim` elements of T.
template <typename T>
HELIX_DEV helix_rsrc row_rsrc(const void* base, long long row, long long ld, int dim) {
    return make_rsrc_u(static_cast<const T*>(base) + row * ld, (unsigned)dim * (unsigned)sizeof(T));
}

// A row's eight channels from c on, at any address. A resource's range is checked word by
// word, so a word that an odd last channel of 16 bits has half of is left out of it, and
// that channel is moved by itself (Tail).
template <typename T>
HELIX_DEV helix_rsrc words_rsrc(const void* base, long long row, long long ld, int dim) {
    return make_rsrc_u(static_cast<const T*>(base) + row * ld, (unsigned)dim * (unsigned)sizeof(T) & ~3u);
}
template <typename T>
struct Tail {
    int last;      // the odd last channel, or -1
    __device__ explicit Tail(int dim) : last(sizeof(T) == 2 && (dim & 1) ? dim - 1 : -1) {}
    __device__ __forceinline__ unsigned load(const void* base, long long row, long long ld) const {
        if (sizeof(T) == 4 || last < 0) return 0;
        return reinterpret_cast<const uint16_t*>(base)[row * ld + last];
    }
    // The channel in the lane and chunk that hold it.
    __device__ __forceinline__ void put(unsigned x, Raw8<T>& v, int c) const {
        if (sizeof(T) == 4 || last < 0) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) v.w[0][i] = c + 2 * i == last ? x : v.w[0][i];
    }
    __device__ __forceinline__ void store(void* base, long long row, long long ld, const float (&v)[8], int c) const {
        if (sizeof(T) == 4 || last < 0) return;
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            if (c + i == last) static_cast<T*>(base)[row * ld + last] = (T)v[i];
    }
};
template <typename T, int NC>
HELIX_DEV void load_row(const void* base, long long row, long long ld, int dim, const int (&c)[NC], Raw8<T> (&o)[NC]) {
    const helix_rsrc r = words_rsrc<T>(base, row, ld, dim);
    const Tail<T> tail(dim);
#pragma unroll
    for (int j = 0; j < NC; ++j) o[j] = buf_load8<T>(r, c[j] * (int)sizeof(T));
    const unsigned x = tail.load(base, row, ld);
#pragma unroll
    for (int j = 0; j < NC; ++j) tail.put(x, o[j], c[j]);
}
template <typename T, int NC>
HELIX_DEV void store_row(void* base, long long row, long long ld, int dim, const int (&c)[NC], const float (&v)[NC][8]) {
    const helix_rsrc r = words_rsrc<T>(base, row, ld, dim);
    const Tail<T> tail(dim);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        buf_store8<T>(r, v[j], c[j] * (int)sizeof(T));
        tail.store(base, row, ld, v[j], c[j]);
    }
}

// The weights of a lane's channels in fp32.
template <typename T, int NC>
HELIX_DEV void load_weights(const void* w, int w_f32, int dim, const int (&c)[NC], float (&o)[NC][8]) {
    if (w_f32) {
        Raw8<float> v[NC];
        load_row<float>(w, 0, 0, dim, c, v);
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) o[j][i] = at8(v[j], i);
    } else {
        Raw8<T> v[NC];
        load_row<T>(w, 0, 0, dim, c, v);
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) o[j][i] = at8(v[j], i);
    }
}

// Sum over the row's waves.
template <int W>
HELIX_DEV float row_sum(float v, float* red) {
    if constexpr (W == 1) return wave_sum(v);
    else return group_sum(v, red);
}

template <typename T, int W, int NC>
__device__ void norm_rows(const HelixNormParams& p) {
    __shared__ float red[NORM_THREADS / 64];
    const int lane = lane_id(), wave = wave_uniform();
    const long long row = W == 1 ? (long long)blockIdx.x * 4 + wave : blockIdx.x;
    if (W == 1 && row >= p.rows) return;
    int c[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) c[j] = (W == 1 ? j : 4 * j + wave) * 512 + 8 * lane;
    Raw8<T> x[NC], r[NC];
    load_row<T>(p.x, row, p.ld_x, p.dim, c, x);
    if (p.residual) load_row<T>(p.residual, row, p.ld_residual, p.dim, c, r);
    float w[NC][8], v[NC][8];
    if (p.weight) load_weights<T>(p.weight, p.w_f32, p.dim, c, w);
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = at8(x[j], i);
    if (p.residual) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] += at8(r[j], i);
    }
    if (p.h) store_row<T>(p.h, row, p.ld_h, p.dim, c, v);
    if (p.weight) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += v[j][i] * v[j][i];
        const float rstd = 1.0f / sqrtf(row_sum<W>(ss, red) / (float)p.dim + p.eps);
        if (p.rstd && lane == 0 && (W == 1 || wave == 0)) p.rstd[row] = rstd;
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * rstd * w[j][i];
    }
    if (p.y) {
        store_row<T>(p.y, row, p.ld_y, p.dim, c, v);
        return;
    }
    const helix_rsrc rq = words_rsrc<uint8_t>(p.q, row, p.ld_q, p.dim);
    const helix_rsrc rs = row_rsrc<uint8_t>(p.scale, row, p.ld_scale, (p.dim + HELIX_BLOCK - 1) / HELIX_BLOCK);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[j][i]));
        const int e = block_exponent(row16_max(top));
        const float inv = exponent_recip(e);
        u32x2 q;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            int d = __builtin_amdgcn_cvt_pk_fp8_f32(v[j][4 * i] * inv, v[j][4 * i + 1] * inv, 0, false);
            q[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[j][4 * i + 2] * inv, v[j][4 * i + 3] * inv, d, true);
        }
        __builtin_amdgcn_raw_buffer_store_b64(q, rq, c[j], 0, 0);
        if (p.dim & 3) {   // the bytes of the last word
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c[j] + i >= (p.dim & ~3) && c[j] + i < p.dim) p.q[row * p.ld_q + c[j] + i] = (uint8_t)(q[i >> 2] >> (8 * (i & 3)));
        }
        __builtin_amdgcn_raw_buffer_store_b8((unsigned char)e, rs, lane & 15 ? (int)0x80000000 : c[j] >> 7, 0, 0);
    }
}

// dx, and dweight's sum over the rows of a part: a workgroup's, row by row in each of
// its waves (W = 1) or in all of them (W = 4). The waves' sums are added in their order.
template <typename T, int W, int NC>
__device__ void norm_bwd_rows(const HelixNormBwdParams& p) {
    __shared__ float red[2][NORM_THREADS / 64];
    __shared__ float sums[W == 1 ? 3 : 1][W == 1 ? NC * 512 : 1];
    const int lane = lane_id(), wave = wave_uniform();
    int c[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) c[j] = (W == 1 ? j : 4 * j + wave) * 512 + 8 * lane;
    float w[NC][8], dw[NC][8];
    load_weights<T>(p.weight, p.w_f32, p.dim, c, w);
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[j][i] = 0.0f;
    const long long first = blockIdx.x * p.part_rows, end = min(p.rows, first + p.part_rows);
    int turn = 0;
    for (long long row = first + (W == 1 ? wave : 0); row < end; row += W == 1 ? 4 : 1) {
        Raw8<T> dy[NC], h[NC], dh[NC];
        load_row<T>(p.dy, row, p.ld_dy, p.dim, c, dy);
        load_row<T>(p.h, row, p.ld_h, p.dim, c, h);
        if (p.dh) load_row<T>(p.dh, row, p.ld_dh, p.dim, c, dh);
        const float rstd = p.rstd[row];
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n = at8(h[j], i) * rstd, g = at8(dy[j], i);
                dot += g * w[j][i] * n;
                dw[j][i] += g * n;
            }
        // Two places in turn: a wave may be at the next row's sum while another reads this one's.
        const float mean = row_sum<W>(dot, red[turn]) / (float)p.dim;
        turn ^= 1;
        float o[NC][8];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n = at8(h[j], i) * rstd;
                o[j][i] = rstd * (at8(dy[j], i) * w[j][i] - n * mean);
            }
            if (p.dh) {
#pragma unroll
                for (int i = 0; i < 8; ++i) o[j][i] += at8(dh[j], i);
            }
        }
        store_row<T>(p.dx, row, p.ld_dx, p.dim, c, o);
    }
    if (!p.dweight) return;
    if constexpr (W == 1) {
        if (wave > 0) {
#pragma unroll
            for (int j = 0; j < NC; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[wave - 1][(j * 8 + i) * 64 + lane] = dw[j][i];
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int o = 0; o < 3; ++o) dw[j][i] += sums[o][(j * 8 + i) * 64 + lane];
    }
    store_row<float>(p.part, blockIdx.x, p.dim, p.dim, c, dw);
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

// dweight from the parts: 32 channels a workgroup, every 32nd part a half of a wave, eight
// loads at a time; the 32 sums are added in their order (512 parts of 2560 channels 5 us; 64 channels a
// workgroup and load by load 12).
extern "C" __global__ __launch_bounds__(1024) void helix_norm_dw(HelixNormBwdParams p) {
    __shared__ float sum[32][33];
    const int half = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < p.dim)
        for (int i = half; i < p.parts; i += 32 * 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = i + 32 * u < p.parts ? p.part[(i + 32LL * u) * p.dim + c] : 0.0f;
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
    sum[half][lane] = s;
    __syncthreads();
    if (half || c >= p.dim) return;
#pragma unroll
    for (int w = 1; w < 32; ++w) s += sum[w][lane];
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

#define NORM_FWD(TAG, T, KIND, W, NC)                                                                             \
    extern "C" __global__ __launch_bounds__(NORM_THREADS) void helix_norm_##TAG##_##KIND##NC(HelixNormParams p) { \
        norm_rows<T, W, NC>(p);                                                                                   \
    }
#define NORM_BWD(TAG, T, KIND, W, NC)                                                                                    \
    extern "C" __global__ __launch_bounds__(NORM_THREADS) void helix_norm_bwd_##TAG##_##KIND##NC(HelixNormBwdParams p) { \
        norm_bwd_rows<T, W, NC>(p);                                                                                      \
    }
#define NORM_ROWS(TAG, T)     \
    NORM_FWD(TAG, T, w, 1, 1) \
    NORM_FWD(TAG, T, w, 1, 2) \
    NORM_FWD(TAG, T, w, 1, 3) \
    NORM_FWD(TAG, T, w, 1, 4) \
    NORM_FWD(TAG, T, g, 4, 1) \
    NORM_FWD(TAG, T, g, 4, 2) \
    NORM_FWD(TAG, T, g, 4, 3) \
    NORM_FWD(TAG, T, g, 4, 4) \
    NORM_FWD(TAG, T, g, 4, 6) \
    NORM_FWD(TAG, T, g, 4, 8) \
    NORM_BWD(TAG, T, w, 1, 1) \
    NORM_BWD(TAG, T, w, 1, 2) \
    NORM_BWD(TAG, T, g, 4, 1) \
    NORM_BWD(TAG, T, g, 4, 2) \
    NORM_BWD(TAG, T, g, 4, 3) \
    NORM_BWD(TAG, T, g, 4, 4) \
    NORM_BWD(TAG, T, g, 4, 6) \
    NORM_BWD(TAG, T, g, 4, 8)
NORM_ROWS(f32, float)
NORM_ROWS(f16, _Float16)
NORM_ROWS(bf16, __bf16)
