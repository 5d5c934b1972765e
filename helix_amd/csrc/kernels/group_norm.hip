// group_norm.hip -- norm of the groups of a row's channels with an activation or a
// gate, into the storage type or 8 bits, and its backward pass (helix_layer.h).
//
// Memory binds it: x (and the gate) are read once and kept in registers between the
// two sums and the output. A group is LP lanes' (4 .. 64 of a wave, or a workgroup's
// 256), each with NC vectors of eight neighbours LP vectors apart; a wave holds 64 / LP
// groups, of one row or of several. Sums cross lanes by moves inside a row of sixteen
// lanes and by shuffles above; the variance is the mean square of x - mean, not a
// difference of sums. A last vector that the group's end cuts is read whole where the
// row goes on behind it, and is written in pieces of four, two and one.
//
// Measured: 8192 rows of 64 groups of 64 with a gate, bf16 into 8 bits, 168 MB in 40 us
// (4.2 TB/s, as a large copy of that share of writes); 2871 rows of 27 groups of 192 in
// fp32, 120 MB in 24 us; backward, 32768 rows of 80 groups of 64 with a gate, bf16,
// 1.7 GB in 370 us (4.6 TB/s). Kept from it, as slower: the next row's loads before this
// one's sums, tails read by element in the same instructions as whole vectors (492 us).
#include "layer_common.h"

namespace {

constexpr int GN_THREADS = 256;

// Weights or biases of a vector in fp32.
template <typename T>
HELIX_DEV void gn_weights(const void* w, int w_f32, int c, int n, float (&o)[8]) {
    if (w_f32) {
        const Raw8<float> v = load8_at<float>(static_cast<const float*>(w) + c, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = at8(v, i);
    } else {
        const Raw8<T> v = load8_at<T>(static_cast<const T*>(w) + c, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = at8(v, i);
    }
}

// The sum over LP neighbouring lanes; all of them have it. 256: over the workgroup,
// through red (one float per wave), which the next call does not use.
template <int LP>
HELIX_DEV float lanes_sum(float v, float* red) {
    if constexpr (LP >= 2) v = add_dpp<0xb1>(v);     // lane ^ 1
    if constexpr (LP >= 4) v = add_dpp<0x4e>(v);     // lane ^ 2
    if constexpr (LP >= 8) v = add_dpp<0x141>(v);    // mirrored in eight
    if constexpr (LP >= 16) v = add_dpp<0x140>(v);   // mirrored in sixteen
    if constexpr (LP >= 32) v += __shfl_xor(v, 16, 64);
    if constexpr (LP >= 64) v += __shfl_xor(v, 32, 64);
    if constexpr (LP == 256) {
        if (lane_id() == 0) red[wave_id()] = v;
        __syncthreads();
        v = (red[0] + red[1]) + (red[2] + red[3]);
    }
    return v;
}

// a(u) and a'(u).
HELIX_DEV void activation(int act, float u, float& a, float& slope) {
    if (act == 0) {
        a = u;
        slope = 1.0f;
        return;
    }
    float open, shut;
    gate(u, open, shut);
    if (act == 1) {
        a = u * open;
        slope = open + a * shut;
    } else {
        a = open;
        slope = open * shut;
    }
}
HELIX_DEV float activation(int act, float u) {
    float a, slope;
    activation(act, u, a, slope);
    return a;
}

HELIX_DEV void quantize8(const float (&v)[8], float inv, u32x2& q) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * inv, v[4 * i + 1] * inv, 0, false);
        q[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * inv, v[4 * i + 3] * inv, d, true);
    }
}

// Units (a row's group each) of a launch: below 2^31, the runtime sees to it. FP8: the
// groups line up with blocks of 128, which are then sixteen neighbouring lanes'.
template <typename T, int LP, int NC, bool FP8>
__device__ void group_norm(const HelixGroupNormParams& p) {
    __shared__ float red[2][GN_THREADS / 64];
    const unsigned unit = blockIdx.x * (GN_THREADS / LP) + threadIdx.x / LP;
    const unsigned row = unit / (unsigned)p.groups;
    const int g = (int)(unit - row * (unsigned)p.groups), l = threadIdx.x % LP;
    const bool here = row < p.rows;
    const int first = g * p.width;
    const T* x = static_cast<const T*>(p.x) + row * p.ld_x + first;
    const T* gt = static_cast<const T*>(p.gate) + row * p.ld_gate + first;
    Raw8<T> xr[NC], gr[NC];
    float w[NC][8], b[NC][8];
    int n[NC];       // of each vector, the channels in the group
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int c = 8 * (l + LP * j);
        n[j] = here ? min(8, p.width - c) : 0;
        const int wide = n[j] > 0 && first + c + 8 <= p.dim ? 8 : n[j];   // what may be read
        xr[j] = load8_at<T>(x + c, wide);
        if (p.gate) gr[j] = load8_at<T>(gt + c, wide);
        gn_weights<T>(p.weight, p.w_f32, first + c, wide, w[j]);
        if (p.bias) gn_weights<T>(p.bias, p.w_f32, first + c, wide, b[j]);
    }
    float v[NC][8], s = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[j][i] = at8(xr[j], i);
            s += i < n[j] ? v[j][i] : 0.0f;
        }
    const float mean = lanes_sum<LP>(s, red[0]) / (float)p.width;
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[j][i] -= mean;
            ss += i < n[j] ? v[j][i] * v[j][i] : 0.0f;
        }
    const float rstd = 1.0f / sqrtf(lanes_sum<LP>(ss, red[1]) / (float)p.width + p.eps);
    if (here && l == 0) {
        if (p.mean) p.mean[unit] = mean;
        if (p.rstd) p.rstd[unit] = rstd;
    }
#pragma unroll
    for (int j = 0; j < NC; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float z = v[j][i] * rstd * w[j][i];
            if (p.bias) z += b[j][i];
            v[j][i] = p.gate ? z * activation(p.act, at8(gr[j], i)) : activation(p.act, z);
        }
        const int c = first + 8 * (l + LP * j);
        if constexpr (FP8) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, n[j] > 0 ? fabsf(v[j][i]) : 0.0f);
            const int e = block_exponent(row16_max(top));
            u32x2 q;
            quantize8(v[j], exponent_recip(e), q);
            if (n[j] > 0) {
                __builtin_memcpy(p.q + row * p.ld_q + c, &q, 8);
                if ((c & 127) == 0) p.scale[row * p.ld_scale + (c >> 7)] = (uint8_t)e;
            }
        } else if (n[j] > 0) {
            store8_at<T>(static_cast<T*>(p.y) + row * p.ld_y + c, v[j], n[j]);
        }
    }
}

// 8 bits, whatever the groups: a workgroup a row, which it keeps in LDS in fp32; a wave
// a group for the sums and the outputs, sixteen lanes a block of 128 for the 8 bits.
template <typename T>
__device__ void group_norm_fp8_any(const HelixGroupNormParams& p) {
    __shared__ float z[16384];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
    const T* gt = static_cast<const T*>(p.gate) + row * p.ld_gate;
    for (int c = threadIdx.x; c < p.dim; c += GN_THREADS) z[c] = (float)x[c];
    __syncthreads();
    const int lane = lane_id();
    for (int g = wave_id(); g < p.groups; g += GN_THREADS / 64) {
        const int first = g * p.width, end = first + p.width;
        float s = 0.0f, ss = 0.0f;
        for (int c = first + lane; c < end; c += 64) s += z[c];
        const float mean = wave_sum(s) / (float)p.width;
        for (int c = first + lane; c < end; c += 64) ss += (z[c] - mean) * (z[c] - mean);
        const float rstd = 1.0f / sqrtf(wave_sum(ss) / (float)p.width + p.eps);
        if (lane == 0) {
            if (p.mean) p.mean[row * p.groups + g] = mean;
            if (p.rstd) p.rstd[row * p.groups + g] = rstd;
        }
        for (int c = first + lane; c < end; c += 64) {
            const float w = p.w_f32 ? static_cast<const float*>(p.weight)[c] : (float)static_cast<const T*>(p.weight)[c];
            float o = (z[c] - mean) * rstd * w;
            if (p.bias) o += p.w_f32 ? static_cast<const float*>(p.bias)[c] : (float)static_cast<const T*>(p.bias)[c];
            z[c] = p.gate ? o * activation(p.act, (float)gt[c]) : activation(p.act, o);
        }
    }
    __syncthreads();
    // (A block is sixteen lanes' of one wave, and all of a wave's lanes go round alike.)
    for (int c0 = 0; c0 < p.dim; c0 += 8 * GN_THREADS) {
        const int c = c0 + 8 * threadIdx.x, n = min(8, p.dim - c);
        float v[8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = i < n ? z[c + i] : 0.0f;
            top = fmaxf(top, fabsf(v[i]));
        }
        const int e = block_exponent(row16_max(top));
        u32x2 q;
        quantize8(v, exponent_recip(e), q);
        if (n >= 8) {
            __builtin_memcpy(p.q + row * p.ld_q + c, &q, 8);
        } else {
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (i < n) p.q[row * p.ld_q + c + i] = (uint8_t)(q[i >> 2] >> (8 * (i & 3)));
        }
        if (n > 0 && (c & 127) == 0) p.scale[row * p.ld_scale + (c >> 7)] = (uint8_t)e;
    }
}

// dx and dgate, and the sums of dweight and dbias over the rows of a part: a workgroup
// works on group_slots groups of as many rows as it has room for (its row slots), row
// after row, and leaves each row slot's sums as a part of its own.
template <typename T, int LP, int NC>
__device__ void group_norm_bwd(const HelixGroupNormBwdParams& p) {
    __shared__ float red[2][2][GN_THREADS / 64];
    const int slot = threadIdx.x / LP, l = threadIdx.x % LP;
    const int g = blockIdx.x * p.group_slots + slot % p.group_slots, rs = slot / p.group_slots;
    const int row_slots = GN_THREADS / LP / p.group_slots;
    const bool mine = g < p.groups;
    const int first = g * p.width;
    float w[NC][8], b[NC][8], dw[NC][8], db[NC][8];
    int n[NC], wide[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int c = 8 * (l + LP * j);
        n[j] = mine ? min(8, p.width - c) : 0;
        wide[j] = n[j] > 0 && first + c + 8 <= p.dim ? 8 : n[j];
        gn_weights<T>(p.weight, p.w_f32, first + c, wide[j], w[j]);
#pragma unroll
        for (int i = 0; i < 8; ++i) b[j][i] = dw[j][i] = db[j][i] = 0.0f;
        if (p.bias) gn_weights<T>(p.bias, p.w_f32, first + c, wide[j], b[j]);
    }
    const long long lo = blockIdx.y * p.part_rows, end = min(p.rows, lo + p.part_rows);
    int turn = 0;
    // (A workgroup that is one group's has one row slot: all its threads go round alike.)
    for (long long row = lo + rs; row < end; row += row_slots) {
        Raw8<T> xr[NC], yr[NC], gr[NC];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = first + 8 * (l + LP * j);
            xr[j] = load8_at<T>(static_cast<const T*>(p.x) + row * p.ld_x + c, wide[j]);
            yr[j] = load8_at<T>(static_cast<const T*>(p.dy) + row * p.ld_dy + c, wide[j]);
            if (p.gate) gr[j] = load8_at<T>(static_cast<const T*>(p.gate) + row * p.ld_gate + c, wide[j]);
        }
        const float mean = mine ? p.mean[row * p.groups + g] : 0.0f, rstd = mine ? p.rstd[row * p.groups + g] : 0.0f;
        float t[NC][8], s = 0.0f, st = 0.0f;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            float dg[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float nn = (at8(xr[j], i) - mean) * rstd, dy = at8(yr[j], i);
                const float z = nn * w[j][i] + b[j][i];
                float a, slope;
                activation(p.act, p.gate ? at8(gr[j], i) : z, a, slope);
                const float dz = dy * (p.gate ? a : slope);
                dg[i] = dy * z * slope;
                t[j][i] = dz * w[j][i];
                if (i < n[j]) {
                    dw[j][i] += dz * nn;
                    db[j][i] += dz;
                    s += t[j][i];
                    st += t[j][i] * nn;
                }
            }
            if (p.gate && n[j] > 0)
                store8_at<T>(static_cast<T*>(p.dgate) + row * p.ld_dgate + first + 8 * (l + LP * j), dg, n[j]);
        }
        // Two places in turn: a wave may be at the next row's sums while another reads this one's.
        const float ms = lanes_sum<LP>(s, red[turn][0]) / (float)p.width;
        const float mt = lanes_sum<LP>(st, red[turn][1]) / (float)p.width;
        turn ^= 1;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = rstd * (t[j][i] - ms - (at8(xr[j], i) - mean) * rstd * mt);
            if (n[j] > 0) store8_at<T>(static_cast<T*>(p.dx) + row * p.ld_dx + first + 8 * (l + LP * j), o, n[j]);
        }
    }
    if (!p.part || !mine) return;
    float* to = p.part + ((long long)blockIdx.y * row_slots + rs) * 2 * p.dim + first;
#pragma unroll
    for (int j = 0; j < NC; ++j)
        if (n[j] > 0) {
            const int c = 8 * (l + LP * j);
            store8_at<float>(to + c, dw[j], n[j]);
            store8_at<float>(to + p.dim + c, db[j], n[j]);
        }
}

}  // namespace

// dweight and dbias from the parts, in their order: 32 channels a workgroup, every 32nd
// part a half of a wave, eight loads at a time.
extern "C" __global__ __launch_bounds__(1024) void helix_group_norm_dw(HelixGroupNormBwdParams p) {
    __shared__ float sum[32][33];
    const int half = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < 2 * p.dim)
        for (int i = half; i < p.parts; i += 32 * 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = i + 32 * u < p.parts ? p.part[(i + 32LL * u) * 2 * p.dim + c] : 0.0f;
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
    sum[half][lane] = s;
    __syncthreads();
    if (half || c >= 2 * p.dim) return;
#pragma unroll
    for (int w = 1; w < 32; ++w) s += sum[w][lane];
    float* to = c < p.dim ? p.dweight : p.dbias;
    if (to) to[c < p.dim ? c : c - p.dim] = s;
}

#define GN_FORM(TAG, T, LP, NC)                                                                                                 \
    extern "C" __global__ __launch_bounds__(GN_THREADS) void helix_group_norm_##TAG##_l##LP##_##NC(HelixGroupNormParams p) {    \
        group_norm<T, LP, NC, false>(p);                                                                                        \
    }                                                                                                                           \
    extern "C" __global__ __launch_bounds__(GN_THREADS) void helix_group_norm_bwd_##TAG##_l##LP##_##NC(HelixGroupNormBwdParams p) { \
        group_norm_bwd<T, LP, NC>(p);                                                                                           \
    }
// (8 bits: groups that line up with blocks of 128.)
#define GN_FORM8(TAG, T, LP, NC)                                                                                                \
    GN_FORM(TAG, T, LP, NC)                                                                                                     \
    extern "C" __global__ __launch_bounds__(GN_THREADS) void helix_group_norm_fp8_##TAG##_l##LP##_##NC(HelixGroupNormParams p) { \
        group_norm<T, LP, NC, true>(p);                                                                                         \
    }
#define GN_FORMS(TAG, T)                                                                                                   \
    GN_FORM8(TAG, T, 4, 1)                                                                                                 \
    GN_FORM8(TAG, T, 8, 1)                                                                                                 \
    GN_FORM8(TAG, T, 16, 1)                                                                                                \
    GN_FORM8(TAG, T, 32, 1)                                                                                                \
    GN_FORM8(TAG, T, 64, 1)                                                                                                \
    GN_FORM8(TAG, T, 64, 2)                                                                                                \
    GN_FORM8(TAG, T, 256, 1)                                                                                               \
    GN_FORM8(TAG, T, 256, 2)                                                                                               \
    GN_FORM8(TAG, T, 256, 4)                                                                                               \
    extern "C" __global__ __launch_bounds__(GN_THREADS) void helix_group_norm_fp8_##TAG##_any(HelixGroupNormParams p) {   \
        group_norm_fp8_any<T>(p);                                                                                          \
    }
GN_FORMS(f32, float)
GN_FORMS(f16, _Float16)
GN_FORMS(bf16, __bf16)
