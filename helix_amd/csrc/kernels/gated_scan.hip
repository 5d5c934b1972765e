// gated_scan.hip -- gated linear recurrence per channel and its backward pass
// (helix_layer.h).
#include "layer_common.h"

namespace {

constexpr int GS_THREADS = 256;

// One thread per channel of a sequence, token by token.
template <typename T>
__device__ void gated_scan(const HelixGatedScanParams& p) {
    const long long i = (long long)blockIdx.x * GS_THREADS + threadIdx.x;
    if (i >= (long long)p.n_seq * p.n_chan) return;
    const long long seq = i / p.n_chan, c = i % p.n_chan;
    const T* g = static_cast<const T*>(p.g) + seq * p.seq_g + c;
    const T* v = static_cast<const T*>(p.v) + seq * p.seq_v + c;
    T* h = static_cast<T*>(p.h) + seq * p.seq_h + c;
    float s = p.h0 ? p.h0[i] : 0.0f;
    for (int t = 0; t < p.n_tok; ++t) {
        float f, u;
        gate((float)g[t * p.tok_g], f, u);
        s = f * s + u * (float)v[t * p.tok_v];
        h[t * p.tok_h] = (T)s;
    }
    if (p.last) p.last[i] = s;
}

template <typename T>
__device__ void gated_scan_bwd(const HelixGatedScanBwdParams& p) {
    const long long i = (long long)blockIdx.x * GS_THREADS + threadIdx.x;
    if (i >= (long long)p.n_seq * p.n_chan) return;
    const long long seq = i / p.n_chan, c = i % p.n_chan;
    const T* dh = static_cast<const T*>(p.dh) + seq * p.seq_dh + c;
    const T* g = static_cast<const T*>(p.g) + seq * p.seq_g + c;
    const T* v = static_cast<const T*>(p.v) + seq * p.seq_v + c;
    const T* h = static_cast<const T*>(p.h) + seq * p.seq_h + c;
    T* dg = static_cast<T*>(p.dg) + seq * p.seq_dg + c;
    T* dv = static_cast<T*>(p.dv) + seq * p.seq_dv + c;
    float carry = p.dh_last ? p.dh_last[i] : 0.0f;   // f_(t+1) lambda_(t+1)
    for (int t = p.n_tok - 1; t >= 0; --t) {
        float f, u;
        gate((float)g[t * p.tok_g], f, u);
        const float lam = carry + (float)dh[t * p.tok_dh];
        const float past = t ? (float)h[(t - 1) * p.tok_h] : p.h0 ? p.h0[i] : 0.0f;
        dv[t * p.tok_dv] = (T)(lam * u);
        dg[t * p.tok_dg] = (T)(lam * (past - (float)v[t * p.tok_v]) * f * u);
        carry = f * lam;
    }
    if (p.dh0) p.dh0[i] = carry;
}

}  // namespace

#define GATED_SCAN_KERNELS(TAG, T)                                                                              \
    extern "C" __global__ __launch_bounds__(GS_THREADS) void helix_gated_scan_##TAG(HelixGatedScanParams p) {   \
        gated_scan<T>(p);                                                                                       \
    }                                                                                                           \
    extern "C" __global__ __launch_bounds__(GS_THREADS) void helix_gated_scan_bwd_##TAG(HelixGatedScanBwdParams p) { \
        gated_scan_bwd<T>(p);                                                                                   \
    }
GATED_SCAN_KERNELS(f32, float)
GATED_SCAN_KERNELS(f16, _Float16)
GATED_SCAN_KERNELS(bf16, __bf16)
