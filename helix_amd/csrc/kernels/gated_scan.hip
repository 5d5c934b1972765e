// gated_scan.hip -- gated linear recurrence per channel and its backward pass
// (helix_layer.h).
//
// A step is s -> f s + b, and steps compose: (A, B) after (A', B') is (A A', A B' +
// B). So a sequence is cut into runs of R tokens, one thread each (for four
// channels): a thread loads its run, folds it to (A, B), learns the state that
// enters its run from the runs before it, and walks the run again from registers.
// Every input is read once and every output written once.
//
//   run       R tokens of 4 channels    a thread's registers (f and b in fp32)
//   tile      4 NW runs of 64 channels  a workgroup of NW waves: lanes 16 q + c hold
//                                       run 4 wave + q of channels 4 c .. 4 c + 3, so
//                                       that a row's 64 channels are read together
//   chunk     a tile of a sequence      joined through scratch, below
//
// Backward, the tokens are taken from the last to the first: with c_t = f_t
// lambda_t the step is c_t = f_t c_(t+1) + f_t dh_t, and lambda_t = dh_t + c_(t+1).
//
// Joining chunks. Each workgroup takes a ticket; tickets go through the chunks in
// order, so whatever a workgroup waits for belongs to one that has started before
// it and does not wait for a later one: the lowest ticket at work never waits, and
// every wait ends. A workgroup publishes its chunk's (A, B) as soon as it has them.
// Then it reads those of the chunks before it in its group of GROUP chunks, all at
// once, and the state that left the group before; the last of a group publishes
// the state that leaves it. A word is its own flag: scratch is filled with ones
// first, and a pattern of ones is a NaN that is never published (any other NaN is
// made the ordinary one). Words are written and read by relaxed atomics of agent
// scope, which go past the L2s of the XCDs. The parts are joined in the order of
// time, whoever arrives first: results do not depend on it.
//
// Memory binds it. 8192 tokens of 4096 channels (bf16) take 51 us, 201 MB moved at
// 4.0 TB/s; 3 x 1003 of 5184 (f32) 47 us, 4.0 TB/s; backward 8 x 4096 of 5120 (bf16)
// 400 us, 5.0 TB/s, where a copy of 4 GiB reaches 4.6. Runs of 4 tokens instead of 8
// took 62-66 us forward (twice the joins per value); backward, which holds twice the
// words of a token, runs of 8 spill and took 422 us, of 2 532. Groups of 16 chunks
// instead of 8 took 65 and 561 us: their words cost a wave of each SIMD. Stores that
// are not kept in the caches (nt) took 2.6% less backward, where two outputs leave;
// nothing forward.
#include "layer_common.h"

namespace {

constexpr int GS_THREADS = 256;

// Four channels of a row, at any address: a wide load where VEC or where there are as many, else the ones below n.
template <typename T>
struct Four {
    typedef T type __attribute__((ext_vector_type(4)));
};
template <typename T, bool VEC>
HELIX_DEV typename Four<T>::type load4(const T* p, int n) {
    typename Four<T>::type w = {(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f};
    if (VEC || n >= 4) {
        __builtin_memcpy(&w, p, sizeof w);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) w[i] = p[i];
    }
    return w;
}
template <typename T, bool VEC>
HELIX_DEV void store4(T* p, const float (&v)[4], int n) {
    if (VEC || n >= 4) {
        const typename Four<T>::type w = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        __builtin_memcpy(p, &w, sizeof w);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

HELIX_DEV unsigned long long peek64(const unsigned long long* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
HELIX_DEV unsigned peek32(const unsigned* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
HELIX_DEV float no_flag(float v) { return v == v ? v : __builtin_nanf(""); }

constexpr unsigned NOT_YET = 0xffffffffu;
// Rounds of a wait, of a microsecond or so: far more than any that ends. Past it a
// wait gives up with what it has (a NaN), so that no kernel can hang.
constexpr int PATIENCE = 1 << 24;

// The state that enters chunk `chunk` of a stream, for one channel (lane), from
// `start` before the first chunk.
HELIX_DEV float state_before(const HelixGatedScanJoin& j, long long stream, int chunk, float start) {
    constexpr int GROUP = HELIX_GS_GROUP;
    const int lane = lane_id();
    const int first = chunk / GROUP * GROUP, n = chunk - first;
    const unsigned long long* part = j.part + ((stream * j.n_chunk + first) * 64 + lane);
    const unsigned* left = j.left + ((stream * j.n_group + first / GROUP - 1) * 64 + lane);
    unsigned long long w[GROUP - 1];
    unsigned s = as_u32(start);
    for (int round = 0; round < PATIENCE; ++round) {
        bool ready = true;
#pragma unroll
        for (int i = 0; i < GROUP - 1; ++i) w[i] = i < n ? peek64(part + 64 * i) : 0;
        if (first) s = peek32(left);
#pragma unroll
        for (int i = 0; i < GROUP - 1; ++i) ready &= (unsigned)w[i] != NOT_YET;
        if (first) ready &= s != NOT_YET;
        if (__all(ready)) break;
        __builtin_amdgcn_s_sleep(1);
    }
    float state = as_f32(s);
#pragma unroll
    for (int i = 0; i < GROUP - 1; ++i)
        if (i < n) state = as_f32((unsigned)w[i]) * state + as_f32((unsigned)(w[i] >> 32));
    return state;
}

// v has been loaded before anything that follows reaches memory.
HELIX_DEV void arrived(float& v) { asm volatile("" : "+v"(v)::"memory"); }

// From the (A, B) of a thread's run of four channels to the state that enters it.
// `start`, the state before the first chunk (64 channels; null: zero), and `end`,
// where the last chunk leaves its state (null: nowhere; maybe start's memory), are of
// the tile's channels, of which there are `width`.
template <int NW>
HELIX_DEV void entering(const HelixGatedScanJoin& j, long long stream, int chunk, const float* start, float* end,
                        int width, const float (&run_a)[4], const float (&run_b)[4], float (&state)[4]) {
    __shared__ float2 sum[NW][64];
    __shared__ float in[NW][64];
    const int lane = lane_id(), wave = wave_id(), q = lane >> 4, c4 = 4 * (lane & 15);
    // Read before the chunk is published, and only by chunks that the last one waits for: `end` may be `start`.
    float s = wave == 0 && start && chunk < HELIX_GS_GROUP && lane < width ? start[lane] : 0.0f;
    float a[4], b[4];   // of the wave's runs up to this one
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = run_a[i];
        b[i] = run_b[i];
#pragma unroll
        for (int d = 1; d < 4; d *= 2) {
            const float pa = __shfl_up(a[i], 16 * d, 64), pb = __shfl_up(b[i], 16 * d, 64);
            if (q >= d) {
                b[i] = a[i] * pb + b[i];
                a[i] = a[i] * pa;
            }
        }
        if (q == 3) sum[wave][c4 + i] = make_float2(a[i], b[i]);
        // and up to the one before it
        const float pa = __shfl_up(a[i], 16, 64), pb = __shfl_up(b[i], 16, 64);
        a[i] = q ? pa : 1.0f;
        b[i] = q ? pb : 0.0f;
    }
    __syncthreads();
    if (wave == 0) {
        const int c = lane;
        const bool many = j.n_chunk > 1, final = chunk == j.n_chunk - 1;
        arrived(s);
        if (many && !final) {
            float ca = 1.0f, cb = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float2 s = sum[w][c];
                cb = s.x * cb + s.y;
                ca = s.x * ca;
            }
            const unsigned long long word = (unsigned long long)as_u32(cb) << 32 | as_u32(no_flag(ca));
            __hip_atomic_store(j.part + ((stream * j.n_chunk + chunk) * 64 + c), word, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        }
        if (many && chunk) s = state_before(j, stream, chunk, s);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            in[w][c] = s;
            s = sum[w][c].x * s + sum[w][c].y;
        }
        if (final) {
            if (end && c < width) end[c] = s;
        } else if (chunk % HELIX_GS_GROUP == HELIX_GS_GROUP - 1) {
            __hip_atomic_store(j.left + ((stream * j.n_group + chunk / HELIX_GS_GROUP) * 64 + c), as_u32(no_flag(s)),
                               __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) state[i] = a[i] * in[wave][c4 + i] + b[i];
}

// Which tile a workgroup takes: its ticket where chunks are joined.
HELIX_DEV unsigned tile_index(const HelixGatedScanJoin& j) {
    __shared__ unsigned t;
    if (j.n_chunk == 1) return blockIdx.x;
    if (threadIdx.x == 0) t = __hip_atomic_fetch_add(j.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    __syncthreads();
    return t;
}

// The tokens of a wave in one tensor, from its first token: a lane's own start at
// `voff`, `tok` bytes apart. A lane without channels is out of range: it reads zeros
// and writes nothing. So is a token past the sequence where rows do not overlap, as
// those that are written never do.
struct WaveRows {
    helix_rsrc r;
    int voff, tok;
};
template <typename T>
HELIX_DEV WaveRows wave_rows(const void* base, long long at, long long tok, int tokens, int width, int skip, bool live) {
    WaveRows w;
    w.tok = (int)tok * (int)sizeof(T);
    const int bytes = tokens > 0 ? (tokens - 1) * w.tok + width * (int)sizeof(T) : 0;
    w.r = make_rsrc_u(static_cast<const T*>(base) + at, bytes);
    w.voff = live ? skip * w.tok + 4 * (int)sizeof(T) * (lane_id() & 15) : (int)0x80000000;
    return w;
}

// What comes after is not started before: or the products that do not need the
// entering state are formed before the wait for it, in more registers than the
// words that they are made of.
template <typename W>
HELIX_DEV void not_earlier(W& w) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(w) / 4); ++i) w[i] = (unsigned)vgpr_fresh((int)w[i]);
}

// A token that does not exist has an infinite gate and brings nothing (u: v, or backward
// dh): the state passes through it. Where a tensor's tokens lie closer than a row is
// long (all of them one row, say), its place is inside the resource's range.
template <typename T>
HELIX_DEV void shut_out(typename Raw4<T>::type& g, typename Raw4<T>::type& u, bool exists) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(g) / 4); ++i) {
        g[i] = exists ? g[i] : inf_bits<T>;
        u[i] = exists ? u[i] : 0;
    }
}

template <typename T, bool VEC, int NW>
HELIX_DEV void gated_scan_tile(const HelixGatedScanParams& p, unsigned tile) {
    constexpr int R = HELIX_GS_RUN;
    const int streams = p.n_seq * p.n_slab;
    const int chunk = tile / streams, stream = tile % streams;
    const int seq = stream / p.n_slab, c0 = (stream % p.n_slab) * 64;
    const int lane = lane_id(), width = min(64, p.n_chan - c0), own = width - 4 * (lane & 15);
    const int tw = (chunk * NW + wave_uniform()) * 4 * R, skip = (lane >> 4) * R;   // the wave's first token, the lane's
    const int tokens = min(4 * R, p.n_tok - tw);                                    // not positive: none
    const long long t = tokens > 0 ? tw : 0;
    const WaveRows g = wave_rows<T>(p.g, seq * p.seq_g + t * p.tok_g + c0, p.tok_g, tokens, width, skip, own > 0);
    const WaveRows v = wave_rows<T>(p.v, seq * p.seq_v + t * p.tok_v + c0, p.tok_v, tokens, width, skip, own > 0);
    typename Raw4<T>::type gw[R], vw[R];
#pragma unroll
    for (int k = 0; k < R; ++k) gw[k] = buf_load4<T, VEC>(g.r, g.voff + k * g.tok, own);
#pragma unroll
    for (int k = 0; k < R; ++k) vw[k] = buf_load4<T, VEC>(v.r, v.voff + k * v.tok, own);
    if (tokens < 4 * R) {
#pragma unroll
        for (int k = 0; k < R; ++k) shut_out<T>(gw[k], vw[k], skip + k < tokens);
    }
    float f[R][4], b[R][4], ra[4], rb[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ra[i] = 1.0f, rb[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < R; ++k) {
        float gf[4], vf[4];
        widen4<T>(gw[k], gf);
        widen4<T>(vw[k], vf);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float u;
            gate(gf[i], f[k][i], u);
            b[k][i] = u * vf[i];
            ra[i] *= f[k][i];
            rb[i] = f[k][i] * rb[i] + b[k][i];
        }
    }
    const long long at = (long long)seq * p.n_chan + c0;
    entering<NW>(p.join, stream, chunk, p.h0 ? p.h0 + at : nullptr, p.last ? p.last + at : nullptr, width, ra, rb, s);
    const WaveRows h = wave_rows<T>(p.h, seq * p.seq_h + t * p.tok_h + c0, p.tok_h, tokens, width, skip, own > 0);
#pragma unroll
    for (int k = 0; k < R; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = f[k][i] * s[i] + b[k][i];
        buf_store4<T, VEC>(h.r, s, h.voff + k * h.tok, own);
    }
}

// A slab of 64 channels moves by four at any alignment; one that n_chan cuts elsewhere
// than at a multiple of four goes channel by channel (QUADS: there is none). With all
// slabs channel by channel 8192 tokens of 4095 channels (bf16) took 91 us, as here 67,
// and backward over 8 x 4096 of 5119 1147, as here 774.
template <bool QUADS, typename P, typename W, typename E>
HELIX_DEV void by_slab(const P& p, W&& wide, E&& each) {
    const unsigned tile = __builtin_amdgcn_readfirstlane(tile_index(p.join));
    if (QUADS || (int)(tile % (p.n_seq * p.n_slab) % p.n_slab) * 64 + 64 <= p.n_chan) wide(tile);
    else each(tile);
}

// Few tokens: one thread per four channels walks them.
template <typename T, bool VEC>
__device__ void gated_scan_steps(const HelixGatedScanParams& p) {
    const int quads = (p.n_chan + 3) >> 2;
    const long long i = (long long)blockIdx.x * GS_THREADS + threadIdx.x;
    const int seq = (int)(i / quads), c = 4 * (int)(i % quads);
    if (seq >= p.n_seq) return;
    const int own = min(4, p.n_chan - c);
    const T* g = static_cast<const T*>(p.g) + seq * p.seq_g + c;
    const T* v = static_cast<const T*>(p.v) + seq * p.seq_v + c;
    T* h = static_cast<T*>(p.h) + seq * p.seq_h + c;
    const long long at = (long long)seq * p.n_chan + c;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (p.h0 && k < own) s[k] = p.h0[at + k];
    for (int t = 0; t < p.n_tok; ++t) {
        const auto gw = load4<T, VEC>(g + t * p.tok_g, own), vw = load4<T, VEC>(v + t * p.tok_v, own);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float f, u;
            gate((float)gw[k], f, u);
            s[k] = f * s[k] + u * (float)vw[k];
        }
        store4<T, VEC>(h + t * p.tok_h, s, own);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (p.last && k < own) p.last[at + k] = s[k];
}

// As gated_scan_tile, with time turned round: chunk 0 and run 0 are the last.
template <typename T, bool VEC, int NW>
HELIX_DEV void gated_scan_bwd_tile(const HelixGatedScanBwdParams& p, unsigned tile) {
    constexpr int R = HELIX_GS_RUN_BWD;
    const int streams = p.n_seq * p.n_slab;
    const int chunk = tile / streams, stream = tile % streams;
    const int seq = stream / p.n_slab, c0 = (stream % p.n_slab) * 64;
    const int lane = lane_id(), width = min(64, p.n_chan - c0), own = width - 4 * (lane & 15);
    // The wave's last token and its first; the lane's last one, from the first on.
    const int hi = p.n_tok - 1 - (chunk * NW + wave_uniform()) * 4 * R;
    const int tokens = min(4 * R, hi + 1), skip = tokens - 1 - (lane >> 4) * R;
    const long long t = tokens > 0 ? hi + 1 - tokens : 0;
    const bool any = own > 0;
    const WaveRows g = wave_rows<T>(p.g, seq * p.seq_g + t * p.tok_g + c0, p.tok_g, tokens, width, skip, any);
    const WaveRows d = wave_rows<T>(p.dh, seq * p.seq_dh + t * p.tok_dh + c0, p.tok_dh, tokens, width, skip, any);
    const WaveRows v = wave_rows<T>(p.v, seq * p.seq_v + t * p.tok_v + c0, p.tok_v, tokens, width, skip, any);
    // h of the token before each; before token 0 there is none (h0 below).
    const int back = t > 0 ? 1 : 0;
    const WaveRows h = wave_rows<T>(p.h, seq * p.seq_h + (t - back) * p.tok_h + c0, p.tok_h, tokens - 1 + back, width,
                                    skip - 1 + back, any);
    typename Raw4<T>::type gw[R], dw[R], vw[R], hw[R];
#pragma unroll
    for (int k = 0; k < R; ++k) gw[k] = buf_load4<T, VEC>(g.r, g.voff - k * g.tok, own);
#pragma unroll
    for (int k = 0; k < R; ++k) dw[k] = buf_load4<T, VEC>(d.r, d.voff - k * d.tok, own);
#pragma unroll
    for (int k = 0; k < R; ++k) vw[k] = buf_load4<T, VEC>(v.r, v.voff - k * v.tok, own);
#pragma unroll
    for (int k = 0; k < R; ++k) hw[k] = buf_load4<T, VEC>(h.r, h.voff - k * h.tok, own);
    if (tokens < 4 * R) {
#pragma unroll
        for (int k = 0; k < R; ++k) shut_out<T>(gw[k], dw[k], skip - k >= 0);
    }
    float f[R][4], u[R][4], ra[4], rb[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ra[i] = 1.0f, rb[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < R; ++k) {
        float gf[4], df[4];
        widen4<T>(gw[k], gf);
        widen4<T>(dw[k], df);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            gate(gf[i], f[k][i], u[k][i]);
            ra[i] *= f[k][i];
            rb[i] = f[k][i] * (rb[i] + df[i]);
        }
    }
    const long long at = (long long)seq * p.n_chan + c0;
    entering<NW>(p.join, stream, chunk, p.dh_last ? p.dh_last + at : nullptr, p.dh0 ? p.dh0 + at : nullptr, width, ra,
                 rb, s);
    const WaveRows dg = wave_rows<T>(p.dg, seq * p.seq_dg + t * p.tok_dg + c0, p.tok_dg, tokens, width, skip, any);
    const WaveRows dv = wave_rows<T>(p.dv, seq * p.seq_dv + t * p.tok_dv + c0, p.tok_dv, tokens, width, skip, any);
#pragma unroll
    for (int k = 0; k < R; ++k) {
        float df[4], vf[4], past[4], og[4], ov[4];
        not_earlier(dw[k]);
        not_earlier(vw[k]);
        not_earlier(hw[k]);
        widen4<T>(dw[k], df);
        widen4<T>(vw[k], vf);
        widen4<T>(hw[k], past);
        if (t == 0 && skip == k) {   // token 0
#pragma unroll
            for (int i = 0; i < 4; ++i) past[i] = p.h0 && i < own ? p.h0[at + 4 * (lane & 15) + i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lam = s[i] + df[i];
            ov[i] = lam * u[k][i];
            og[i] = ov[i] * f[k][i] * (past[i] - vf[i]);
            s[i] = f[k][i] * lam;
        }
        buf_store4<T, VEC, HELIX_NT_L2>(dv.r, ov, dv.voff - k * dv.tok, own);
        buf_store4<T, VEC, HELIX_NT_L2>(dg.r, og, dg.voff - k * dg.tok, own);
    }
}

template <typename T, bool VEC>
__device__ void gated_scan_bwd_steps(const HelixGatedScanBwdParams& p) {
    const int quads = (p.n_chan + 3) >> 2;
    const long long i = (long long)blockIdx.x * GS_THREADS + threadIdx.x;
    const int seq = (int)(i / quads), c = 4 * (int)(i % quads);
    if (seq >= p.n_seq) return;
    const int own = min(4, p.n_chan - c);
    const T* dh = static_cast<const T*>(p.dh) + seq * p.seq_dh + c;
    const T* g = static_cast<const T*>(p.g) + seq * p.seq_g + c;
    const T* v = static_cast<const T*>(p.v) + seq * p.seq_v + c;
    const T* h = static_cast<const T*>(p.h) + seq * p.seq_h + c;
    T* dg = static_cast<T*>(p.dg) + seq * p.seq_dg + c;
    T* dv = static_cast<T*>(p.dv) + seq * p.seq_dv + c;
    const long long at = (long long)seq * p.n_chan + c;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f}, h0[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (p.dh_last && k < own) s[k] = p.dh_last[at + k];
        if (p.h0 && k < own) h0[k] = p.h0[at + k];
    }
    for (int t = p.n_tok - 1; t >= 0; --t) {
        const auto gw = load4<T, VEC>(g + t * p.tok_g, own), vw = load4<T, VEC>(v + t * p.tok_v, own),
                   dw = load4<T, VEC>(dh + t * p.tok_dh, own);
        auto hw = load4<T, false>(nullptr, 0);
        if (t) hw = load4<T, VEC>(h + (t - 1) * p.tok_h, own);
        float og[4], ov[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float f, u;
            gate((float)gw[k], f, u);
            const float lam = s[k] + (float)dw[k];
            ov[k] = lam * u;
            og[k] = ov[k] * f * ((t ? (float)hw[k] : h0[k]) - (float)vw[k]);
            s[k] = f * lam;
        }
        store4<T, VEC>(dv + t * p.tok_dv, ov, own);
        store4<T, VEC>(dg + t * p.tok_dg, og, own);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (p.dh0 && k < own) p.dh0[at + k] = s[k];
}

}  // namespace

// Ones into the scratch that chunks are joined through, 16 bytes a thread.
extern "C" __global__ __launch_bounds__(GS_THREADS) void helix_gated_scan_fill(uint4* p, long long n) {
    const long long i = (long long)blockIdx.x * GS_THREADS + threadIdx.x;
    if (i < n) p[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

#define GATED_SCAN_TILE(TAG, T, VTAG, VEC, NW)                                                                       \
    extern "C" __global__ __launch_bounds__(64 * NW) void helix_gated_scan_##TAG##VTAG##_w##NW(HelixGatedScanParams p) { \
        by_slab<VEC>(p, [&](unsigned t) { gated_scan_tile<T, true, NW>(p, t); },                                     \
                     [&](unsigned t) { if constexpr (!VEC) gated_scan_tile<T, false, NW>(p, t); });                  \
    }                                                                                                                \
    extern "C" __global__                                                                                            \
        __launch_bounds__(64 * NW) void helix_gated_scan_bwd_##TAG##VTAG##_w##NW(HelixGatedScanBwdParams p) {        \
        by_slab<VEC>(p, [&](unsigned t) { gated_scan_bwd_tile<T, true, NW>(p, t); },                                 \
                     [&](unsigned t) { if constexpr (!VEC) gated_scan_bwd_tile<T, false, NW>(p, t); });              \
    }
#define GATED_SCAN_KERNELS(TAG, T, VTAG, VEC)                                                                        \
    GATED_SCAN_TILE(TAG, T, VTAG, VEC, 4)                                                                            \
    GATED_SCAN_TILE(TAG, T, VTAG, VEC, 8)                                                                            \
    extern "C" __global__ __launch_bounds__(GS_THREADS) void helix_gated_scan_##TAG##VTAG##_steps(HelixGatedScanParams p) { \
        gated_scan_steps<T, VEC>(p);                                                                                 \
    }                                                                                                                \
    extern "C" __global__                                                                                            \
        __launch_bounds__(GS_THREADS) void helix_gated_scan_bwd_##TAG##VTAG##_steps(HelixGatedScanBwdParams p) {     \
        gated_scan_bwd_steps<T, VEC>(p);                                                                             \
    }
GATED_SCAN_KERNELS(f32, float, _v, true)
GATED_SCAN_KERNELS(f32, float, _s, false)
GATED_SCAN_KERNELS(f16, _Float16, _v, true)
GATED_SCAN_KERNELS(f16, _Float16, _s, false)
GATED_SCAN_KERNELS(bf16, __bf16, _v, true)
GATED_SCAN_KERNELS(bf16, __bf16, _s, false)
