// delta_rule.hip -- the gated delta rule (helix_layer.h): per value head, with the state S of
// N keys x P values in fp32,
//     S_t = e^(g_t) S_(t-1) + beta_t k_t (v_t - e^(g_t) S_(t-1)' k_t)',   o_t = scale S_t' q_t
//
// Few tokens go one by one (helix_delta_steps_*). More go in chunks of 64: with G the sums of
// g from the chunk's start, E_ij = exp(G_i - G_j) for j <= i, A_ij = beta_i E_ij (k_i . k_j)
// below the diagonal and X = (1 + A)^-1 diag(beta),
//     D = X (V - e^G K S),   O = scale (e^G Q S + (E . Q K') D),   S' = e^(G_63) S + (e^(G_63 - G) K)' D
// X and P = scale E . Q K' need no state: helix_delta_prep_* forms them for all chunks at once.
// helix_delta_walk_* then goes through the chunks of a sequence, a workgroup for 16 or 32 columns
// of a head's state, whose columns do not meet.
//
// 8192 tokens of 64 heads of 128 x 64 in bf16: 318 us, where memory's part is 34 (174 MB). 28 us
// form the first segment's operands, the rest are 128 steps of the walk (below).
#include "delta_common.h"

namespace {

// ---- token by token -----------------------------------------------------------------------
//
// A workgroup has 64 columns of a state in registers: lane 16 kg + cl of wave w columns
// 4 cl .. + 3 of the rows 16 i + 4 w + kg. k'S and q'S are summed over a token's old state
// together (q'S' = e^g q'S + (q . k) d), so that a token meets one barrier. Memory binds a
// batch of single tokens (the state is read and written once: 64 of 64 heads of 128 x 64, 270 MB,
// 47 us, 5.7 TB/s with the cache's part), latency few sequences (one token of one 5.2 us, 1.1 to
// 1.4 for each that follows: the loads of its row, nine sums over lanes and a meeting in LDS).
template <typename T, int NR>
__device__ void delta_steps(const HelixDeltaParams& p) {
    __shared__ float kq[2][HELIX_DR_STEPS][16 * NR];
    __shared__ float red[2][4][16][12];
    const int tid = threadIdx.x, cl = tid & 15, kg = tid >> 4, w = wave_uniform();
    const int slices = (p.n_val + 63) / 64;
    const int slice = blockIdx.x % slices;
    const long long sh = blockIdx.x / slices;
    const long long seq = sh / p.n_head;
    const int h = (int)(sh % p.n_head), hk = h / p.share;
    const int p0 = 64 * slice + 4 * cl, own = min(4, p.n_val - p0);
    const unsigned bytes = (unsigned)p.n_key * (unsigned)p.n_val * 4u;
    f32x4 S[NR];
    {
        const helix_rsrc r = make_rsrc_u(p.s0 + sh * p.n_key * p.n_val, p.s0 ? bytes : 0u);   // none: reads 0
#pragma unroll
        for (int i = 0; i < NR; ++i)
            S[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                 r, own > 0 ? ((16 * i + kg) * p.n_val + p0) * 4 : (int)0x80000000, 0, 0));
    }
    const T* q = static_cast<const T*>(p.q) + seq * p.seq_q + hk * p.head_q;
    const T* k = static_cast<const T*>(p.k) + seq * p.seq_k + hk * p.head_k;
    const T* v = static_cast<const T*>(p.v) + seq * p.seq_v + h * p.head_v;
    T* o = static_cast<T*>(p.o) + seq * p.seq_o + h * p.head_o;
    const float* g = p.g + seq * p.seq_g + h;
    const float* beta = p.beta + seq * p.seq_b + h;
    float vn[4], gn = 0.0f, bn = 0.0f;
    auto ahead = [&](int t) {
        if (t >= p.n_tok) return;
        gn = g[t * p.tok_g];
        bn = beta[t * p.tok_b];
#pragma unroll
        for (int c = 0; c < 4; ++c) vn[c] = c < own ? (float)v[t * p.tok_v + p0 + c] : 0.0f;
    };
    ahead(0);
    for (int t0 = 0; t0 < p.n_tok; t0 += HELIX_DR_STEPS) {
        const int len = min(HELIX_DR_STEPS, p.n_tok - t0);
        if (t0) __syncthreads();
        for (int i = tid; i < len * 16 * NR; i += 256) {
            const int t = i / (16 * NR), n = i % (16 * NR);
            kq[0][t][n] = n < p.n_key ? (float)k[(t0 + t) * p.tok_k + n] : 0.0f;
            kq[1][t][n] = n < p.n_key ? (float)q[(t0 + t) * p.tok_q + n] : 0.0f;
        }
        __syncthreads();
        for (int t = 0; t < len; ++t) {
            float vt[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) vt[c] = vn[c];
            const float a = expf(gn), b = bn;
            ahead(t0 + t + 1);
            float kn[NR], part[9];
#pragma unroll
            for (int j = 0; j < 9; ++j) part[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                kn[i] = kq[0][t][16 * i + kg];
                const float qn = kq[1][t][16 * i + kg];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    part[c] = fmaf(kn[i], S[i][c], part[c]);
                    part[4 + c] = fmaf(qn, S[i][c], part[4 + c]);
                }
                part[8] = fmaf(qn, kn[i], part[8]);
            }
#pragma unroll
            for (int j = 0; j < 9; ++j) {
                part[j] += __shfl_xor(part[j], 16, 64);
                part[j] += __shfl_xor(part[j], 32, 64);
            }
            // (Two places in turn: a wave may be at the next token while another reads this one's.)
            float (&rd)[4][16][12] = red[t & 1];
            if ((kg & 3) == 0) {
#pragma unroll
                for (int j = 0; j < 9; ++j) rd[w][cl][j] = part[j];
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 9; ++j) part[j] = (rd[0][cl][j] + rd[1][cl][j]) + (rd[2][cl][j] + rd[3][cl][j]);
            float d[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) d[c] = b * (vt[c] - a * part[c]);
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) S[i][c] = fmaf(a, S[i][c], kn[i] * d[c]);
            if (kg == 0) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c < own) o[(t0 + t) * p.tok_o + p0 + c] = (T)(p.scale * (a * part[4 + c] + part[8] * d[c]));
            }
        }
    }
    const helix_rsrc r = make_rsrc_u(p.s + sh * p.n_key * p.n_val, bytes);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int n = 16 * i + kg, off = (n * p.n_val + p0) * 4;
        if (n >= p.n_key) continue;
        if (own >= 4) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, S[i]), r, off, 0, 0);
        } else {
#pragma unroll
            for (int c = 0; c < 3; ++c)
                if (c < own) __builtin_amdgcn_raw_buffer_store_b32(as_u32(S[i][c]), r, off + 4 * c, 0, 0);
        }
    }
}

// ---- X and P ------------------------------------------------------------------------------

// 16 x 16 x 16 in fp32, c += a b: a[r] = A[c][4 q + r] of the lane, b a result's registers. (The sum's order, 4 q + r for
// step r and group q, is the same on both sides.)
HELIX_DEV f32x4 dr_mfma_f32(const f32x4& a, const f32x4& b, f32x4 c) {
#pragma unroll
    for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
    return c;
}

constexpr int DR_LD = DR_C + 4;   // fp32 rows of a chunk's square matrices in LDS

// A workgroup a chunk of a head. Wave w: rows 16 w .. of K K' and Q K'; the inverse of A's diagonal block w by forward
// substitution, a column a lane; then block column w of the inverse, from the diagonal down:
//     T_iw = -T_ii (sum over j of A_ij T_jw),  w <= j < i
// on fp32 matrix instructions, T_jw staying in the registers it was formed in. (Products of powers of A would be fewer steps,
// but keys that repeat make the powers large, and they cancel.) BWD: T' and P' with X, without P.
// Four workgroups a CU hide one another's chains: P takes the place of K's parts in LDS, T that of A (twice as fast as two a
// CU). 2048 tokens of 64 heads, bf16, 128 keys: 27 us, the writing of 37 KB a chunk at 2.8 TB/s.
template <typename T, int NK>
struct PrepLds {
    union {
        __bf16 k[dr_planes<T> * DR_C * NK];
        float p[DR_C][DR_LD];
    };
    float a[DR_C][DR_LD], d[4][16][20], b[DR_C];
    double g[DR_C];
};
template <typename T, int NK, bool ODD, bool BWD>
__device__ void delta_prep(const HelixDeltaParams& p, unsigned id, PrepLds<T, NK>& lds) {
    constexpr int NPL = dr_planes<T>;
    __bf16* const sK = lds.k;
    auto &sP = lds.p, &sA = lds.a;
    auto& sD = lds.d;
    auto& sG = lds.g;
    auto& sB = lds.b;
    // (Wave w has w + 1 blocks of the products: turned from workgroup to workgroup, every SIMD gets each.)
    const int tid = threadIdx.x, lane = lane_id(), w = (wave_uniform() + (int)id) & 3, c = lane & 15, q = lane >> 4;
    const int ch = (int)(id % (unsigned)p.n_chunk);
    const unsigned sh = id / (unsigned)p.n_chunk;
    const int seq = (int)(sh / (unsigned)p.n_head), h = (int)(sh % (unsigned)p.n_head), hk = h / p.share;
    const long long t0 = (long long)(p.chunk0 + ch) * DR_C;
    const int len = (int)min((long long)DR_C, p.n_tok - t0);
    const Rows<T, ODD> rk(p.k, seq * p.seq_k + hk * p.head_k + t0 * p.tok_k, p.tok_k, len, p.n_key);
    const Rows<T, ODD> rq(p.q, seq * p.seq_q + hk * p.head_q + t0 * p.tok_q, p.tok_q, len, p.n_key);
    // K's parts into LDS; the wave's rows of Q in registers.
    constexpr int PER = DR_C * (NK / 8) / 256;
    Raw8<T> kr[PER], qr[NK / 32];
#pragma unroll
    for (int i = 0; i < PER; ++i) kr[i] = rk.load8((tid + 256 * i) / (NK / 8), 8 * ((tid + 256 * i) % (NK / 8)));
#pragma unroll
    for (int s = 0; s < NK / 32; ++s) qr[s] = rq.load8(16 * w + c, 32 * s + 8 * q);
    if (w == 0) {
        const float gl = lane < len ? p.g[seq * p.seq_g + (t0 + lane) * p.tok_g + h] : 0.0f;
        const float bl = lane < len ? p.beta[seq * p.seq_b + (t0 + lane) * p.tok_b + h] : 0.0f;
        const double G = dr_log_decay(gl);
        const double end = __shfl(G, 63, 64);
        sG[lane] = G * 1.4426950408889634074;
        sB[lane] = bl;
        float* dec = p.decay + id * (HELIX_DR_DECAY / 4ll);
        dec[lane] = exp_diff(G, 0.0);
        dec[64 + lane] = exp_diff(end, G);
        dec[128 + lane] = bl;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int row = (tid + 256 * i) / (NK / 8), col = 8 * ((tid + 256 * i) % (NK / 8));
        bf16x8 o[NPL];
        dr_operand<T>(kr[i], p.n_key - col, o);
        dr_put8<NPL, NK, DR_C>(sK, row, col, o);
    }
    __syncthreads();
    DrAcc kk[4], qk[4];
#pragma unroll
    for (int s = 0; s < NK / 32; ++s) {
        const int col = 32 * s + 8 * q;
        bf16x8 ak[NPL], aq[NPL];
        dr_get8<NPL, NK, DR_C>(sK, 16 * w + c, col, ak);
        dr_operand<T>(qr[s], p.n_key - col, aq);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > w) break;
            bf16x8 b[NPL];
            dr_get8<NPL, NK, DR_C>(sK, 16 * j + c, col, b);
            dr_mfma<NPL, NPL>(ak, b, kk[j]);
            dr_mfma<NPL, NPL>(aq, b, qk[j]);
        }
    }
    f32x4 pv[4];
    {
        double Gi[4];
        const f32x4 beta = *reinterpret_cast<const f32x4*>(&sB[16 * w + 4 * q]);
#pragma unroll
        for (int r = 0; r < 4; ++r) Gi[r] = sG[16 * w + 4 * q + r];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > w) break;
            const double Gj = sG[16 * j + c];
            const f32x4 k = dr_sum<NPL>(kk[j]), x = dr_sum<NPL>(qk[j]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float e = __builtin_amdgcn_exp2f((float)(Gi[r] - Gj));
                float a = beta[r] * (e * k[r]);
                if (j == w) {
                    if (c > 4 * q + r) e = 0.0f;
                    if (c >= 4 * q + r) a = 0.0f;
                }
                pv[j][r] = j == w && c > 4 * q + r ? 0.0f : p.scale * (e * x[r]);
                sA[16 * w + 4 * q + r][16 * j + c] = a;
            }
        }
    }
    __syncthreads();
    // P by rows, 0 above the diagonal where fragments reach.
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j > (w | 1)) break;
#pragma unroll
        for (int r = 0; r < 4; ++r) sP[16 * w + 4 * q + r][16 * j + c] = j <= w ? pv[j][r] : 0.0f;
    }
    // Diagonal block w: lane c its column c (the four groups alike), four rows at a time.
    {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = i == c ? 1.0f : 0.0f;
#pragma unroll
        for (int jb = 0; jb < 16; jb += 4) {
#pragma unroll
            for (int i = jb + 1; i < 16; ++i) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(&sA[16 * w + i][16 * w + jb]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (jb + j < i) x[i] = fmaf(-a[j], x[jb + j], x[i]);
            }
        }
        if (q == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sD[w][i][c] = x[i];
        }
    }
    __syncthreads();
    f32x4 t[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) t[0][r] = sD[w][4 * q + r][c];
#pragma unroll
    for (int step = 1; step < 4; ++step) {
        const int i = w + step;
        if (i > 3) break;
        f32x4 m = zero4();
#pragma unroll
        for (int j = 0; j < step; ++j)
            m = dr_mfma_f32(*reinterpret_cast<const f32x4*>(&sA[16 * i + c][16 * (w + j) + 4 * q]), t[j], m);
        const f32x4 a = *reinterpret_cast<const f32x4*>(&sD[i][c][4 * q]);
        t[step] = dr_mfma_f32(-a, m, zero4());
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            // (t[i - w], by a choice of constants.)
            const float v = i < w ? 0.0f : i == w ? t[0][r] : i == w + 1 ? t[1][r] : i == w + 2 ? t[2][r] : t[3][r];
            sA[16 * i + 4 * q + r][16 * w + c] = v;
        }
    __syncthreads();
    // Fragments: row 16 w + c, columns 32 ks + 8 q ..
    auto emit = [&](char* to, int frag, const float (&v)[8]) {
        bf16x8 o[3];
        dr_split8<3>(v, o);
#pragma unroll
        for (int k = 0; k < 3; ++k)
            *reinterpret_cast<bf16x8*>(to + ((long long)id * 18 + frag * 3 + k) * HELIX_DR_FRAG + 16 * lane) = o[k];
    };
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        float v[8];
        const int row = 16 * w + c, col = 32 * ks + 8 * q;
        if (ks == 0 || w > 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = sA[row][col + e] * sB[col + e];
            emit(p.x, dr_low(w, ks), v);
            if constexpr (!BWD) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = sP[row][col + e];
                emit(p.p, dr_low(w, ks), v);
            }
        }
        if constexpr (BWD) {
            if (ks == 1 || w < 2) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = sA[col + e][row];
                emit(p.tt, dr_up(w, ks), v);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = sP[col + e][row];
                emit(p.pt, dr_up(w, ks), v);
            }
        }
    }
}

// ---- the walk -----------------------------------------------------------------------------
//
// Sixteen columns of a state, and two kinds of waves. The first four carry the state: wave w
// forms rows 16 w .. of K S, of R = V - e^G K S and of D = X R, and keeps the rows NK / 4 w ..
// of S in registers. The other four do what nothing waits for: they bring K's rows into LDS
// and form the outputs, a phase behind. S, R, D and e^(G_63 - G) D go from wave to wave
// through LDS, in bf16 parts and with the index that the next product sums over running inside
// a row. A chunk is three barriers; what does not depend on the state is loaded as soon as the
// chunk before has used its registers. K is read in the first phase alone (K' as operands of
// the third is kept in registers), so that its next rows can take its place.
// What bounds it is the chain of a chunk: three products that wait for one another, each with its
// way through LDS, beside 70 KB of loads into the CU. 2048 tokens of 64 heads of 128 x 64, bf16,
// 32 chunks: 70 us, 2.2 a chunk; without the loads 1.7, without the outputs 1.6, the state's waves
// alone 1.4. Tried on earlier forms, of the time of a whole prompt of 8192 tokens: the two kinds
// of waves 0.76, rows in LDS turned by their number (dr_at) with V and outputs through LDS 0.82. No
// gain: loads two chunks ahead, LDS reads moved before the barriers, priorities of the waves. Slower:
// Q S in the second phase (1.28 of the walk's time), K's operands straight from memory (1.35).
// With 32 columns a product's operands are loaded and split once for two blocks of columns
// (32 chunks of 256 heads, KEEP: 240 us with 16 columns, 167 with 32 and two workgroups a CU).
// KEEP: no outputs and no waves for them; the states before the chunks and D are stored (fp32)
// for the backward pass.
template <typename T, int NK, bool KEEP, int NC>
struct WalkLds {
    static constexpr int COLS = 16 * NC;   // columns of the workgroup
    typedef typename std::conditional<KEEP, float, T>::type Out;   // D, or o
    __bf16 k[dr_planes<T> * DR_C * NK], s[3 * COLS * NK], r[3 * COLS * DR_C], u[3 * COLS * DR_C];
    __bf16 d[KEEP ? 8 : 3 * COLS * DR_C];
    T v[DR_C][COLS + 16 / sizeof(T)];
    float dec[2][HELIX_DR_DECAY / 4];
    Out out[DR_C][COLS + 16 / sizeof(Out)];
};
template <typename T, int NK, bool ODD, bool KEEP, int NC>
__device__ void delta_walk(const HelixDeltaParams& p, WalkLds<T, NK, KEEP, NC>& lds) {
    constexpr int NPL = dr_planes<T>, NT = NK / 64, KS = NK / 32;
    constexpr int COLS = 16 * NC;
    typedef typename WalkLds<T, NK, KEEP, NC>::Out Out;
    __bf16 *const sK = lds.k, *const sS = lds.s, *const sR = lds.r, *const sU = lds.u, *const sD = lds.d;
    auto& sV = lds.v;
    auto& sDec = lds.dec;
    auto& sOut = lds.out;
    const int tid = threadIdx.x & 255, lane = lane_id(), w = wave_uniform() & 3, c = lane & 15, q = lane >> 4;
    const unsigned id = xcd_logical_id(blockIdx.x, p.n_walk);   // a head's slices share an XCD's cache
    const int slice = (int)(id % (unsigned)p.n_slice);
    const unsigned sh = id / (unsigned)p.n_slice;
    const int seq = (int)(sh / (unsigned)p.n_head), h = (int)(sh % (unsigned)p.n_head), hk = h / p.share;
    const int p0 = COLS * slice, P = p.n_val, N = p.n_key;
    const unsigned state_bytes = (unsigned)N * (unsigned)P * 4u;
    const int row0 = 16 * w + 4 * q, last = p.n_chunk - 1;
    const long long base = (long long)sh * p.n_chunk;
    auto first = [&](int ch) { return (long long)(p.chunk0 + ch) * DR_C; };
    auto tokens = [&](int ch) { return (int)min((long long)DR_C, p.n_tok - first(ch)); };

    if (wave_uniform() >= 4) {
        // K's rows, the columns of V's (two or four lanes a row) and the decays: loaded, and laid out in LDS.
        constexpr int PER = DR_C * (NK / 8) / 256;
        Raw8<T> kr[PER], vr;
        f32x4 dec;
        // (The addresses of all this are formed where they are used: kept, they would take a second workgroup's registers.)
        auto load_k = [&](int ch) {
            const int tid = vgpr_fresh(threadIdx.x) & 255, vrow = tid / (2 * NC) & 63, vcol = 8 * (tid % (2 * NC));
            ch = min(ch, last);
            const Rows<T, ODD> rk(p.k, seq * p.seq_k + hk * p.head_k + first(ch) * p.tok_k, p.tok_k, tokens(ch), N);
            const Rows<T, ODD> rv(p.v, seq * p.seq_v + h * p.head_v + first(ch) * p.tok_v, p.tok_v, tokens(ch), P);
#pragma unroll
            for (int i = 0; i < PER; ++i) kr[i] = rk.load8((tid + 256 * i) / (NK / 8), 8 * ((tid + 256 * i) % (NK / 8)));
            if (tid < 128 * NC) vr = rv.load8(vrow, p0 + vcol);
            if (tid >= 256 - HELIX_DR_DECAY / 16)
                dec = *reinterpret_cast<const f32x4*>(p.decay + (base + ch) * (HELIX_DR_DECAY / 4) + 4 * (tid - (256 - HELIX_DR_DECAY / 16)));
        };
        auto put_k = [&](int ch) {
            const int tid = vgpr_fresh(threadIdx.x) & 255, vrow = tid / (2 * NC) & 63, vcol = 8 * (tid % (2 * NC));
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int row = (tid + 256 * i) / (NK / 8), col = 8 * ((tid + 256 * i) % (NK / 8));
                bf16x8 o[NPL];
                dr_operand<T>(kr[i], N - col, o);
                dr_put8<NPL, NK, DR_C>(sK, row, col, o);
            }
            if (tid < 128 * NC) *reinterpret_cast<Raw8<T>*>(&sV[vrow][vcol]) = vr;
            if (tid >= 256 - HELIX_DR_DECAY / 16) *reinterpret_cast<f32x4*>(&sDec[ch & 1][4 * (tid - (256 - HELIX_DR_DECAY / 16))]) = dec;
        };
        // What a chunk left in sOut, by the lanes that have V's places.
        auto store_out = [&](int ch) {
            const int tid = vgpr_fresh(threadIdx.x) & 255, vrow = tid / (2 * NC) & 63, vcol = 8 * (tid % (2 * NC));
            if (tid >= 128 * NC) return;
            const Raw8<Out> v = *reinterpret_cast<const Raw8<Out>*>(&sOut[vrow][vcol]);
            if constexpr (KEEP) {
                store8_at<float>(p.keep_d + ((base + ch) * DR_C + vrow) * P + p0 + vcol, v, P - p0 - vcol);
            } else if (vrow < tokens(ch)) {
                store8_at<T>(static_cast<T*>(p.o) + seq * p.seq_o + h * p.head_o + (first(ch) + vrow) * p.tok_o + p0 + vcol, v,
                             P - p0 - vcol);
            }
        };
        Raw8<T> qr[KS];
        bf16x8 pf[2][3];
        auto load_q = [&](int ch) {
            const int tid = vgpr_fresh(threadIdx.x) & 255, c = tid & 15, q = (tid & 63) >> 4;
            ch = min(ch, last);
            const Rows<T, ODD> rq(p.q, seq * p.seq_q + hk * p.head_q + first(ch) * p.tok_q, p.tok_q, tokens(ch), N);
#pragma unroll
            for (int s = 0; s < KS; ++s) qr[s] = rq.load8(16 * w + c, 32 * s + 8 * q);
        };
        auto load_p = [&](int ch) {
            const char* pp = p.p + (base + min(ch, last)) * (6 * 3 * HELIX_DR_FRAG) + 16 * lane;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                if (ks && w < 2) break;
#pragma unroll
                for (int k = 0; k < 3; ++k) pf[ks][k] = *reinterpret_cast<const bf16x8*>(pp + (dr_low(w, ks) * 3 + k) * HELIX_DR_FRAG);
            }
        };
        load_k(0);
        if constexpr (!KEEP) {
            load_q(0);
            load_p(0);
        }
        put_k(0);
        load_k(1);
        for (int ch = 0; ch <= last; ++ch) {
            dr_barrier();   // K, V and S are there
            f32x4 o[NC];
            if constexpr (!KEEP) {
                typename DrAccOf<NC>::type qs[NC];
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int col = 32 * s + 8 * q;
                    bf16x8 a[NPL], b[3];
                    dr_operand<T>(qr[s], N - col, a);
#pragma unroll
                    for (int n = 0; n < NC; ++n) {
                        dr_get8<3, NK, COLS>(sS, 16 * n + c, col, b);
                        dr_mfma<NPL, 3>(a, b, qs[n]);
                    }
                }
                const f32x4 start = p.scale * *reinterpret_cast<const f32x4*>(&sDec[ch & 1][row0]);
#pragma unroll
                for (int n = 0; n < NC; ++n) o[n] = qs[n].sum() * start;
                load_q(ch + 1);
            }
            if (ch) store_out(ch - 1);
            dr_barrier();   // R is there; K and V have been read
            put_k(ch + 1);
            load_k(ch + 2);
            dr_barrier();   // D is there
            if constexpr (!KEEP) {
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    if (ks && w < 2) break;
#pragma unroll
                    for (int n = 0; n < NC; ++n) {
                        bf16x8 b[3];
                        dr_get8<3, DR_C, COLS>(sD, 16 * n + c, 32 * ks + 8 * q, b);
                        o[n] = dr_mfma<3, 3>(pf[ks], b, o[n]);
                    }
                }
                load_p(ch + 1);
#pragma unroll
                for (int n = 0; n < NC; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sOut[row0 + r][16 * n + c] = (T)o[n][r];
            }
        }
        dr_barrier();   // the last outputs are there
        if (last >= 0) store_out(last);
        return;
    }

    // Register r of tile i, columns n: S[NT 16 w + 16 i + 4 q + r][p0 + 16 n + c].
    auto state_off = [&](int i, int n, int r) {
        const int row = NT * 16 * w + 16 * i + 4 * q + r, col = p0 + 16 * n + c;
        return row < N && col < P ? (row * P + col) * 4 : (int)0x80000000;
    };
    f32x4 S[NT][NC];
    bf16x8 xf[2][3];
    auto put_state = [&](helix_rsrc to) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) __builtin_amdgcn_raw_buffer_store_b32(as_u32(S[i][n][r]), to, state_off(i, n, r), 0, 0);
    };
    auto load_x = [&](int ch) {
        const char* x = p.x + (base + min(ch, last)) * (6 * 3 * HELIX_DR_FRAG) + 16 * lane;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (ks && w < 2) break;
#pragma unroll
            for (int k = 0; k < 3; ++k) xf[ks][k] = *reinterpret_cast<const bf16x8*>(x + (dr_low(w, ks) * 3 + k) * HELIX_DR_FRAG);
        }
    };
    auto put_s = [&] {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int n = 0; n < NC; ++n)
                dr_put4<3, NK, COLS>(sS, 16 * n + c, NT * 16 * w + 16 * i + 4 * q, S[i][n][0], S[i][n][1], S[i][n][2], S[i][n][3]);
    };
    {
        const helix_rsrc r0 = make_rsrc_u(p.s0 + (long long)sh * N * P, p.s0 ? state_bytes : 0u);   // none: reads 0
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[i][n][r] = buf_f32(r0, state_off(i, n, r), 0);
    }
    load_x(0);
    put_s();
    for (int ch = 0; ch <= last; ++ch) {
        dr_barrier();   // K, V and S are there
        if constexpr (KEEP) put_state(make_rsrc_u(p.keep_s + (base + ch) * N * P, state_bytes));
        const float* const dec = sDec[ch & 1];
        typename DrAccOf<NC>::type ks_[NC];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int col = 32 * s + 8 * q;
            bf16x8 a[NPL], b[3];
            dr_get8<NPL, NK, DR_C>(sK, 16 * w + c, col, a);
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                dr_get8<3, NK, COLS>(sS, 16 * n + c, col, b);
                dr_mfma<NPL, 3>(a, b, ks_[n]);
            }
        }
        bf16x8 kt[2][NT][NPL];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < NT; ++i) dr_get8_t<NPL, NK, DR_C>(sK, 32 * ks + 8 * q, NT * 16 * w + 16 * i, c, kt[ks][i]);
        const f32x4 start = *reinterpret_cast<const f32x4*>(dec + row0);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            f32x4 R = ks_[n].sum();
#pragma unroll
            for (int r = 0; r < 4; ++r) R[r] = (float)sV[row0 + r][16 * n + c] - start[r] * R[r];
            dr_put4<3, DR_C, COLS, sizeof(T) == 4>(sR, 16 * n + c, row0, R[0], R[1], R[2], R[3]);   // (V at the end of fp32)
        }
        dr_barrier();   // R is there; K and V have been read
        typename DrAccOf<NC>::type ds[NC];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (ks && w < 2) break;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                bf16x8 b[3];
                dr_get8<3, DR_C, COLS>(sR, 16 * n + c, 32 * ks + 8 * q, b);
                dr_mfma<3, 3>(xf[ks], b, ds[n]);
            }
        }
        const f32x4 left = *reinterpret_cast<const f32x4*>(dec + 64 + row0);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const f32x4 D = ds[n].sum();
            dr_put4<3, DR_C, COLS>(sU, 16 * n + c, row0, D[0] * left[0], D[1] * left[1], D[2] * left[2], D[3] * left[3]);
            if constexpr (KEEP) {
#pragma unroll
                for (int r = 0; r < 4; ++r) sOut[row0 + r][16 * n + c] = D[r];
            } else {
                dr_put4<3, DR_C, COLS>(sD, 16 * n + c, row0, D[0], D[1], D[2], D[3]);
            }
        }
        load_x(ch + 1);
        const float all = dec[63];
        dr_barrier();   // D is there
        typename DrAccOf<NC>::type up[NT][NC];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                bf16x8 b[3];
                dr_get8<3, DR_C, COLS>(sU, 16 * n + c, 32 * ks + 8 * q, b);
#pragma unroll
                for (int i = 0; i < NT; ++i) dr_mfma<NPL, 3>(kt[ks][i], b, up[i][n]);
            }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int n = 0; n < NC; ++n) S[i][n] = all * S[i][n] + up[i][n].sum();
        put_s();
    }
    dr_barrier();
    if (p.s) put_state(make_rsrc_u(p.s + (long long)sh * N * P, state_bytes));
}

template <typename T, int NK, bool ODD, bool BWD>
__device__ void prep_kernel(const HelixDeltaParams& p) {
    __shared__ __attribute__((aligned(16))) PrepLds<T, NK> lds;
    delta_prep<T, NK, ODD, BWD>(p, blockIdx.x, lds);
}
template <typename T, int NK, bool ODD, bool KEEP, int NC>
__device__ void walk_kernel(const HelixDeltaParams& p) {
    __shared__ __attribute__((aligned(16))) WalkLds<T, NK, KEEP, NC> lds;
    delta_walk<T, NK, ODD, KEEP, NC>(p, lds);
}

// A walk whose workgroups leave room on every CU, and behind it the operands of the chunks that the next walk takes: 32 chunks
// of 64 heads take 70 us by themselves, and 94 with the next 32 chunks' operands, which are 28 in a launch of their own.
template <typename T, int NK, bool ODD>
__device__ void delta_walk_ahead(const HelixDeltaParams& p) {
    if constexpr (sizeof(T) == 4) return walk_kernel<T, NK, ODD, false, 1>(p);   // (fp32's take a CU's LDS and registers)
    __shared__ __attribute__((aligned(16))) union {
        WalkLds<T, NK, false, 1> walk;
        PrepLds<T, NK> prep;
    } lds;
    if (blockIdx.x < p.n_walk) return delta_walk<T, NK, ODD, false, 1>(p, lds.walk);
    if (threadIdx.x >= 256) return;   // (barriers wait for the waves that are left)
    HelixDeltaParams n = p;
    n.chunk0 += n.n_chunk;
    n.n_chunk = n.n_next;
    n.x = n.next_x;
    n.p = n.next_p;
    n.decay = n.next_decay;
    delta_prep<T, NK, ODD, false>(n, blockIdx.x - p.n_walk, lds.prep);
}

// ---- backward -----------------------------------------------------------------------------
//
// With dO, and E the gradient of the state after a chunk (dS of the one before it, or the
// caller's):
//     dD = P' dO + (e^(G_63 - G) K) E,   Z = T' dD,   dV = beta Z
//     dS = e^(G_63) E + scale (e^G Q)' dO - (e^G K)' dV
// from the last chunk to the first: helix_delta_back_*, spread and laid out as the walk. Its
// second four waves bring K, Q and dO and form what does not wait for E, P' dO and
// scale (e^G Q)' dO of the chunk after the one that the first four are at. It leaves E and Z for
// the kernels below. Bound as the walk is: 32 chunks of 256 heads of 128 x 64, bf16, 333 us with 16
// columns a workgroup, 257 with 32.
template <typename T, int NK, bool ODD, int NC>
__device__ void delta_back(const HelixDeltaParams& p) {
    constexpr int NPL = dr_planes<T>, NT = NK / 64, KS = NK / 32, COLS = 16 * NC;
    __shared__ __attribute__((aligned(16))) __bf16 sK[NPL * DR_C * NK], sQ[NPL * DR_C * NK], sE[3 * COLS * NK];
    __shared__ __attribute__((aligned(16))) __bf16 sO[NPL * COLS * DR_C], sW[3 * COLS * DR_C], sR[3 * COLS * DR_C], sU[3 * COLS * DR_C];
    __shared__ f32x4 sPO[NC][4][64], sQW[NC][NT][4][64];   // P' dO, where Z then is, and Q' (scale e^G dO), as lanes hold them
    __shared__ __attribute__((aligned(16))) float sDec[2][HELIX_DR_DECAY / 4];
    const int tid = threadIdx.x & 255, lane = lane_id(), w = wave_uniform() & 3, c = lane & 15, q = lane >> 4;
    const unsigned id = xcd_logical_id(blockIdx.x, gridDim.x);
    const int slice = (int)(id % (unsigned)p.n_slice);
    const unsigned sh = id / (unsigned)p.n_slice;
    const int seq = (int)(sh / (unsigned)p.n_head), h = (int)(sh % (unsigned)p.n_head), hk = h / p.share;
    const int p0 = COLS * slice, P = p.n_val, N = p.n_key;
    const unsigned state_bytes = (unsigned)N * (unsigned)P * 4u;
    const int row0 = 16 * w + 4 * q, last = p.n_chunk - 1;
    const long long base = (long long)sh * p.n_chunk;
    auto first = [&](int ch) { return (long long)(p.chunk0 + ch) * DR_C; };
    auto tokens = [&](int ch) { return (int)min((long long)DR_C, p.n_tok - first(ch)); };

    if (wave_uniform() >= 4) {
        if (last < 0) return;
        constexpr int PER = DR_C * (NK / 8) / 256;
        Raw8<T> kr[PER], qr[PER];
        bf16x8 pf[2][3];
        unsigned vo[NC][4];
        f32x4 start, dec;
        // (The addresses of all this are formed where they are used: kept, they would take a second workgroup's registers.)
        auto load_q = [&](int ch) {   // Q's rows, dO and its decays
            const int tid = vgpr_fresh(threadIdx.x) & 255, c = tid & 15, row0 = tid >> 4 << 2;
            ch = max(ch, 0);
            const Rows<T, ODD> rq(p.q, seq * p.seq_q + hk * p.head_q + first(ch) * p.tok_q, p.tok_q, tokens(ch), N);
            const Rows<T> ro(p.d_o, seq * p.seq_o + h * p.head_o + first(ch) * p.tok_o, p.tok_o, tokens(ch), P);
#pragma unroll
            for (int i = 0; i < PER; ++i) qr[i] = rq.load8((tid + 256 * i) / (NK / 8), 8 * ((tid + 256 * i) % (NK / 8)));
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) vo[n][r] = ro.raw(row0 + r, p0 + 16 * n + c);
            start = *reinterpret_cast<const f32x4*>(p.decay + (base + ch) * (HELIX_DR_DECAY / 4) + row0);
        };
        auto load_k = [&](int ch) {   // K's rows, all decays, and the fragments of P'
            const int tid = vgpr_fresh(threadIdx.x) & 255, lane = tid & 63;
            ch = max(ch, 0);
            const Rows<T, ODD> rk(p.k, seq * p.seq_k + hk * p.head_k + first(ch) * p.tok_k, p.tok_k, tokens(ch), N);
#pragma unroll
            for (int i = 0; i < PER; ++i) kr[i] = rk.load8((tid + 256 * i) / (NK / 8), 8 * ((tid + 256 * i) % (NK / 8)));
            if (tid < HELIX_DR_DECAY / 16) dec = *reinterpret_cast<const f32x4*>(p.decay + (base + ch) * (HELIX_DR_DECAY / 4) + 4 * tid);
            const char* pt = p.pt + (base + ch) * (6 * 3 * HELIX_DR_FRAG) + 16 * lane;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                if (ks == 0 && w > 1) continue;
#pragma unroll
                for (int k = 0; k < 3; ++k) pf[ks][k] = *reinterpret_cast<const bf16x8*>(pt + (dr_up(w, ks) * 3 + k) * HELIX_DR_FRAG);
            }
        };
        auto put_rows = [&](__bf16* to, const Raw8<T> (&v)[PER]) {
            const int tid = vgpr_fresh(threadIdx.x) & 255;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int row = (tid + 256 * i) / (NK / 8), col = 8 * ((tid + 256 * i) % (NK / 8));
                bf16x8 o[NPL];
                dr_operand<T>(v[i], N - col, o);
                dr_put8<NPL, NK, DR_C>(to, row, col, o);
            }
        };
        auto put_q = [&] {
            put_rows(sQ, qr);
            const int tid = vgpr_fresh(threadIdx.x) & 255, c = tid & 15, row0 = tid >> 4 << 2;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                float o[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = raw_f32<T>(vo[n][r]);
                dr_put4<NPL, DR_C, COLS, sizeof(T) == 4>(sO, 16 * n + c, row0, o[0], o[1], o[2], o[3]);
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] *= p.scale * start[r];
                dr_put4<3, DR_C, COLS, sizeof(T) == 4>(sW, 16 * n + c, row0, o[0], o[1], o[2], o[3]);   // (dO at the end of fp32)
            }
        };
        auto put_k = [&](int ch) {
            put_rows(sK, kr);
            if (tid < HELIX_DR_DECAY / 16) *reinterpret_cast<f32x4*>(&sDec[ch & 1][4 * tid]) = dec;
        };
        f32x4 po[NC], qw[NC][NT];
        auto form = [&] {
            const int fresh = vgpr_fresh(lane), c = fresh & 15, q = fresh >> 4;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                po[n] = zero4();
#pragma unroll
                for (int i = 0; i < NT; ++i) qw[n][i] = zero4();
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                if (ks == 1 || w < 2) {
#pragma unroll
                    for (int n = 0; n < NC; ++n) {
                        bf16x8 o[NPL];
                        dr_get8<NPL, DR_C, COLS>(sO, 16 * n + c, 32 * ks + 8 * q, o);
                        po[n] = dr_mfma<3, NPL>(pf[ks], o, po[n]);
                    }
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    bf16x8 a[NPL];
                    dr_get8_t<NPL, NK, DR_C>(sQ, 32 * ks + 8 * q, NT * 16 * w + 16 * i, c, a);
#pragma unroll
                    for (int n = 0; n < NC; ++n) {
                        bf16x8 b[3];
                        dr_get8<3, DR_C, COLS>(sW, 16 * n + c, 32 * ks + 8 * q, b);
                        qw[n][i] = dr_mfma<NPL, 3>(a, b, qw[n][i]);
                    }
                }
            }
        };
        auto leave = [&] {
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                sPO[n][w][lane] = po[n];
#pragma unroll
                for (int i = 0; i < NT; ++i) sQW[n][i][w][lane] = qw[n][i];
            }
        };
        load_q(last);
        load_k(last);
        put_q();
        put_k(last);
        load_q(last - 1);
        dr_barrier();
        form();
        leave();
        load_k(last - 1);
        for (int ch = last; ch >= 0; --ch) {
            dr_barrier();   // K, E and what does not depend on E are there
            if (ch) put_q();
            load_q(ch - 2);
            dr_barrier();   // dD is there; K has been read
            if (ch) form();
            put_k(ch - 1);
            load_k(ch - 2);
            dr_barrier();   // dV is there
            const int tid = vgpr_fresh(threadIdx.x) & 255, lane = tid & 63, c = tid & 15, row0 = tid >> 4 << 2;
            const f32x4 beta = *reinterpret_cast<const f32x4*>(&sDec[ch & 1][128 + row0]);
            const Rows<float> rz(p.keep_z, (base + ch) * DR_C * P, P, DR_C, P);
            const Rows<T> rv(p.dv, (((long long)seq * p.n_tok + first(ch)) * p.row_head + h) * P, (long long)p.row_head * P, tokens(ch), P);
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const f32x4 Z = sPO[n][w][lane];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    rz.store(row0 + r, p0 + 16 * n + c, Z[r]);
                    rv.store(row0 + r, p0 + 16 * n + c, Z[r] * beta[r]);
                }
            }
            if (ch) leave();
        }
        return;
    }

    auto state_off = [&](int i, int n, int r) {
        const int row = NT * 16 * w + 16 * i + 4 * q + r, col = p0 + 16 * n + c;
        return row < N && col < P ? (row * P + col) * 4 : (int)0x80000000;
    };
    f32x4 E[NT][NC];
    auto put_state = [&](helix_rsrc to) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) __builtin_amdgcn_raw_buffer_store_b32(as_u32(E[i][n][r]), to, state_off(i, n, r), 0, 0);
    };
    auto put_e = [&] {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int n = 0; n < NC; ++n)
                dr_put4<3, NK, COLS>(sE, 16 * n + c, NT * 16 * w + 16 * i + 4 * q, E[i][n][0], E[i][n][1], E[i][n][2], E[i][n][3]);
    };
    bf16x8 tf[2][3];
    auto load_t = [&](int ch) {
        const char* tt = p.tt + (base + max(ch, 0)) * (6 * 3 * HELIX_DR_FRAG) + 16 * lane;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (ks == 0 && w > 1) continue;
#pragma unroll
            for (int k = 0; k < 3; ++k) tf[ks][k] = *reinterpret_cast<const bf16x8*>(tt + (dr_up(w, ks) * 3 + k) * HELIX_DR_FRAG);
        }
    };
    {
        const helix_rsrc r0 = make_rsrc_u(p.d_s + (long long)sh * N * P, p.d_s ? state_bytes : 0u);   // none: reads 0
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) E[i][n][r] = buf_f32(r0, state_off(i, n, r), 0);
    }
    if (last >= 0) {
        load_t(last);
        put_e();
        dr_barrier();
    }
    for (int ch = last; ch >= 0; --ch) {
        dr_barrier();   // K, E and what does not depend on E are there
        put_state(make_rsrc_u(p.keep_e + (base + ch) * N * P, state_bytes));
        const float* const dec = sDec[ch & 1];
        typename DrAccOf<NC>::type ke[NC];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int col = 32 * s + 8 * q;
            bf16x8 a[NPL], b[3];
            dr_get8<NPL, NK, DR_C>(sK, 16 * w + c, col, a);
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                dr_get8<3, NK, COLS>(sE, 16 * n + c, col, b);
                dr_mfma<NPL, 3>(a, b, ke[n]);
            }
        }
        bf16x8 kt[2][NT][NPL];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < NT; ++i) dr_get8_t<NPL, NK, DR_C>(sK, 32 * ks + 8 * q, NT * 16 * w + 16 * i, c, kt[ks][i]);
        const f32x4 left = *reinterpret_cast<const f32x4*>(dec + 64 + row0);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
#pragma unroll
            for (int i = 0; i < NT; ++i) E[i][n] = dec[63] * E[i][n] + sQW[n][i][w][lane];
            const f32x4 dd = ke[n].sum() * left + sPO[n][w][lane];
            dr_put4<3, DR_C, COLS>(sR, 16 * n + c, row0, dd[0], dd[1], dd[2], dd[3]);
        }
        dr_barrier();   // dD is there; K has been read
        typename DrAccOf<NC>::type zs[NC];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (ks == 0 && w > 1) continue;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                bf16x8 b[3];
                dr_get8<3, DR_C, COLS>(sR, 16 * n + c, 32 * ks + 8 * q, b);
                dr_mfma<3, 3>(tf[ks], b, zs[n]);
            }
        }
        const f32x4 factor = -(*reinterpret_cast<const f32x4*>(dec + 128 + row0) * *reinterpret_cast<const f32x4*>(dec + row0));
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const f32x4 Z = zs[n].sum(), u = Z * factor;
            dr_put4<3, DR_C, COLS>(sU, 16 * n + c, row0, u[0], u[1], u[2], u[3]);
            sPO[n][w][lane] = Z;
        }
        load_t(ch - 1);
        dr_barrier();   // dV is there
        typename DrAccOf<NC>::type up[NT][NC];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                bf16x8 b[3];
                dr_get8<3, DR_C, COLS>(sU, 16 * n + c, 32 * ks + 8 * q, b);
#pragma unroll
                for (int i = 0; i < NT; ++i) dr_mfma<NPL, 3>(kt[ks][i], b, up[i][n]);
            }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int n = 0; n < NC; ++n) E[i][n] += up[i][n].sum();
        put_e();
    }
    put_state(make_rsrc_u(p.ds0 + (long long)sh * N * P, state_bytes));
}

// The other gradients, a chunk of a head of queries and keys a workgroup, its value heads one
// after another. With D, Z, E and the state S before the chunk:
//     U = dO S',  B = Z S',  L = D E';   dP = dO D' for j <= i,  dA = -Z D' below the diagonal
//     M_P = scale dP . E_ij,  M_A = beta_i dA . E_ij       (summed over the heads that share)
//     dQ = scale e^G U + M_P K
//     dK = e^(G_63 - G) L - e^G beta B + M_P' Q + (M_A + M_A') K
//     dbeta = Z . V - e^G (K . B) + sum_j dA . E_ij . K K'
// and g_t has the sum over i >= t of what G_i has: M_P . Q K' + M_A . K K' by rows less by
// columns, scale e^G (Q . U) - e^G beta (K . B) - e^(G_63 - G) (K . L), and for the last one the
// sum of e^(G_63 - G) (K . L) and e^(G_63) (S . E); in fp64, as neighbours nearly cancel.
// Two kernels, as the registers do not hold both: the triangles first (helix_delta_pairs_*, a
// wave a block of 16 x 16), which read dO, Z, D and V, then the products with the states
// (helix_delta_grad_*), which read dO, Z and D again, S and E. Memory binds both, behind the LDS
// that dO, Z and D pass: 8192 chunks of heads of 128 x 64, bf16, 440 MB in 130 us and 970 MB
// in 300, 3.3 TB/s.
template <typename T, int NK, bool ODD>
__device__ void delta_pairs(const HelixDeltaParams& p) {
    constexpr int NPL = dr_planes<T>, TH = 640;
    constexpr int kKQ = 2 * NPL * DR_C * NK, kOZD = (NPL + 6) * DR_C * DR_C;
    __shared__ __attribute__((aligned(16))) __bf16 sBig[kKQ > kOZD ? kKQ : kOZD];
    __shared__ double sG[DR_C];
    __shared__ __attribute__((aligned(16))) float sB[DR_C];
    __shared__ float sRow[4][DR_C], sCol[4][DR_C], sBeta[4][DR_C], sZV[DR_C];
    __bf16* const sK = sBig;
    __bf16* const sQ = sBig + NPL * DR_C * NK;
    __bf16* const sO = sBig;
    __bf16* const sZ = sBig + NPL * DR_C * DR_C;
    __bf16* const sD = sZ + 3 * DR_C * DR_C;
    const int tid = threadIdx.x, lane = lane_id(), w = wave_uniform(), c = lane & 15, q = lane >> 4;
    const unsigned id = blockIdx.x;
    const int ch = (int)(id % (unsigned)p.n_chunk);
    const unsigned sk = id / (unsigned)p.n_chunk;
    const int seq = (int)(sk / (unsigned)p.n_qk), hk = (int)(sk % (unsigned)p.n_qk);
    const long long t0 = (long long)(p.chunk0 + ch) * DR_C;
    const int len = (int)min((long long)DR_C, p.n_tok - t0), P = p.n_val, N = p.n_key;
    const int tb = (w >= 1) + (w >= 3) + (w >= 6), jb = w - tb * (tb + 1) / 2;   // the wave's block
    {
        const Rows<T, ODD> rk(p.k, seq * p.seq_k + hk * p.head_k + t0 * p.tok_k, p.tok_k, len, N);
        const Rows<T, ODD> rq(p.q, seq * p.seq_q + hk * p.head_q + t0 * p.tok_q, p.tok_q, len, N);
        for (int i = tid; i < DR_C * (NK / 8); i += TH) {
            const int row = i / (NK / 8), col = 8 * (i % (NK / 8));
            bf16x8 k[NPL], qq[NPL];
            dr_operand<T>(rk.load8(row, col), N - col, k);
            dr_operand<T>(rq.load8(row, col), N - col, qq);
            dr_put8<NPL, NK, DR_C>(sK, row, col, k);
            dr_put8<NPL, NK, DR_C>(sQ, row, col, qq);
        }
    }
    // A pass over 64 columns of a head's values, loaded while the one before is at work: a row's eight by the first 512 threads.
    Raw8<T> no, nv;
    Raw8<float> nz, nd;
    float ng, nb;
    auto load = [&](int hs, int pb) {
        if (hs >= p.share) return;
        const int tid = vgpr_fresh(threadIdx.x), srow = tid / 8, scol = 8 * (tid % 8), lane = tid & 63;
        const int h = hk * p.share + hs;
        const long long at = ((long long)seq * p.n_head + h) * p.n_chunk + ch;
        const Rows<T, ODD> ro(p.d_o, seq * p.seq_o + h * p.head_o + t0 * p.tok_o, p.tok_o, len, P);
        const Rows<T, ODD> rv(p.v, seq * p.seq_v + h * p.head_v + t0 * p.tok_v, p.tok_v, len, P);
        const Rows<float> rz(p.keep_z, at * DR_C * P, P, DR_C, P), rd(p.keep_d, at * DR_C * P, P, DR_C, P);
        if (tid < 512) {
            no = ro.load8(srow, pb + scol);
            nz = rz.load8(srow, pb + scol);
            nd = rd.load8(srow, pb + scol);
            nv = rv.load8(srow, pb + scol);
        }
        nb = p.decay[at * (HELIX_DR_DECAY / 4) + 128 + lane];
        ng = lane < len ? p.g[seq * p.seq_g + (t0 + lane) * p.tok_g + h] : 0.0f;
    };
    load(0, 0);
    __syncthreads();
    f32x4 kk, qk, mp = zero4(), ma = zero4();
    {
        DrAcc x, y;
#pragma unroll
        for (int s = 0; s < NK / 32; ++s) {
            const int col = 32 * s + 8 * q;
            bf16x8 a[NPL], b[NPL];
            dr_get8<NPL, NK, DR_C>(sK, 16 * jb + c, col, b);
            dr_get8<NPL, NK, DR_C>(sK, 16 * tb + c, col, a);
            dr_mfma<NPL, NPL>(a, b, x);
            dr_get8<NPL, NK, DR_C>(sQ, 16 * tb + c, col, a);
            dr_mfma<NPL, NPL>(a, b, y);
        }
        kk = dr_sum<NPL>(x);
        qk = dr_sum<NPL>(y);
    }
    for (int hs = 0; hs < p.share; ++hs) {
        const long long at = ((long long)seq * p.n_head + hk * p.share + hs) * p.n_chunk + ch;
        const double G = dr_log_decay(ng) * 1.4426950408889634074;
        const float bl = nb;
        f32x4 dP = zero4(), dA = zero4();
        float zv = 0.0f;
        for (int pb = 0; pb < P; pb += 64) {
            // (Addresses formed from these are formed here, not kept over the loop.)
            const int tid = vgpr_fresh(threadIdx.x), srow = tid / 8, scol = 8 * (tid % 8), c = tid & 15, q = (tid & 63) >> 4;
            __syncthreads();   // what these overwrite has been read
            if (tid < 512) {
                const int n = P - pb - scol;
                bf16x8 o[NPL], z[3], d[3];
                dr_operand<T>(no, n, o);
                dr_operand<float, true>(nz, n, z);
                dr_operand<float, true>(nd, n, d);
#pragma unroll
                for (int e = 0; e < 8; ++e) zv += e < n ? at8(nz, e) * at8(nv, e) : 0.0f;
                dr_put8<NPL, DR_C, DR_C>(sO, srow, scol, o);
                dr_put8<3, DR_C, DR_C>(sZ, srow, scol, z);
                dr_put8<3, DR_C, DR_C>(sD, srow, scol, d);
            }
            load(pb + 64 < P ? hs : hs + 1, pb + 64 < P ? pb + 64 : 0);
            __syncthreads();
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const int col = 32 * ks + 8 * q;
                bf16x8 ao[NPL], az[3], bd[3];
                dr_get8<3, DR_C, DR_C>(sD, 16 * jb + c, col, bd);
                dr_get8<NPL, DR_C, DR_C>(sO, 16 * tb + c, col, ao);
                dP = dr_mfma<NPL, 3>(ao, bd, dP);
                dr_get8<3, DR_C, DR_C>(sZ, 16 * tb + c, col, az);
                dA = dr_mfma<3, 3>(az, bd, dA);
            }
        }
        const int tid = vgpr_fresh(threadIdx.x), lane = tid & 63, c = tid & 15, q = lane >> 4;
        if (w == 0) {
            sG[lane] = G;
            sB[lane] = bl;
        }
        if (tid < 512) {
            zv = add_dpp<0xb1>(zv);   // eight lanes a row
            zv = add_dpp<0x4e>(zv);
            zv = add_dpp<0x141>(zv);
            if ((tid & 7) == 0) sZV[tid / 8] = zv;
        }
        __syncthreads();
        {
            const int j = 16 * jb + c;
            const double Gj = sG[j];
            const f32x4 beta = *reinterpret_cast<const f32x4*>(&sB[16 * tb + 4 * q]);
            float pair[4], bs[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * tb + 4 * q + r;
                const float e = __builtin_amdgcn_exp2f((float)(sG[i] - Gj));
                const bool in = tb > jb || j <= i, below = tb > jb || j < i;
                const float m = in ? p.scale * (e * dP[r]) : 0.0f, a = below ? -(e * dA[r]) : 0.0f;
                mp[r] += m;
                ma[r] += beta[r] * a;
                bs[r] = below ? a * kk[r] : 0.0f;
                pair[r] = in ? m * qk[r] + beta[r] * bs[r] : 0.0f;
            }
            const float row = row16_sum4(pair[0], pair[1], pair[2], pair[3], lane), b = row16_sum4(bs[0], bs[1], bs[2], bs[3], lane);
            float col = (pair[0] + pair[1]) + (pair[2] + pair[3]);
            col += __shfl_xor(col, 16, 64);
            col += __shfl_xor(col, 32, 64);
            if (c < 4) {
                sRow[jb][16 * tb + 4 * q + c] = row;
                sBeta[jb][16 * tb + 4 * q + c] = b;
            }
            if (q == 0) sCol[tb][j] = col;
        }
        __syncthreads();
        if (w == 9) {
            // Lane = token: what G and beta have of the triangles, and Z . V.
            const int tile = lane >> 4;
            double own = 0.0;
            float db = sZV[lane];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if (x <= tile) {
                    own += sRow[x][lane];
                    db += sBeta[x][lane];
                }
                if (x >= tile) own -= sCol[x][lane];
            }
            p.pair_g[at * DR_C + lane] = own;
            p.pair_b[at * DR_C + lane] = db;
        }
    }
    float* to = p.tri + (long long)id * (2 * 10 * 256) + 4 * lane;
    *reinterpret_cast<f32x4*>(to + 256 * w) = mp;
    *reinterpret_cast<f32x4*>(to + 256 * (10 + w)) = ma;
}

// A wave has 16 of the keys' columns (U, B, L, dQ, dK for its tokens; its rows of S and E straight
// from memory), of all tokens or, with 64 keys, half of them. dO, Z and D are in LDS, by parts,
// 64 columns at a time; K, Q and the triangles at the end.
template <typename T, int NK, bool ODD>
__device__ void delta_grad(const HelixDeltaParams& p) {
    constexpr int NPL = dr_planes<T>, W = NK / 16, TH = 512;
    constexpr int RG = 8 / W, RT = 4 / RG;   // groups of waves along the tokens, and row tiles of a wave
    constexpr int kKQ = 2 * NPL * DR_C * NK, kM = 3 * DR_C * DR_C, kOZD = (NPL + 6) * DR_C * DR_C;
    __shared__ __attribute__((aligned(16))) __bf16 sBig[kKQ + kM > kOZD ? kKQ + kM : kOZD];
    __shared__ __attribute__((aligned(16))) float sDec[HELIX_DR_DECAY / 4];
    __shared__ float sDot[3][W][DR_C], sSE[W];
    __bf16* const sK = sBig;
    __bf16* const sQ = sBig + NPL * DR_C * NK;
    __bf16* const sM = sBig + kKQ;
    __bf16* const sO = sBig;
    __bf16* const sZ = sBig + NPL * DR_C * DR_C;
    __bf16* const sD = sZ + 3 * DR_C * DR_C;
    const int tid = threadIdx.x, lane = lane_id(), w = wave_uniform(), c = lane & 15, q = lane >> 4;
    const unsigned id = blockIdx.x;
    const int ch = (int)(id % (unsigned)p.n_chunk);
    const unsigned sk = id / (unsigned)p.n_chunk;
    const int seq = (int)(sk / (unsigned)p.n_qk), hk = (int)(sk % (unsigned)p.n_qk);
    const long long t0 = (long long)(p.chunk0 + ch) * DR_C;
    const int len = (int)min((long long)DR_C, p.n_tok - t0), P = p.n_val, N = p.n_key;
    const int cw = RG == 1 ? w : w % W, n0 = 16 * cw, i0 = RG == 1 ? 0 : w / W * RT;   // the wave's columns, and first row tile
    const Rows<T, ODD> rk(p.k, seq * p.seq_k + hk * p.head_k + t0 * p.tok_k, p.tok_k, len, N);
    const Rows<T, ODD> rq(p.q, seq * p.seq_q + hk * p.head_q + t0 * p.tok_q, p.tok_q, len, N);
    f32x4 dq[RT], dk[RT];
    typename Raw4<T>::type kv[RT], qv[RT];   // k and q at (16 (i0 + i) + 4 q + r, n0 + c), as they are stored
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        dq[i] = dk[i] = zero4();
        unsigned k4[4], q4[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            k4[r] = rk.raw(16 * (i0 + i) + 4 * q + r, n0 + c);
            q4[r] = rq.raw(16 * (i0 + i) + 4 * q + r, n0 + c);
        }
        kv[i] = pack4<T>(k4);
        qv[i] = pack4<T>(q4);
    }
    // A pass over 64 columns of a head's values, loaded while the one before is at work: the thread's row of dO, Z and D, and
    // the wave's rows of S and E.
    struct Ahead {
        Raw8<T> o;
        Raw8<float> z, d, s[2], e[2];
        f32x4 dec;
    } next;
    auto load = [&](int hs, int pb) {
        if (hs >= p.share) return;
        const int tid = vgpr_fresh(threadIdx.x), c = tid & 15, q = (tid & 63) >> 4, h = hk * p.share + hs;
        const long long at = ((long long)seq * p.n_head + h) * p.n_chunk + ch;
        const Rows<T, ODD> ro(p.d_o, seq * p.seq_o + h * p.head_o + t0 * p.tok_o, p.tok_o, len, P);
        const Rows<float> rz(p.keep_z, at * DR_C * P, P, DR_C, P), rd(p.keep_d, at * DR_C * P, P, DR_C, P);
        const Rows<float> rs(p.keep_s, at * N * P, P, N, P), re(p.keep_e, at * N * P, P, N, P);
        const int row = tid / 8, col = pb + 8 * (tid % 8);
        next.o = ro.load8(row, col);
        next.z = rz.load8(row, col);
        next.d = rd.load8(row, col);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            next.s[ks] = rs.load8(n0 + c, pb + 32 * ks + 8 * q);
            next.e[ks] = re.load8(n0 + c, pb + 32 * ks + 8 * q);
        }
        if (tid < HELIX_DR_DECAY / 16) next.dec = *reinterpret_cast<const f32x4*>(p.decay + at * (HELIX_DR_DECAY / 4) + 4 * tid);
    };
    load(0, 0);
    for (int hs = 0; hs < p.share; ++hs) {
        const long long at = (((long long)seq * p.n_head + hk * p.share + hs) * p.n_chunk + ch) * DR_C + lane;
        double own = 0.0;
        float db = 0.0f;
        if (w == 0) {
            own = p.pair_g[at];
            db = p.pair_b[at];
        }
        float se = 0.0f, dots[3][RT];   // (of row 16 (i0 + i) + 4 q + c % 4)
#pragma unroll
        for (int i = 0; i < RT; ++i) dots[0][i] = dots[1][i] = dots[2][i] = 0.0f;
        for (int pb = 0; pb < P; pb += 64) {
            // (Addresses formed from these are formed here, not kept over the loop.)
            const int fresh = vgpr_fresh(tid), lane = fresh & 63, c = lane & 15, q = lane >> 4;
            __syncthreads();   // what these overwrite has been read
            {
                const int row = fresh / 8, col = 8 * (fresh % 8), n = P - pb - col;
                bf16x8 o[NPL], z[3], d[3];
                dr_operand<T>(next.o, n, o);
                dr_operand<float, true>(next.z, n, z);
                dr_operand<float, true>(next.d, n, d);
                dr_put8<NPL, DR_C, DR_C>(sO, row, col, o);
                dr_put8<3, DR_C, DR_C>(sZ, row, col, z);
                dr_put8<3, DR_C, DR_C>(sD, row, col, d);
            }
            if (tid < HELIX_DR_DECAY / 16) *reinterpret_cast<f32x4*>(&sDec[4 * tid]) = next.dec;
            bf16x8 bs[2][3], be[2][3];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const int n = P - pb - 32 * ks - 8 * q;
                dr_operand<float, true>(next.s[ks], n, bs[ks]);
                dr_operand<float, true>(next.e[ks], n, be[ks]);
#pragma unroll
                for (int e = 0; e < 8; ++e) se += e < n ? at8(next.s[ks], e) * at8(next.e[ks], e) : 0.0f;
            }
            load(pb + 64 < P ? hs : hs + 1, pb + 64 < P ? pb + 64 : 0);
            __syncthreads();
            // Row tile by row tile: each product goes into the gradients (and its dot with q or k) at once.
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int tile = 16 * (i0 + i), row = tile + 4 * q;
                DrAcc U, B, L;
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const int col = 32 * ks + 8 * q;
                    bf16x8 ao[NPL], az[3], ad[3];
                    dr_get8<NPL, DR_C, DR_C>(sO, tile + c, col, ao);
                    dr_mfma<NPL, 3>(ao, bs[ks], U);
                    dr_get8<3, DR_C, DR_C>(sZ, tile + c, col, az);
                    dr_mfma<3, 3>(az, bs[ks], B);
                    dr_get8<3, DR_C, DR_C>(sD, tile + c, col, ad);
                    dr_mfma<3, 3>(ad, be[ks], L);
                }
                const f32x4 start = *reinterpret_cast<const f32x4*>(&sDec[row]), left = *reinterpret_cast<const f32x4*>(&sDec[64 + row]),
                            beta = *reinterpret_cast<const f32x4*>(&sDec[128 + row]);
                const f32x4 u = U.sum(), b = B.sum(), l = L.sum();
                dq[i] += p.scale * start * u;
                dk[i] += left * l - start * beta * b;
                float x[4];
                widen4<T>(fresh4<T>(qv[i]), x);
                dots[0][i] += row16_sum4(x[0] * u[0], x[1] * u[1], x[2] * u[2], x[3] * u[3], lane);
                widen4<T>(fresh4<T>(kv[i]), x);
                dots[1][i] += row16_sum4(x[0] * b[0], x[1] * b[1], x[2] * b[2], x[3] * b[3], lane);
                dots[2][i] += row16_sum4(x[0] * l[0], x[1] * l[1], x[2] * l[2], x[3] * l[3], lane);
                __builtin_amdgcn_sched_barrier(0);   // (the next tile's reads would not fit in the registers)
            }
        }
        se = wave_sum(se);
        if (lane == 0 && i0 == 0) sSE[cw] = se;
        if (c < 4) {
#pragma unroll
            for (int i = 0; i < RT; ++i) {
#pragma unroll
                for (int j = 0; j < 3; ++j) sDot[j][cw][16 * (i0 + i) + 4 * q + c] = dots[j][i];
            }
        }
        __syncthreads();
        if (w == 0) {
            // Lane = token.
            const int h = hk * p.share + hs;
            float dot[3];
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                dot[j] = 0.0f;
#pragma unroll
                for (int x = 0; x < W; ++x) dot[j] += sDot[j][x][lane];
            }
            float sse = 0.0f;
#pragma unroll
            for (int x = 0; x < W; ++x) sse += sSE[x];
            const float start = sDec[lane], left = sDec[64 + lane], beta = sDec[128 + lane];
            const double tail = (double)left * dot[2];
            own += (double)(p.scale * start) * dot[0] - (double)(start * beta) * dot[1] - tail;
            const double tails = __shfl(wave_incl_sum(tail), 63, 64);
            if (lane == 63) own += tails + (double)sDec[63] * sse;
            const double incl = wave_incl_sum(own);
            const double dg = __shfl(incl, 63, 64) - incl + own;
            if (lane < len) {
                const long long to = ((long long)seq * p.n_tok + t0 + lane) * p.row_head + h;
                p.dg[to] = (float)dg;
                p.dbeta[to] = db - start * dot[1];
            }
        }
    }
    // The triangles' products, once for all heads.
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DR_C * (NK / 8) / TH; ++i) {
        const int row = (tid + TH * i) / (NK / 8), col = 8 * ((tid + TH * i) % (NK / 8));
        const Raw8<T> kr = rk.load8(row, col), qr = rq.load8(row, col);
        bf16x8 k[NPL], qq[NPL];
        dr_operand<T>(kr, N - col, k);
        dr_operand<T>(qr, N - col, qq);
        dr_put8<NPL, NK, DR_C>(sK, row, col, k);
        dr_put8<NPL, NK, DR_C>(sQ, row, col, qq);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {   // M_P, then M_A
        if (m) __syncthreads();   // M_P has been read
        for (int x = w; x < 10; x += 8) {
            // Stored by columns: M[j][i]; 0 above the diagonal.
            const int tb = (x >= 1) + (x >= 3) + (x >= 6), jb = x - tb * (tb + 1) / 2;
            const f32x4 v = *reinterpret_cast<const f32x4*>(p.tri + (long long)id * (2 * 10 * 256) + 256 * (10 * m + x) + 4 * lane);
            dr_put4<3, DR_C, DR_C>(sM, 16 * jb + c, 16 * tb + 4 * q, v[0], v[1], v[2], v[3]);
            if (tb != jb) dr_put4<3, DR_C, DR_C>(sM, 16 * tb + c, 16 * jb + 4 * q, 0.0f, 0.0f, 0.0f, 0.0f);
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            bf16x8 bk[NPL], bq[NPL];
            dr_get8_t<NPL, NK, DR_C>(sK, 32 * ks + 8 * q, n0, c, bk);
            if (m == 0) dr_get8_t<NPL, NK, DR_C>(sQ, 32 * ks + 8 * q, n0, c, bq);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                bf16x8 a[3];
                const int tile = i0 + i;
                // M[i][j] over j: columns of what is stored; M'[j][i] over i: its rows.
                if (2 * ks <= tile) {
                    dr_get8_t<3, DR_C, DR_C>(sM, 32 * ks + 8 * q, 16 * tile, c, a);
                    if (m == 0) dq[i] = dr_mfma<3, NPL>(a, bk, dq[i]);
                    else dk[i] = dr_mfma<3, NPL>(a, bk, dk[i]);
                }
                if (2 * ks + 1 >= tile) {
                    dr_get8<3, DR_C, DR_C>(sM, 16 * tile + c, 32 * ks + 8 * q, a);
                    if (m == 0) dk[i] = dr_mfma<3, NPL>(a, bq, dk[i]);
                    else dk[i] = dr_mfma<3, NPL>(a, bk, dk[i]);
                }
            }
        }
    }
    const long long to = (((long long)seq * p.n_tok + t0) * p.row_qk + hk) * N;
    const Rows<T> oq(p.dq, to, (long long)p.row_qk * N, len, N), ok(p.dk, to, (long long)p.row_qk * N, len, N);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            oq.store(16 * (i0 + i) + 4 * q + r, n0 + c, dq[i][r]);
            ok.store(16 * (i0 + i) + 4 * q + r, n0 + c, dk[i][r]);
        }
}

}  // namespace

#define DR_STEPS(TAG, T, NK)                                                                                                             \
    extern "C" __global__ __launch_bounds__(256) void helix_delta_steps_##TAG##_##NK(HelixDeltaParams p) { delta_steps<T, NK / 16>(p); }
// _s: rows of an odd width. _c16, _c32: columns of a workgroup. Waves a SIMD where LDS has room for two workgroups a CU.
#define DR_KERNELS(TAG, T, NK, SUF, ODD)                                                                                                                    \
    extern "C" __global__ __launch_bounds__(256) void helix_delta_prep_##TAG##_##NK##SUF(HelixDeltaParams p) { prep_kernel<T, NK, ODD, false>(p); }          \
    extern "C" __global__ __launch_bounds__(256) void helix_delta_prep_bwd_##TAG##_##NK##SUF(HelixDeltaParams p) { prep_kernel<T, NK, ODD, true>(p); }       \
    extern "C" __global__ __launch_bounds__(640, sizeof(T) == 4 && NK == 128 ? 3 : 5) void helix_delta_pairs_##TAG##_##NK##SUF(HelixDeltaParams p) { delta_pairs<T, NK, ODD>(p); }               \
    extern "C" __global__ __launch_bounds__(512) void helix_delta_grad_##TAG##_##NK##SUF(HelixDeltaParams p) { delta_grad<T, NK, ODD>(p); }                 \
    extern "C" __global__ __launch_bounds__(512, sizeof(T) == 4 ? 2 : 4) void helix_delta_walk_##TAG##_##NK##SUF##_c16(HelixDeltaParams p) { delta_walk_ahead<T, NK, ODD>(p); } \
    extern "C" __global__ __launch_bounds__(512) void helix_delta_keep_##TAG##_##NK##SUF##_c16(HelixDeltaParams p) { walk_kernel<T, NK, ODD, true, 1>(p); }  \
    extern "C" __global__ __launch_bounds__(512) void helix_delta_back_##TAG##_##NK##SUF##_c16(HelixDeltaParams p) { delta_back<T, NK, ODD, 1>(p); }        \
    extern "C" __global__ __launch_bounds__(512) void helix_delta_walk_##TAG##_##NK##SUF##_c32(HelixDeltaParams p) { walk_kernel<T, NK, ODD, false, 2>(p); } \
    extern "C" __global__ __launch_bounds__(512, sizeof(WalkLds<T, NK, true, 2>) <= 81920 ? 4 : 2) void helix_delta_keep_##TAG##_##NK##SUF##_c32(HelixDeltaParams p) { walk_kernel<T, NK, ODD, true, 2>(p); }
// (fp32 of 128 keys and 32 columns would not fit in LDS.)
#define DR_BACK(TAG, T, NK, SUF, ODD)                                                                                                                \
    extern "C" __global__ __launch_bounds__(512) void helix_delta_back_##TAG##_##NK##SUF##_c32(HelixDeltaParams p) { delta_back<T, NK, ODD, 2>(p); }
DR_STEPS(f32, float, 64)
DR_KERNELS(f32, float, 64, , false)
DR_BACK(f32, float, 64, , false)
DR_STEPS(f32, float, 128)
DR_KERNELS(f32, float, 128, , false)
DR_STEPS(f16, _Float16, 64)
DR_KERNELS(f16, _Float16, 64, , false)
DR_BACK(f16, _Float16, 64, , false)
DR_KERNELS(f16, _Float16, 64, _s, true)
DR_BACK(f16, _Float16, 64, _s, true)
DR_STEPS(f16, _Float16, 128)
DR_KERNELS(f16, _Float16, 128, , false)
DR_BACK(f16, _Float16, 128, , false)
DR_KERNELS(f16, _Float16, 128, _s, true)
DR_BACK(f16, _Float16, 128, _s, true)
DR_STEPS(bf16, __bf16, 64)
DR_KERNELS(bf16, __bf16, 64, , false)
DR_BACK(bf16, __bf16, 64, , false)
DR_KERNELS(bf16, __bf16, 64, _s, true)
DR_BACK(bf16, __bf16, 64, _s, true)
DR_STEPS(bf16, __bf16, 128)
DR_KERNELS(bf16, __bf16, 128, , false)
DR_BACK(bf16, __bf16, 128, , false)
DR_KERNELS(bf16, __bf16, 128, _s, true)
DR_BACK(bf16, __bf16, 128, _s, true)
