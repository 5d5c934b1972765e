// delta_rule.hip -- the gated delta rule (helix_layer.h): per value head, with the state S of
// N keys x P values in fp32,
//     S_t = e^(g_t) S_(t-1) + beta_t k_t (v_t - e^(g_t) S_(t-1)' k_t)',   o_t = scale S_t' q_t
//
// Few tokens go one by one (helix_delta_steps_*). More go in chunks of 64: with G the sums of
// g from the chunk's start, E_ij = exp(G_i - G_j) for j <= i, A_ij = beta_i E_ij (k_i . k_j)
// below the diagonal and X = (1 + A)^-1 diag(beta),
//     D = X (V - e^G K S),   O = scale (e^G Q S + (E . Q K') D),   S' = e^(G_63) S + (e^(G_63 - G) K)' D
// X and P = scale E . Q K' need no state: helix_delta_prep_* forms them for all chunks at once.
// helix_delta_walk_* then goes through the chunks of a sequence, a workgroup for 16 columns of
// a head's state, whose columns do not meet.
#include "delta_common.h"

namespace {

// ---- token by token -----------------------------------------------------------------------
//
// A workgroup has 64 columns of a state in registers: lane 16 kg + cl of wave w columns
// 4 cl .. + 3 of the rows 16 i + 4 w + kg. k'S and q'S are summed over a token's old state
// together (q'S' = e^g q'S + (q . k) d), so that a token meets one barrier. Memory binds a
// batch of single tokens (the state is read and written once), latency few sequences.
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
// on fp32 matrix instructions, T_jw staying in the registers it was formed in. BWD: X' and P' as well, without P.
template <typename T, int NK, bool BWD>
__device__ void delta_prep(const HelixDeltaParams& p) {
    constexpr int NPL = dr_planes<T>, NO = dr_out_planes<T>, KP = NK + 8;
    __shared__ __bf16 sK[NPL][DR_C][KP];
    __shared__ float sA[DR_C][DR_LD], sX[DR_C][DR_LD], sP[DR_C][DR_LD];
    __shared__ float sD[4][16][20];
    __shared__ double sG[DR_C];
    __shared__ float sB[DR_C];
    const int tid = threadIdx.x, lane = lane_id(), w = wave_uniform(), c = lane & 15, q = lane >> 4;
    const unsigned id = blockIdx.x;
    const int ch = (int)(id % (unsigned)p.n_chunk);
    const unsigned sh = id / (unsigned)p.n_chunk;
    const int seq = (int)(sh / (unsigned)p.n_head), h = (int)(sh % (unsigned)p.n_head), hk = h / p.share;
    const long long t0 = (long long)(p.chunk0 + ch) * DR_C;
    const int len = (int)min((long long)DR_C, p.n_tok - t0);
    const Rows<T> rk(p.k, seq * p.seq_k + hk * p.head_k + t0 * p.tok_k, p.tok_k, len, p.n_key);
    const Rows<T> rq(p.q, seq * p.seq_q + hk * p.head_q + t0 * p.tok_q, p.tok_q, len, p.n_key);
    // K's parts into LDS; the wave's rows of Q in registers.
    constexpr int PER = DR_C * (NK / 8) / 256;
    Raw8<T> kr[PER], qr[NK / 32];
#pragma unroll
    for (int i = 0; i < PER; ++i) kr[i] = rk.load8((tid + 256 * i) / (NK / 8), 8 * ((tid + 256 * i) % (NK / 8)));
#pragma unroll
    for (int s = 0; s < NK / 32; ++s) qr[s] = rq.load8(16 * w + c, 32 * s + 8 * q);
    const float gl = lane < len ? p.g[seq * p.seq_g + (t0 + lane) * p.tok_g + h] : 0.0f;
    const float bl = lane < len ? p.beta[seq * p.seq_b + (t0 + lane) * p.tok_b + h] : 0.0f;
    const double G = dr_log_decay(gl);
    const double end = __shfl(G, 63, 64);
    if (w == 0) {
        sG[lane] = G;
        sB[lane] = bl;
        float* dec = p.decay + id * (HELIX_DR_DECAY / 4ll);
        dec[lane] = exp_diff(G, 0.0);
        dec[64 + lane] = exp_diff(end, G);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int row = (tid + 256 * i) / (NK / 8), col = 8 * ((tid + 256 * i) % (NK / 8));
        bf16x8 o[NPL];
        dr_operand<T>(kr[i], p.n_key - col, o);
#pragma unroll
        for (int k = 0; k < NPL; ++k) *reinterpret_cast<bf16x8*>(&sK[k][row][col]) = o[k];
    }
    __syncthreads();
    f32x4 kk[4], qk[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) kk[j] = qk[j] = zero4();
#pragma unroll
    for (int s = 0; s < NK / 32; ++s) {
        const int col = 32 * s + 8 * q;
        bf16x8 ak[NPL], aq[NPL];
        dr_get8<NPL>(&sK[0][16 * w + c][col], DR_C * KP, ak);
        dr_operand<T>(qr[s], p.n_key - col, aq);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > w) continue;
            bf16x8 b[NPL];
            dr_get8<NPL>(&sK[0][16 * j + c][col], DR_C * KP, b);
            kk[j] = dr_mfma<NPL, NPL>(ak, b, kk[j]);
            qk[j] = dr_mfma<NPL, NPL>(aq, b, qk[j]);
        }
    }
    // (Blocks above the diagonal that fragments reach are 0.)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int jj = 16 * j + c;
        const double Gj = sG[jj];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * w + 4 * q + r;
            const float e = j <= w && jj <= i ? exp_diff(sG[i], Gj) : 0.0f;
            sA[i][jj] = jj < i && j <= w ? sB[i] * (e * kk[j][r]) : 0.0f;
            sP[i][jj] = jj <= i && j <= w ? p.scale * (e * qk[j][r]) : 0.0f;
            if (j > w) sX[i][jj] = 0.0f;
        }
    }
    __syncthreads();
    // Diagonal block w: lane c its column c (the four groups alike).
    {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = i == c ? 1.0f : 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (j < i) s = fmaf(-sA[16 * w + i][16 * w + j], x[j], s);
            x[i] = s;
        }
        if (q == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sD[w][i][c] = x[i];
        }
    }
    __syncthreads();
    {
        f32x4 t[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) t[0][r] = sD[w][4 * q + r][c];
        const float b = sB[16 * w + c];
        auto put = [&](int i, const f32x4& v) {
#pragma unroll
            for (int r = 0; r < 4; ++r) sX[16 * i + 4 * q + r][16 * w + c] = v[r] * b;
        };
        put(w, t[0]);
#pragma unroll
        for (int step = 1; step < 4; ++step) {
            const int i = w + step;
            if (i > 3) break;
            f32x4 m = zero4();
#pragma unroll
            for (int j = 0; j < step; ++j)
                m = dr_mfma_f32(*reinterpret_cast<const f32x4*>(&sA[16 * i + c][16 * (w + j) + 4 * q]), t[j], m);
            f32x4 a = *reinterpret_cast<const f32x4*>(&sD[i][c][4 * q]);
            a = -a;
            t[step] = dr_mfma_f32(a, m, zero4());
            put(i, t[step]);
        }
    }
    __syncthreads();
    // Fragments: row 16 w + c, columns 32 ks + 8 q ..
    auto emit = [&](char* to, int frag, const float (&v)[8], auto parts) {
        constexpr int N = decltype(parts)::value;
        bf16x8 o[N];
        dr_split8<N>(v, o);
#pragma unroll
        for (int k = 0; k < N; ++k)
            *reinterpret_cast<bf16x8*>(to + ((long long)id * 6 * N + frag * N + k) * HELIX_DR_FRAG + 16 * lane) = o[k];
    };
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        float v[8];
        const int row = 16 * w + c, col = 32 * ks + 8 * q;
        if (ks == 0 || w > 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = sX[row][col + e];
            emit(p.x, dr_low(w, ks), v, std::integral_constant<int, 3>{});
            if constexpr (!BWD) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = sP[row][col + e];
                emit(p.p, dr_low(w, ks), v, std::integral_constant<int, NO>{});
            }
        }
        if constexpr (BWD) {
            if (ks == 1 || w < 2) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = sX[col + e][row];
                emit(p.xt, dr_up(w, ks), v, std::integral_constant<int, 3>{});
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = sP[col + e][row];
                emit(p.pt, dr_up(w, ks), v, std::integral_constant<int, 3>{});
            }
        }
    }
}

// ---- the walk -----------------------------------------------------------------------------
//
// Sixteen columns of a state, four waves. Wave w forms rows 16 w .. of K S and Q S, of
// R = V - e^G K S and of D = X R, and keeps the rows NK / 4 w .. of S in registers. S, R, D and
// e^(G_63 - G) D go from wave to wave through LDS, in bf16 parts and with the index that the
// next product sums over running inside a row. A chunk is three barriers; everything that does
// not depend on the state (K's rows, the fragments of X and P, the wave's rows of Q and V) is
// loaded a chunk ahead.
// KEEP: no outputs; the states before the chunks and D are stored (fp32) for the backward pass.
template <typename T, int NK, bool KEEP>
__device__ void delta_walk(const HelixDeltaParams& p) {
    constexpr int NPL = dr_planes<T>, NO = dr_out_planes<T>, KP = NK + 8, TP = DR_C + 8, NT = NK / 64, KS = NK / 32;
    __shared__ __bf16 sK[2][NPL][DR_C][KP];
    __shared__ __bf16 sS[3][16][KP];
    __shared__ __bf16 sR[3][16][TP], sU[3][16][TP], sD[KEEP ? 1 : NO][KEEP ? 1 : 16][TP];
    const int tid = threadIdx.x, lane = lane_id(), w = wave_uniform(), c = lane & 15, q = lane >> 4;
    const unsigned id = xcd_logical_id(blockIdx.x, gridDim.x);   // a head's slices share an XCD's cache
    const int slice = (int)(id % (unsigned)p.n_slice);
    const unsigned sh = id / (unsigned)p.n_slice;
    const int seq = (int)(sh / (unsigned)p.n_head), h = (int)(sh % (unsigned)p.n_head), hk = h / p.share;
    const int p0 = 16 * slice, P = p.n_val, N = p.n_key;
    const unsigned state_bytes = (unsigned)N * (unsigned)P * 4u;
    const int row0 = 16 * w + 4 * q;
    // Register r of tile i: S[n = NT 16 w + 16 i + 4 q + r][p0 + c].
    auto state_off = [&](int i, int r) {
        const int n = NT * 16 * w + 16 * i + 4 * q + r;
        return n < N && p0 + c < P ? (n * P + p0 + c) * 4 : (int)0x80000000;
    };
    f32x4 S[NT];
    {
        const helix_rsrc r0 = make_rsrc_u(p.s0 + (long long)sh * N * P, p.s0 ? state_bytes : 0u);   // none: reads 0
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[i][r] = buf_f32(r0, state_off(i, r), 0);
    }
    constexpr int PER = DR_C * (NK / 8) / 256;
    struct Ahead {
        Raw8<T> k[PER], q[KEEP ? 1 : KS];
        bf16x8 x[2][3], p[KEEP ? 1 : 2][KEEP ? 1 : NO];
        unsigned v[4];
        f32x4 start, left;
        float all;
    } next;
    auto load = [&](int ch) {
        const long long t0 = (long long)(p.chunk0 + ch) * DR_C;
        const int len = (int)min((long long)DR_C, p.n_tok - t0);
        const Rows<T> rk(p.k, seq * p.seq_k + hk * p.head_k + t0 * p.tok_k, p.tok_k, len, N);
        const Rows<T> rv(p.v, seq * p.seq_v + h * p.head_v + t0 * p.tok_v, p.tok_v, len, P);
#pragma unroll
        for (int i = 0; i < PER; ++i) next.k[i] = rk.load8((tid + 256 * i) / (NK / 8), 8 * ((tid + 256 * i) % (NK / 8)));
        const long long at = (long long)sh * p.n_chunk + ch;
        const char* x = p.x + at * (6 * 3 * HELIX_DR_FRAG) + 16 * lane;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (ks && w < 2) break;
#pragma unroll
            for (int k = 0; k < 3; ++k) next.x[ks][k] = *reinterpret_cast<const bf16x8*>(x + (dr_low(w, ks) * 3 + k) * HELIX_DR_FRAG);
        }
        if constexpr (!KEEP) {
            const Rows<T> rq(p.q, seq * p.seq_q + hk * p.head_q + t0 * p.tok_q, p.tok_q, len, N);
#pragma unroll
            for (int s = 0; s < KS; ++s) next.q[s] = rq.load8(16 * w + c, 32 * s + 8 * q);
            const char* pp = p.p + at * (6 * NO * HELIX_DR_FRAG) + 16 * lane;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                if (ks && w < 2) break;
#pragma unroll
                for (int k = 0; k < NO; ++k) next.p[ks][k] = *reinterpret_cast<const bf16x8*>(pp + (dr_low(w, ks) * NO + k) * HELIX_DR_FRAG);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) next.v[r] = rv.raw(row0 + r, p0 + c);
        const float* dec = p.decay + at * (HELIX_DR_DECAY / 4);
        next.start = *reinterpret_cast<const f32x4*>(dec + row0);
        next.left = *reinterpret_cast<const f32x4*>(dec + 64 + row0);
        next.all = dec[63];
    };
    auto put_k = [&](int buf) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int row = (tid + 256 * i) / (NK / 8), col = 8 * ((tid + 256 * i) % (NK / 8));
            bf16x8 o[NPL];
            dr_operand<T>(next.k[i], N - col, o);
#pragma unroll
            for (int k = 0; k < NPL; ++k) *reinterpret_cast<bf16x8*>(&sK[buf][k][row][col]) = o[k];
        }
    };
    auto put_s = [&] {
#pragma unroll
        for (int i = 0; i < NT; ++i)
            dr_put4<3>(&sS[0][c][NT * 16 * w + 16 * i + 4 * q], 16 * KP, S[i][0], S[i][1], S[i][2], S[i][3]);
    };
    load(0);
    put_k(0);
    put_s();
    for (int ch = 0; ch < p.n_chunk; ++ch) {
        const int buf = ch & 1;
        const Ahead now = next;
        if (ch + 1 < p.n_chunk) load(ch + 1);
        const long long at = (long long)sh * p.n_chunk + ch;
        const long long t0 = (long long)(p.chunk0 + ch) * DR_C;
        const int len = (int)min((long long)DR_C, p.n_tok - t0);
        __syncthreads();
        if constexpr (KEEP) {
            const helix_rsrc rs = make_rsrc_u(p.keep_s + at * N * P, state_bytes);
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) __builtin_amdgcn_raw_buffer_store_b32(as_u32(S[i][r]), rs, state_off(i, r), 0, 0);
        }
        f32x4 ks_ = zero4(), qs = zero4();
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int col = 32 * s + 8 * q;
            bf16x8 a[NPL], b[3];
            dr_get8<NPL>(&sK[buf][0][16 * w + c][col], DR_C * KP, a);
            dr_get8<3>(&sS[0][c][col], 16 * KP, b);
            ks_ = dr_mfma<NPL, 3>(a, b, ks_);
            if constexpr (!KEEP) {
                bf16x8 aq[NPL];
                dr_operand<T>(now.q[s], N - col, aq);
                qs = dr_mfma<NPL, 3, NO>(aq, b, qs);
            }
        }
        f32x4 R;
#pragma unroll
        for (int r = 0; r < 4; ++r) R[r] = raw_f32<T>(now.v[r]) - now.start[r] * ks_[r];
        dr_put4<3>(&sR[0][c][row0], 16 * TP, R[0], R[1], R[2], R[3]);
        __syncthreads();
        f32x4 D = zero4();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (ks && w < 2) break;
            bf16x8 b[3];
            dr_get8<3>(&sR[0][c][32 * ks + 8 * q], 16 * TP, b);
            D = dr_mfma<3, 3>(now.x[ks], b, D);
        }
        dr_put4<3>(&sU[0][c][row0], 16 * TP, D[0] * now.left[0], D[1] * now.left[1], D[2] * now.left[2], D[3] * now.left[3]);
        if constexpr (KEEP) {
            const Rows<float> rd(p.keep_d, at * DR_C * P, P, DR_C, P);
#pragma unroll
            for (int r = 0; r < 4; ++r) rd.store(row0 + r, p0 + c, D[r]);
        } else {
            dr_put4<NO>(&sD[0][c][row0], 16 * TP, D[0], D[1], D[2], D[3]);
        }
        __syncthreads();
        if constexpr (!KEEP) {
            f32x4 o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = p.scale * now.start[r] * qs[r];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                if (ks && w < 2) break;
                bf16x8 b[NO];
                dr_get8<NO>(&sD[0][c][32 * ks + 8 * q], 16 * TP, b);
                o = dr_mfma<NO, NO, NO>(now.p[ks], b, o);
            }
            const Rows<T> ro(p.o, seq * p.seq_o + h * p.head_o + t0 * p.tok_o, p.tok_o, len, P);
#pragma unroll
            for (int r = 0; r < 4; ++r) ro.store(row0 + r, p0 + c, o[r]);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) S[i] *= now.all;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            bf16x8 b[3];
            dr_get8<3>(&sU[0][c][32 * ks + 8 * q], 16 * TP, b);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                bf16x8 a[NPL];
                dr_get8_t<NPL>(&sK[buf][0][32 * ks + 8 * q][NT * 16 * w + 16 * i], KP, DR_C * KP, c, a);
                S[i] = dr_mfma<NPL, 3>(a, b, S[i]);
            }
        }
        put_s();
        if (ch + 1 < p.n_chunk) put_k(buf ^ 1);
    }
    if (p.s) {
        const helix_rsrc r1 = make_rsrc_u(p.s + (long long)sh * N * P, state_bytes);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) __builtin_amdgcn_raw_buffer_store_b32(as_u32(S[i][r]), r1, state_off(i, r), 0, 0);
    }
}

}  // namespace

#define DR_KERNELS(TAG, T, NK)                                                                                              \
    extern "C" __global__ __launch_bounds__(256) void helix_delta_steps_##TAG##_##NK(HelixDeltaParams p) {                  \
        delta_steps<T, NK / 16>(p);                                                                                         \
    }                                                                                                                       \
    extern "C" __global__ __launch_bounds__(256) void helix_delta_prep_##TAG##_##NK(HelixDeltaParams p) {                   \
        delta_prep<T, NK, false>(p);                                                                                        \
    }                                                                                                                       \
    extern "C" __global__ __launch_bounds__(256) void helix_delta_walk_##TAG##_##NK(HelixDeltaParams p) {                   \
        delta_walk<T, NK, false>(p);                                                                                        \
    }
DR_KERNELS(f32, float, 64)
DR_KERNELS(f32, float, 128)
DR_KERNELS(f16, _Float16, 64)
DR_KERNELS(f16, _Float16, 128)
DR_KERNELS(bf16, __bf16, 64)
DR_KERNELS(bf16, __bf16, 128)
