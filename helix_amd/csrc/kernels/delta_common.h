// delta_common.h -- what the delta rule's kernels share: operands of 16 x 16 x 32
// matrix instructions in bf16 parts, rows of tokens, decays.
//
// v_mfma_f32_16x16x32_bf16, lane = 16 q + c:  A[i][k]: lane holds A[c][8 q + e], e = 0..7;
// B[k][j]: B[8 q + e][c];  D[i][j]: register r holds D[4 q + r][c].
//
// An fp32 value is three bf16 parts, and a product of two the six products of parts i, j
// with i + j <= 2: fp32's own accuracy (helix_common.h). A bf16 element is one part, an f16
// one two, exactly. Operands that only a 16-bit output takes are in three parts too: an output
// may be a small difference of large sums, which two parts (2^-18 of each) would be seen in.
#ifndef HELIX_DELTA_COMMON_H
#define HELIX_DELTA_COMMON_H

#include "layer_common.h"

namespace {

constexpr int DR_C = HELIX_DR_CHUNK;

// Rows of W = 64 or 128 elements in LDS, without padding: the place of a row's chunk of eight (16 bytes), turned by its row so
// that the sixteen rows' chunks which lanes read together, in whichever groups the hardware takes them, are on banks of
// their own.
template <int W>
HELIX_DEV int dr_at(int row, int chunk) {
    static_assert(W == 64 || W == 128, "rows of 64 or 128");
    return row * W + 8 * (W == 128 ? chunk ^ (row & 15) : chunk ^ (row >> 1 & 7));
}

template <typename T> constexpr int dr_planes = __is_same(T, float) ? 3 : __is_same(T, _Float16) ? 2 : 1;

// Products of the parts i, j with i + j < 3, smallest first.
template <int NA, int NB>
HELIX_DEV f32x4 dr_mfma(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x4 acc) {
#pragma unroll
    for (int sum = 2; sum >= 0; --sum)
#pragma unroll
        for (int i = sum; i >= 0; --i)
            if (i < NA && sum - i < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[sum - i], acc, 0, 0, 0);
    return acc;
}

// The same into a sum of its own for each i + j: three chains, so that none of the products waits for the one before it.
struct DrAcc {
    f32x4 s[3];
    __device__ __forceinline__ DrAcc() { s[0] = s[1] = s[2] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }
    __device__ __forceinline__ f32x4 sum() const { return (s[2] + s[1]) + s[0]; }
};
// Sums of a wave that has NC blocks of columns: with two, their chains are enough side by side, and one sum for each spares
// registers.
struct DrAcc1 {
    f32x4 s;
    __device__ __forceinline__ DrAcc1() { s = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }
    __device__ __forceinline__ f32x4 sum() const { return s; }
};
template <int NC> struct DrAccOf { typedef DrAcc type; };
template <> struct DrAccOf<2> { typedef DrAcc1 type; };
template <int NA, int NB>
HELIX_DEV void dr_mfma(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], DrAcc1& acc) {
    acc.s = dr_mfma<NA, NB>(a, b, acc.s);
}
// Of products with NPL parts on both sides; one part's have one sum.
template <int NPL>
HELIX_DEV f32x4 dr_sum(const DrAcc& a) { return NPL == 1 ? a.s[0] : a.sum(); }
template <int NA, int NB>
HELIX_DEV void dr_mfma(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], DrAcc& acc) {
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int sum = 2; sum >= 0; --sum)
            if (sum - i >= 0 && sum - i < NB)
                acc.s[sum] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[sum - i], acc.s[sum], 0, 0, 0);
}

// END: of values that may reach the end of fp32, which lies past bf16's: the first part stays a number, the others have the rest.
// (What is not finite stays so: the rest of an infinity is one.)
template <int NPL, bool END = false>
HELIX_DEV void dr_split2(float a, float b, unsigned (&w)[NPL]) {
    if constexpr (NPL == 3 && END) {
        constexpr float kTop = 0x1.fep127f;   // bf16's largest
        w[0] = pk_bf16(__builtin_amdgcn_fmed3f(a, -kTop, kTop), __builtin_amdgcn_fmed3f(b, -kTop, kTop));
        split2_pair(sub_lo(a, w[0]), sub_hi(b, w[0]), w[1], w[2]);
    } else if constexpr (NPL == 3) split3_pair(a, b, w[0], w[1], w[2]);
    else if constexpr (NPL == 2) split2_pair(a, b, w[0], w[1]);
    else w[0] = pk_bf16(a, b);
}
template <int NPL, bool END = false>
HELIX_DEV void dr_split8(const float (&v)[8], bf16x8 (&o)[NPL]) {
    u32x4 q[NPL];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        unsigned w[NPL];
        dr_split2<NPL, END>(v[2 * e], v[2 * e + 1], w);
#pragma unroll
        for (int k = 0; k < NPL; ++k) q[k][e] = w[k];
    }
#pragma unroll
    for (int k = 0; k < NPL; ++k) o[k] = __builtin_bit_cast(bf16x8, q[k]);
}

// Eight stored elements as an operand's parts, those from n on cleared. OWN: of what the kernels stored, not the caller.
template <typename T, bool OWN = false>
HELIX_DEV void dr_operand(const Raw8<T>& v, int n, bf16x8 (&o)[dr_planes<T>]) {
    if constexpr (__is_same(T, __bf16)) {
        u32x4 w = v.w[0];
        if (n < 8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] &= (2 * e < n ? 0xffffu : 0u) | (2 * e + 1 < n ? 0xffff0000u : 0u);
        }
        o[0] = __builtin_bit_cast(bf16x8, w);
    } else {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = e < n ? at8(v, e) : 0.0f;
        dr_split8<dr_planes<T>, !OWN>(f, o);
    }
}

// The rows of a chunk's tokens of one head: `len` of them of `width` elements, `tok` elements apart. ODD: of 16 bits and an
// odd width, whose last element is half of a word that a wide load finds out of the resource's range.
template <typename T, bool ODD = false>
struct Rows {
    helix_rsrc r;
    int tok, len, width;
    __device__ Rows(const void* base, long long at, long long tok_, int len_, int width_) : tok((int)tok_), len(len_), width(width_) {
        r = make_rsrc_u(static_cast<const T*>(base) + at, len > 0 ? (unsigned)(((len - 1) * tok_ + width) * (long long)sizeof(T)) : 0u);
    }
    // Eight elements from (row, col) on; what lies outside is unspecified past the row's end and 0 past the tokens.
    __device__ __forceinline__ Raw8<T> load8(int row, int col) const {
        const int off = row < len && col < width ? (row * tok + col) * (int)sizeof(T) : (int)0x80000000;
        if constexpr (!ODD || sizeof(T) == 4) {
            return buf_load8<T>(r, off);
        } else {
            Raw8<T> o;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned a = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(r, col + 2 * e < width ? off + 4 * e : (int)0x80000000, 0, 0);
                const unsigned b = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(r, col + 2 * e + 1 < width ? off + 4 * e + 2 : (int)0x80000000, 0, 0);
                o.w[0][e] = a | b << 16;
            }
            return o;
        }
    }
    __device__ __forceinline__ unsigned raw(int row, int col) const {
        const int off = row < len && col < width ? (row * tok + col) * (int)sizeof(T) : (int)0x80000000;
        if constexpr (sizeof(T) == 4) return (unsigned)__builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
        else return (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
    }
    __device__ __forceinline__ void store(int row, int col, float v) const {
        const int off = row < len && col < width ? (row * tok + col) * (int)sizeof(T) : (int)0x80000000;
        io_store<T, 0>(r, v, off, 0);
    }
};
template <typename T>
HELIX_DEV float raw_f32(unsigned w) {
    if constexpr (sizeof(T) == 4) return as_f32(w);
    else return io_f32<T>((unsigned short)w);
}

// Four values of a result's registers (rows i .. i + 3, i a multiple of 4, of a column) as parts, side by side in row `row`
// of planes of ROWS rows of W.
template <int NPL, int W, int ROWS, bool END = false>
HELIX_DEV void dr_put4(__bf16* planes, int row, int i, float a, float b, float c, float d) {
    unsigned lo[NPL], hi[NPL];
    dr_split2<NPL, END>(a, b, lo);
    dr_split2<NPL, END>(c, d, hi);
    __bf16* to = planes + dr_at<W>(row, i >> 3) + (i & 4);
#pragma unroll
    for (int k = 0; k < NPL; ++k) *reinterpret_cast<u32x2*>(to + k * ROWS * W) = u32x2{lo[k], hi[k]};
}
// An operand's eight elements: columns col .. col + 7 (a multiple of 8) of row `row`.
template <int NPL, int W, int ROWS>
HELIX_DEV void dr_get8(const __bf16* planes, int row, int col, bf16x8 (&o)[NPL]) {
    const __bf16* from = planes + dr_at<W>(row, col >> 3);
#pragma unroll
    for (int k = 0; k < NPL; ++k) o[k] = *reinterpret_cast<const bf16x8*>(from + k * ROWS * W);
}
template <int NPL, int W, int ROWS>
HELIX_DEV void dr_put8(__bf16* planes, int row, int col, const bf16x8 (&v)[NPL]) {
    __bf16* to = planes + dr_at<W>(row, col >> 3);
#pragma unroll
    for (int k = 0; k < NPL; ++k) *reinterpret_cast<bf16x8*>(to + k * ROWS * W) = v[k];
}
// Rows row .. row + 7 of column col + c, by transposed reads: the operand of a product that sums over the rows. All sixteen
// lanes of a group name the same row (a multiple of 8) and col (of 16).
template <int NPL, int W, int ROWS>
HELIX_DEV void dr_get8_t(const __bf16* planes, int row, int col, int c, bf16x8 (&o)[NPL]) {
    const int r = row + (c >> 2), at = col + 4 * (c & 3);
    const __bf16* p0 = planes + dr_at<W>(r, at >> 3) + (at & 4);
    const __bf16* p1 = planes + dr_at<W>(r + 4, at >> 3) + (at & 4);
#pragma unroll
    for (int k = 0; k < NPL; ++k) {
        const u32x2 a = lds_read_tr16(p0 + k * ROWS * W), b = lds_read_tr16(p1 + k * ROWS * W);
        o[k] = __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]});
    }
}

// Four raw elements side by side, as widen4 takes them.
template <typename T>
HELIX_DEV typename Raw4<T>::type pack4(const unsigned (&e)[4]) {
    if constexpr (sizeof(T) == 4) return u32x4{e[0], e[1], e[2], e[3]};
    else return u32x2{e[0] | e[1] << 16, e[2] | e[3] << 16};
}

// The same elements, to be widened where they are used: a loop would keep them in twice the registers.
template <typename T>
HELIX_DEV typename Raw4<T>::type fresh4(typename Raw4<T>::type v) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) v[i] = (unsigned)vgpr_fresh((int)v[i]);
    return v;
}

// A barrier that the waves of a workgroup may meet in different places of the program (as many times each).
HELIX_DEV void dr_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

HELIX_DEV f32x4 zero4() { return f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }

// Sums of g from a chunk's start, lane = token, in fp64 (differences of neighbouring ones count). Tokens past the end have
// g = 0. What e^g cannot tell from e^-100000, infinity among it, counts as that: differences of infinities would be NaN.
HELIX_DEV double dr_log_decay(float g) { return wave_incl_sum(g < -1e5f ? -1e5 : (double)g); }

// Fragment of the block in row tile w, columns 32 ks .., of a lower triangle (ks = 0 for w < 2), or of an upper one (ks = 1
// alone for w > 1).
HELIX_DEV int dr_low(int w, int ks) { return w < 2 ? w : 2 * w - 2 + ks; }
HELIX_DEV int dr_up(int w, int ks) { return w < 2 ? 2 * w + ks : w + 2; }

}  // namespace

#endif
