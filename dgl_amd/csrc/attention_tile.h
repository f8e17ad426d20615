// Building blocks of the attention kernels (attention.hip, attention_step.hip): element types, matrix-instruction
// operands, staging of 64-row tiles in LDS, and the scalar part of a score.
//
// All products run on the 16 x 16 matrix instructions with the reduction index split over the four 16-lane groups of a
// wave (lane = 16 g + c).  An accumulator holds column c and rows 4 g + r, r = 0..3.  Two products are chained without
// leaving registers: S^T = K Q^T leaves lane (g, c) with the scores of query c against keys 4 g + r, which is the operand
// layout the second product O^T = V^T P^T needs for its reduction over keys - the key that a reduction slot stands for is
// free as long as both operands agree, so no shuffle sits between the two.
#pragma once
#include "common.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

#define ATTN_ROWS 64          // rows of a staged tile
#define ATTN_LOG2E 1.4426950408889634f
#define ATTN_LN2 0.6931471805599453f

__device__ __forceinline__ float attn_inf() { return __builtin_inff(); }

// maximum / sum over the four 16-lane groups, in every lane
__device__ __forceinline__ float group_max(float x) {
    u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
    s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float group_sum(float x) {
    u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Maximum as a median with infinity: one instruction, where fmaxf first quiets operands it cannot prove to be no signalling
// NaN.  (A NaN score makes its row NaN through the sum, whatever the maximum is.)
__device__ __forceinline__ float fast_max(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, __builtin_inff()); }

// Selections by masks of bits (all ones: keep).  A comparison into a scalar register and a v_cndmask from it take 27 cycles
// of a wave here, a subtraction, a shift and a v_bfi 15.
// (the shift is written in assembly: the compiler would turn it back into the comparison)
__device__ __forceinline__ unsigned mask_below(int x, int limit) {       // x < limit
    unsigned m;
    asm("v_ashrrev_i32 %0, 31, %1" : "=v"(m) : "v"(x - limit));
    return m;
}
__device__ __forceinline__ unsigned mask_equal(int a, int b) {
    unsigned d;
    asm("v_min_u32 %0, 1, %1" : "=v"(d) : "v"(a ^ b));
    return d - 1u;
}
__device__ __forceinline__ float keep_or(unsigned mask, float x, float other) {
    return __uint_as_float((__float_as_uint(x) & mask) | (__float_as_uint(other) & ~mask));
}
__device__ __forceinline__ float keep_or_zero(unsigned mask, float x) { return __uint_as_float(__float_as_uint(x) & mask); }

// tanh to about 4 ulp: 1 - 2 / (e^{2y} + 1) away from zero, its odd series (to y^11) near it, where the difference would cancel
__device__ __forceinline__ float attn_tanh(float y) {
    const float e = __builtin_amdgcn_exp2f(y * (2.0f * ATTN_LOG2E));
    const float far = fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
    const float z = y * y;
    float p = fmaf(z, -8.8632355e-3f, 2.1869488e-2f);
    p = fmaf(z, p, -5.3968254e-2f);
    p = fmaf(z, p, 1.3333334e-1f);
    p = fmaf(z, p, -3.3333334e-1f);
    const float near = fmaf(y * z, p, y);
    return z < 0.16f ? near : far;
}
// A capped score cap tanh(x / cap) is cap - 2 cap r with r = 1 / (e^{2x/cap} + 1), in 11 issue slots instead of 23: off by up to
// 3 cap 2^-24 absolutely, which 16-bit operands and probabilities drown.  Binary32 takes 2 cap h with h = tanh / 2 =
// (e^{2x/cap} / 2 - 1/2) / (e^{2x/cap} + 1): the difference is exact near zero, what remains is a quarter of that, for three more
// operations.  Above CAP_PRECISE the relative error of small scores would count (4e-6 at 64): there tanh is taken to a few ulp.
// 1 - tanh^2 = 4 (r - r^2) = 4 (1/4 - h^2).
#define CAP_PRECISE 64.0f
enum { CAP_NONE = 0, CAP_FAST = 1, CAP_EXACT = 2 };
__device__ __forceinline__ float cap_r(float y2) { return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y2) + 1.0f); }

__device__ __forceinline__ float cap_h(float y2) {
    // limited from above, or infinity / infinity would follow; v_minimum3_f32 leaves a NaN what it is (fmin and the median drop it)
    const float e = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(y2, 60.0f));
    return fmaf(e, 0.5f, -0.5f) * __builtin_amdgcn_rcpf(e + 1.0f);
}

// scale, 2 log2(e) scale / cap and the cap itself have to be ordinary binary32 numbers (a cap that underflows would be none)
inline bool score_params_fit(float scale, float cap) {
    const float s = scale < 0.0f ? -scale : scale;
    return s <= 1e38f && (cap == 0.0f || (cap >= 0x1p-126f && cap < 3.0e38f && s / cap <= 1e38f));
}

// the scalar part of a score, in units of log2
struct ScoreParams {
    float mul, mul2, cap2, slope2;     // factor of the dot product; 2 log2(e) scale / cap; cap log2(e); slope log2(e)
    int cap, bias;
};
__device__ __forceinline__ ScoreParams score_params(float scale, float cap, int bias, const float *slope, int h) {
    ScoreParams p;
    p.cap = cap > 0.0f ? (cap <= CAP_PRECISE ? CAP_FAST : CAP_EXACT) : CAP_NONE;
    p.mul = p.cap ? scale / cap : scale * ATTN_LOG2E;
    p.mul2 = p.mul * (2.0f * ATTN_LOG2E);
    p.cap2 = cap * ATTN_LOG2E;
    p.bias = bias;
    p.slope2 = bias ? slope[h] * ATTN_LOG2E : 0.0f;
    return p;
}
// without the bias, for a single dot product (th: its tanh, 0 without a cap)
__device__ __forceinline__ float score_of(const ScoreParams &p, float dot, float &th) {
    th = 0.0f;
    if (p.cap == CAP_NONE) return dot * p.mul;
    th = p.cap == CAP_FAST ? 2.0f * cap_h(dot * p.mul2) : attn_tanh(dot * p.mul);
    return p.cap2 * th;
}

// ---- element types -----------------------------------------------------------------------------------------------
// F32: operands as three bfloat16 terms (below), so none is rounded.  F16 / BF16: the tile operands are the inputs
// as they are, probabilities and score gradients are rounded to the type (relative error 2^-11 / 2^-8 each, independent
// from term to term), accumulation is binary32.
enum { ATTN_F32 = 0, ATTN_F16 = 1, ATTN_BF16 = 2 };

template <int TYPE> struct Elem { typedef unsigned short raw; static constexpr int bytes = 2; };
template <> struct Elem<ATTN_F32> { typedef float raw; static constexpr int bytes = 4; };

template <int TYPE> __device__ __forceinline__ float elem_to_float(typename Elem<TYPE>::raw x) {
    if constexpr (TYPE == ATTN_F32) return x;
    else if constexpr (TYPE == ATTN_F16) {
        float f = (float)__builtin_bit_cast(_Float16, x);
        asm("" : "+v"(f));     // keeps the conversion apart: mixed-precision FMAs stay the sign of split_f16.h's assembly
        return f;
    } else return __uint_as_float((unsigned)x << 16);
}

// four consecutive elements stored with one access (8 or 16 bytes)
template <int TYPE> __device__ __forceinline__ void store4(typename Elem<TYPE>::raw *p, f32x4 v) {
    if constexpr (TYPE == ATTN_F32) *reinterpret_cast<f32x4 *>(p) = v;
    else if constexpr (TYPE == ATTN_F16) *reinterpret_cast<f16x4 *>(p) = __builtin_convertvector(v, f16x4);
    else *reinterpret_cast<bf16x4 *>(p) = __builtin_convertvector(v, bf16x4);
}

// the value that a store of x leaves
template <int TYPE> __device__ __forceinline__ f32x4 rounded4(f32x4 x) {
    if constexpr (TYPE == ATTN_F32) return x;
    else if constexpr (TYPE == ATTN_F16) {
        const u32x2 h = __builtin_bit_cast(u32x2, __builtin_convertvector(x, f16x4));
        return f32x4{elem_to_float<TYPE>((unsigned short)h[0]), elem_to_float<TYPE>((unsigned short)(h[0] >> 16)),
                     elem_to_float<TYPE>((unsigned short)h[1]), elem_to_float<TYPE>((unsigned short)(h[1] >> 16))};
    } else {
        const u32x2 h = __builtin_bit_cast(u32x2, __builtin_convertvector(x, bf16x4));
        return f32x4{__uint_as_float(h[0] << 16), __uint_as_float(h[0] & 0xffff0000u), __uint_as_float(h[1] << 16),
                     __uint_as_float(h[1] & 0xffff0000u)};
    }
}

template <int TYPE> __device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 acc) {      // 32 reduction slots
    if constexpr (TYPE == ATTN_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}

// Binary32 operands are split into terms when they are loaded: the score's factor goes into the one that stays in registers
// (one more rounding of 2^-24 per element, as the split's own), and scaled() leaves the products as they are.
__device__ __forceinline__ float score_factor(const ScoreParams &p) { return p.cap == CAP_FAST ? p.mul2 : p.mul; }
template <int TYPE> __device__ __forceinline__ float scaled(float dot, float factor) { return TYPE == ATTN_F32 ? dot : dot * factor; }

// ---- binary32 operands as three bfloat16 terms ----------------------------------------------------------------------
// x = hi + mid + lo exactly (8 significand bits each, by truncation); a product is hh + hm + mh + hl + lh + mm, what is left
// out is below 2^-23 of it.  Six bfloat16 products of 17 cycles replace eight binary32 ones of 32 per 16 x 16 x 32 block -
// and the binary32 matrix instructions of gfx950 hold the vector ALU back for their whole duration (measured: a stream of
// them beside vector work takes the sum of both times), the bfloat16 ones for two thirds of theirs.
struct Split3 {
    float hi, mid, lo;             // bfloat16 values in binary32 (lo: its upper half counts)
};
__device__ __forceinline__ Split3 split3(float x) {
    Split3 s;
    s.hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    const float r = x - s.hi;
    s.mid = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
    s.lo = r - s.mid;
    return s;
}
__device__ __forceinline__ unsigned pack_upper(float a, float b) {       // upper halves: a in the low half of the word
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// Shape of a tile of ATTN_ROWS rows of DP (padded head size) elements in LDS: one plane of 16-bit elements, or three of a
// binary32 tile's terms.  A plane's rows are DP / 8 pieces of 16 bytes; pieces are permuted so that the access
// patterns spread over all 64 banks: 16 rows at one piece (operand reads, staging writes) and 16 rows at two neighbouring
// pieces (transposing reads).
template <int TYPE, int DP> struct Shape {
    typedef typename Elem<TYPE>::raw raw;
    static constexpr int terms = TYPE == ATTN_F32 ? 3 : 1;
    static constexpr int mma = TYPE == ATTN_F16 ? ATTN_F16 : ATTN_BF16;
    static constexpr int vec = 16 / Elem<TYPE>::bytes;               // elements of a 16-byte global access
    static constexpr int pieces = DP / 8;                            // 16-byte pieces of a plane's row
    static constexpr int chunks = DP < 32 ? 1 : DP / 32;             // reductions of 32 over the head size
    static constexpr int dt = DP / 16;                               // 16-row tiles over the head size
    static constexpr int plane = ATTN_ROWS * DP * 2, bytes = terms * plane;
    static constexpr int per_row = DP / vec;                         // 16-byte global pieces of a row
    // operands of one 16-row block: A from LDS, B in registers.  Heads of 16 fill half of the 32 slots; binary32 puts two
    // terms side by side there: A [h m], [h l] against B [h m], [m h], [l h] are the six products in three instructions.
    static constexpr int a_regs = DP < 32 && terms == 3 ? 2 : terms * chunks, b_regs = terms * chunks;
};
// (the permutation looks at the row within its block of 16 alone: blocks differ by a constant, which an LDS access adds free)
template <int TYPE, int DP> __device__ __forceinline__ unsigned piece_at(int row, int piece) {
    constexpr int P = Shape<TYPE, DP>::pieces, SH = P == 2 ? 3 : P == 4 ? 2 : P == 8 ? 1 : 0;
    const int low = row & 15;
    return (unsigned)((row >> 4) * 16 * P + low * P + (piece ^ ((low >> SH) & (P - 1)))) * 16u;
}

template <int TYPE, int DP> struct RowFrag { u32x4 c[Shape<TYPE, DP>::a_regs]; };     // A: 16 rows of a tile
template <int TYPE, int DP> struct ColFrag { u32x4 c[Shape<TYPE, DP>::b_regs]; };     // B: 16 rows kept in registers

template <int TYPE, int DP> __device__ __forceinline__ void row_frag(RowFrag<TYPE, DP> &f, const char *tile, int row, int g) {
    typedef Shape<TYPE, DP> S;
    if constexpr (DP < 32) {
        const char *at = tile + piece_at<TYPE, DP>(row, g & 1);
        if constexpr (S::terms == 3) {
            f.c[0] = *reinterpret_cast<const u32x4 *>(at + (g >> 1) * S::plane);
            f.c[1] = *reinterpret_cast<const u32x4 *>(at + (g >> 1) * 2 * S::plane);
        } else {
            f.c[0] = *reinterpret_cast<const u32x4 *>(at);           // (the upper slots meet zeros)
        }
    } else {
#pragma unroll
        for (int k = 0; k < S::chunks; ++k)
#pragma unroll
            for (int p = 0; p < S::terms; ++p)
                f.c[k * S::terms + p] = *reinterpret_cast<const u32x4 *>(tile + p * S::plane + piece_at<TYPE, DP>(row, 4 * k + g));
    }
}

// eight elements of a row in global memory from element d on; zeros beyond the head size
template <int TYPE> struct Eight { u32x4 w[Elem<TYPE>::bytes / 2]; };
template <int TYPE> __device__ __forceinline__ Eight<TYPE> load_eight(const typename Elem<TYPE>::raw *row, int d, bool live) {
    Eight<TYPE> x;
#pragma unroll
    for (int i = 0; i < Elem<TYPE>::bytes / 2; ++i)
        x.w[i] = live ? *reinterpret_cast<const u32x4 *>(row + d + i * (16 / Elem<TYPE>::bytes)) : u32x4{0, 0, 0, 0};
    return x;
}
template <int TYPE> __device__ __forceinline__ float eight_at(const Eight<TYPE> &x, int i) {
    if constexpr (TYPE == ATTN_F32) return __uint_as_float(x.w[i >> 2][i & 3]);
    else return elem_to_float<TYPE>((unsigned short)(x.w[0][i >> 1] >> (16 * (i & 1))));
}
// the first element that lane group g holds of chunk k, and whether it is the group that counts it (heads of 16: two groups
// hold the same)
template <int DP> __device__ __forceinline__ int frag_d(int k, int g) { return DP < 32 ? 8 * (g & 1) : 32 * k + 8 * g; }
template <int DP> __device__ __forceinline__ bool frag_counts(int g) { return DP >= 32 || g < 2; }

// (`factor` only for binary32 operands: score_factor)
template <int TYPE, int DP> __device__ __forceinline__ void col_frag(ColFrag<TYPE, DP> &f, const Eight<TYPE> (&x)[Shape<TYPE, DP>::chunks], int g, float factor = 1.0f) {
    typedef Shape<TYPE, DP> S;
#pragma unroll
    for (int k = 0; k < S::chunks; ++k) {
        if constexpr (S::terms == 1) {
            f.c[k] = x[k].w[0];
            if (DP < 32 && g >= 2) f.c[k] = u32x4{0, 0, 0, 0};
        } else {
            u32x4 t[3];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const Split3 a = split3(factor * eight_at<TYPE>(x[k], 2 * i)), b = split3(factor * eight_at<TYPE>(x[k], 2 * i + 1));
                t[0][i] = pack_upper(a.hi, b.hi);
                t[1][i] = pack_upper(a.mid, b.mid);
                t[2][i] = pack_upper(a.lo, b.lo);
            }
            if constexpr (DP < 32) {
                f.c[0] = g < 2 ? t[0] : t[1];
                f.c[1] = g < 2 ? t[1] : t[0];
                f.c[2] = g < 2 ? t[2] : t[0];
            } else {
#pragma unroll
                for (int p = 0; p < 3; ++p) f.c[3 * k + p] = t[p];
            }
        }
    }
}

// accumulator + (16 tile rows) . (16 register rows): rows 4 g + r, column c
template <int TYPE, int DP>
__device__ __forceinline__ f32x4 dot_block(const RowFrag<TYPE, DP> &a, const ColFrag<TYPE, DP> &b, f32x4 acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f}) {
    typedef Shape<TYPE, DP> S;
    if constexpr (S::terms == 1) {
#pragma unroll
        for (int k = 0; k < S::chunks; ++k) acc = mfma32<S::mma>(a.c[k], b.c[k], acc);
    } else if constexpr (DP < 32) {
        acc = mfma32<S::mma>(a.c[1], b.c[2], acc);
        acc = mfma32<S::mma>(a.c[0], b.c[1], acc);
        acc = mfma32<S::mma>(a.c[0], b.c[0], acc);
    } else {
#pragma unroll
        for (int k = 0; k < S::chunks; ++k) {        // the small products first
            acc = mfma32<S::mma>(a.c[3 * k], b.c[3 * k + 2], acc);
            acc = mfma32<S::mma>(a.c[3 * k + 2], b.c[3 * k], acc);
            acc = mfma32<S::mma>(a.c[3 * k + 1], b.c[3 * k + 1], acc);
            acc = mfma32<S::mma>(a.c[3 * k], b.c[3 * k + 1], acc);
            acc = mfma32<S::mma>(a.c[3 * k + 1], b.c[3 * k], acc);
            acc = mfma32<S::mma>(a.c[3 * k], b.c[3 * k], acc);
        }
    }
    return acc;
}

// The second product of a chain: out[d][column] += sum over the rows of two 16-row blocks 2 tp, 2 tp + 1 of
// tile[row][d] * w[row][column]; w0 / w1 are results of dot_block for the two blocks (probabilities, score gradients),
// rounded to 16 bits here - or split into three terms.  The tile is read transposed: ds_read_b64_tr_b16 gives lane c of a
// 16-lane group element c mod 4 of the addresses of lanes c / 4 + 4 j, so lane s points at four elements of row s / 4.
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 read_transposed(const char *p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p));
}
template <int TYPE, int DP, int N, int DT>
__device__ __forceinline__ void accumulate(f32x4 (&out)[N][DT], const char *tile, int tp, const f32x4 (&w0)[N], const f32x4 (&w1)[N], int g, int c) {
    typedef Shape<TYPE, DP> S;
    static_assert(DT == S::dt, "accumulators of another head size");
    u32x4 b[N][S::terms];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if constexpr (TYPE == ATTN_F16) {
            const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_convertvector(w0[n], f16x4)), hi = __builtin_bit_cast(u32x2, __builtin_convertvector(w1[n], f16x4));
            b[n][0] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        } else if constexpr (TYPE == ATTN_BF16) {
            const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_convertvector(w0[n], bf16x4)), hi = __builtin_bit_cast(u32x2, __builtin_convertvector(w1[n], bf16x4));
            b[n][0] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const Split3 x = split3(i < 2 ? w0[n][2 * i] : w1[n][2 * i - 4]), y = split3(i < 2 ? w0[n][2 * i + 1] : w1[n][2 * i - 3]);
                b[n][0][i] = pack_upper(x.hi, y.hi);
                b[n][1][i] = pack_upper(x.mid, y.mid);
                b[n][2][i] = pack_upper(x.lo, y.lo);
            }
        }
    }
#pragma unroll
    for (int d = 0; d < S::dt; ++d) {
        u32x4 a[S::terms];
#pragma unroll
        for (int p = 0; p < S::terms; ++p) {
            const char *at = tile + piece_at<TYPE, DP>(4 * g + (c >> 2), 2 * d + ((c >> 1) & 1)) + 8 * (c & 1) + p * S::plane + 64 * DP * tp;
            const u32x2 lo = read_transposed(at), hi = read_transposed(at + 32 * DP);
            a[p] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if constexpr (S::terms == 3) {
                out[n][d] = mfma32<S::mma>(a[0], b[n][2], out[n][d]);
                out[n][d] = mfma32<S::mma>(a[2], b[n][0], out[n][d]);
                out[n][d] = mfma32<S::mma>(a[1], b[n][1], out[n][d]);
                out[n][d] = mfma32<S::mma>(a[0], b[n][1], out[n][d]);
                out[n][d] = mfma32<S::mma>(a[1], b[n][0], out[n][d]);
            }
            out[n][d] = mfma32<S::mma>(a[0], b[n][0], out[n][d]);
        }
    }
}

// ---- staging ------------------------------------------------------------------------------------------------------
// Two [rows][D] matrices pass through LDS tile by tile, in pieces of 16 bytes that a thread holds between its global loads and its
// LDS writes: `held` rows, `step` apart, of one piece (two for the widest rows) of both matrices, so that every thread has the
// same share of the work - binary32 pieces are split into their terms here.  The narrowest rows have 128 pieces: two waves take
// one matrix, two the other.  Row strides are scalars and a piece's offset from the tile is below 2^32 (the launcher's check), so
// that a load is a scalar address plus a 32-bit offset.
template <int TYPE, int DP> struct Stager {
    typedef Shape<TYPE, DP> S;
    static constexpr int held = S::per_row >= 16 ? 4 : S::per_row >= 8 ? 2 : 1, step = ATTN_ROWS / held, units = step * S::per_row;
    static constexpr bool both = units >= 256;
    static constexpr int plans = both ? units / 256 : 1;
    static_assert(step % 16 == 0 && (both || units == 128), "a thread's rows share their permutation");
    u32x4 r[both ? 2 : 1][plans][held];
    int id[plans][held];
    unsigned off[both ? 2 : 1][plans], at[plans];
    int grp[plans];
    bool in[plans];
    int which;                                   // !both: the wave's matrix
    unsigned rb0, rb1;                           // bytes between rows

    __device__ __forceinline__ void init(int64_t stride0, int64_t stride1, int D) {
        const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
        which = !both && wave >= 2;
        rb0 = (unsigned)(stride0 * Elem<TYPE>::bytes);
        rb1 = (unsigned)(stride1 * Elem<TYPE>::bytes);
#pragma unroll
        for (int x = 0; x < plans; ++x) {
            const int u = (int)threadIdx.x + 256 * x - (which ? 128 : 0), piece = u % S::per_row;
            grp[x] = u / S::per_row;
            in[x] = piece * S::vec < D;
            if constexpr (both) {
                off[0][x] = (unsigned)grp[x] * rb0 + 16u * (unsigned)piece;
                off[1][x] = (unsigned)grp[x] * rb1 + 16u * (unsigned)piece;
            } else {
                off[0][x] = (unsigned)grp[x] * (which ? rb1 : rb0) + 16u * (unsigned)piece;
            }
            at[x] = S::terms == 1 ? piece_at<TYPE, DP>(grp[x], piece) : piece_at<TYPE, DP>(grp[x], piece >> 1) + 8 * (piece & 1);
        }
    }
    // the tiles that start at t0 / t1 with `rows` rows left (rows beyond are zero); ids: the rows' document ids or nullptr
    __device__ __forceinline__ void load(const char *t0, const char *t1, int rows, const int *ids) {
#pragma unroll
        for (int m = 0; m < (both ? 2 : 1); ++m) {
            const char *t = both ? (m ? t1 : t0) : (which ? t1 : t0);
            const unsigned rb = both ? (m ? rb1 : rb0) : (which ? rb1 : rb0);
#pragma unroll
            for (int x = 0; x < plans; ++x)
#pragma unroll
                for (int i = 0; i < held; ++i) {
                    const bool live = in[x] && (rows >= ATTN_ROWS || grp[x] + step * i < rows);
                    r[m][x][i] = live ? *reinterpret_cast<const u32x4 *>(t + (uint64_t)((unsigned)(step * i) * rb) + off[m][x]) : u32x4{0, 0, 0, 0};
                }
        }
        if (ids != nullptr) {
#pragma unroll
            for (int x = 0; x < plans; ++x)
#pragma unroll
                for (int i = 0; i < held; ++i) id[x][i] = grp[x] + step * i < rows ? ids[grp[x] + step * i] : -1;
        }
    }
    // Rows of padding (document id < 0) may hold anything: they are staged as zeros, so that a NaN among them does not send
    // the whole tile down the careful path.
    __device__ __forceinline__ void write(char *l0, char *l1, bool skip) {
#pragma unroll
        for (int x = 0; x < plans; ++x) {
#pragma unroll
            for (int m = 0; m < (both ? 2 : 1); ++m) {
                char *l = (both ? (m ? l1 : l0) : (which ? l1 : l0)) + at[x];
#pragma unroll
                for (int i = 0; i < held; ++i) {
                    u32x4 v = r[m][x][i];
                    if (skip) {
                        unsigned keep;
                        asm("v_ashrrev_i32 %0, 31, %1" : "=v"(keep) : "v"(id[x][i]));
#pragma unroll
                        for (int w = 0; w < 4; ++w) v[w] &= ~keep;
                    }
                    char *to = l + 16 * S::pieces * step * i;
                    if constexpr (S::terms == 1) {
                        *reinterpret_cast<u32x4 *>(to) = v;
                    } else {                     // four binary32 elements are half a piece of each plane
                        Split3 y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = split3(__uint_as_float(v[e]));
                        *reinterpret_cast<u32x2 *>(to) = u32x2{pack_upper(y[0].hi, y[1].hi), pack_upper(y[2].hi, y[3].hi)};
                        *reinterpret_cast<u32x2 *>(to + S::plane) = u32x2{pack_upper(y[0].mid, y[1].mid), pack_upper(y[2].mid, y[3].mid)};
                        *reinterpret_cast<u32x2 *>(to + 2 * S::plane) = u32x2{pack_upper(y[0].lo, y[1].lo), pack_upper(y[2].lo, y[3].lo)};
                    }
                }
            }
        }
    }
};
