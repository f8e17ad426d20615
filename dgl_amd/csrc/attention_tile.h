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
// A capped score cap tanh(x / cap) is cap - 2 cap r with r = 1 / (e^{2x/cap} + 1): off by about cap 2^-24 absolutely, no
// more than a binary32 score of that size is anyhow, in 11 issue slots instead of 23.  Above CAP_PRECISE the relative error
// of small scores would count (4e-6 at 64): there tanh is taken to a few ulp.  In both, 1 - tanh^2 = 4 (r - r^2).
#define CAP_PRECISE 64.0f
enum { CAP_NONE = 0, CAP_FAST = 1, CAP_EXACT = 2 };
__device__ __forceinline__ float cap_r(float y2) { return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y2) + 1.0f); }

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
    th = p.cap == CAP_FAST ? fmaf(-2.0f, cap_r(dot * p.mul2), 1.0f) : attn_tanh(dot * p.mul);
    return p.cap2 * th;
}

// ---- element types -----------------------------------------------------------------------------------------------
// F32: binary32 matrix instructions (FMA chains: no operand is rounded).  F16 / BF16: the tile operands are the inputs
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

// Shape of a tile of ATTN_ROWS rows of DP (padded head size) elements.
template <int TYPE, int DP> struct Shape {
    typedef typename Elem<TYPE>::raw raw;
    static constexpr bool wide = TYPE == ATTN_F32;
    static constexpr int vec = 16 / Elem<TYPE>::bytes;               // elements of a 16-byte access
    // rows are padded by 16 bytes: the 16-byte reads of 8 neighbouring rows then fall on different banks
    static constexpr int dk = wide ? DP : (DP < 32 ? 32 : DP);       // reduction length over the head size (16-bit: multiples of 32)
    static constexpr int ld = dk + vec;                              // row stride, elements
    static constexpr int ldt = ATTN_ROWS + 8;                        // row stride of a transposed 16-bit tile
    static constexpr int chunks = wide ? DP / 16 : dk / 32;          // operand registers sets over the head size
    static constexpr int dt = DP / 16;                               // 16-row tiles over the head size
    static constexpr int row_bytes = ATTN_ROWS * ld * Elem<TYPE>::bytes;
    static constexpr int t_bytes = wide ? 0 : DP * ldt * 2;          // transposed copy (binary32 reads columns in place)
    static constexpr int per_row = DP / vec;                         // 16-byte pieces of a row
    static constexpr int units = ATTN_ROWS / 4 * per_row;            // pieces of 4 rows x 16 bytes
};

// operand registers of one 16-row block over the head size
template <int TYPE, int DP> struct Frag {
    u32x4 c[Shape<TYPE, DP>::chunks];
};

// lane (g, c) of a block whose row c starts at `row`: binary32 takes d = 16 k + 4 g + i, 16-bit d = 32 k + 8 g + i
template <int TYPE, int DP>
__device__ __forceinline__ void frag_from_lds(Frag<TYPE, DP> &f, const typename Elem<TYPE>::raw *tile, int row, int g) {
    typedef Shape<TYPE, DP> S;
#pragma unroll
    for (int k = 0; k < S::chunks; ++k)
        f.c[k] = *reinterpret_cast<const u32x4 *>(tile + row * S::ld + (S::wide ? 16 * k + 4 * g : 32 * k + 8 * g));
}
template <int TYPE, int DP>
__device__ __forceinline__ void frag_from_global(Frag<TYPE, DP> &f, const typename Elem<TYPE>::raw *row, bool live, int D, int g) {
    typedef Shape<TYPE, DP> S;
#pragma unroll
    for (int k = 0; k < S::chunks; ++k) {
        const int d = S::wide ? 16 * k + 4 * g : 32 * k + 8 * g;
        f.c[k] = live && d < D ? *reinterpret_cast<const u32x4 *>(row + d) : u32x4{0, 0, 0, 0};
    }
}

template <int TYPE> __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 acc) {
    if constexpr (TYPE == ATTN_F32) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], acc, 0, 0, 0);
        return acc;
    } else if constexpr (TYPE == ATTN_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    }
}

// acc[row 4g+r][column c] += (tile rows 16 t ..) . (block whose operand registers are b)
template <int TYPE, int DP>
__device__ __forceinline__ f32x4 dot_block(const Frag<TYPE, DP> &a, const Frag<TYPE, DP> &b, f32x4 acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f}) {
#pragma unroll
    for (int k = 0; k < Shape<TYPE, DP>::chunks; ++k) acc = mfma16<TYPE>(a.c[k], b.c[k], acc);
    return acc;
}

// The second product of a chain: out[d][column] += sum over the rows of a pair of 16-row blocks 2 tp, 2 tp + 1 of
// tile[row][d] * w[row][column]; w0 / w1 are accumulators of dot_block for the two blocks.  Binary32 reads the row-major
// tile by columns; 16-bit types read the transposed copy, whose rows are stored in the order 8 g + 4 (t mod 2) + r of
// every 32, so that a lane's eight reduction slots are one 16-byte read.
template <int TYPE, int DP, int N, int DT>
__device__ __forceinline__ void accumulate(f32x4 (&out)[N][DT], const typename Elem<TYPE>::raw *tile,
                                           const typename Elem<TYPE>::raw *tile_t, int tp, const f32x4 (&w0)[N],
                                           const f32x4 (&w1)[N], int g, int c) {
    typedef Shape<TYPE, DP> S;
    static_assert(DT == S::dt, "accumulators of another head size");
    if constexpr (S::wide) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int d = 0; d < S::dt; ++d) {
                    const float a = tile[(32 * tp + 16 * t + 4 * g + r) * S::ld + 16 * d + c];
#pragma unroll
                    for (int n = 0; n < N; ++n)
                        out[n][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, t ? w1[n][r] : w0[n][r], out[n][d], 0, 0, 0);
                }
    } else {
        u32x4 b[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            u32x2 lo, hi;
            if constexpr (TYPE == ATTN_F16) {
                lo = __builtin_bit_cast(u32x2, __builtin_convertvector(w0[n], f16x4));
                hi = __builtin_bit_cast(u32x2, __builtin_convertvector(w1[n], f16x4));
            } else {
                lo = __builtin_bit_cast(u32x2, __builtin_convertvector(w0[n], bf16x4));
                hi = __builtin_bit_cast(u32x2, __builtin_convertvector(w1[n], bf16x4));
            }
            b[n] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
#pragma unroll
        for (int d = 0; d < S::dt; ++d) {
            const u32x4 a = *reinterpret_cast<const u32x4 *>(tile_t + (16 * d + c) * S::ldt + 32 * tp + 8 * g);
#pragma unroll
            for (int n = 0; n < N; ++n) out[n][d] = mfma16<TYPE>(a, b[n], out[n][d]);
        }
    }
}

// ---- staging ------------------------------------------------------------------------------------------------------
// One unit = 4 consecutive rows x 16 bytes, held by one thread between its global loads and its LDS writes.
struct Unit {
    u32x4 r[4];
};

template <int TYPE, int DP> __device__ __forceinline__ void unit_place(int u, int &grp, int &piece) {
    typedef Shape<TYPE, DP> S;
    if constexpr (S::wide) {
        piece = u % S::per_row;
        grp = u / S::per_row;
    } else {           // neighbouring threads take neighbouring row groups: their transposed 8-byte writes are contiguous
        grp = u % (ATTN_ROWS / 4);
        piece = u / (ATTN_ROWS / 4);
    }
}

// What a thread knows about its unit of every tile: byte offsets of the four rows from the tile's first (below 2^32 by the
// launcher's check, so that a load is a scalar address plus a 32-bit offset)
struct UnitPlan {
    unsigned off, row_bytes;
    int grp;
    bool in;                                   // the piece lies within the head size
};
template <int TYPE, int DP> __device__ __forceinline__ UnitPlan unit_plan(int u, int64_t stride, int D) {
    UnitPlan p;
    int piece;
    unit_place<TYPE, DP>(u, p.grp, piece);
    p.row_bytes = (unsigned)(stride * Elem<TYPE>::bytes);
    p.off = 4u * (unsigned)p.grp * p.row_bytes + 16u * (unsigned)piece;
    p.in = piece * Shape<TYPE, DP>::vec < D;
    return p;
}
// the rows of a tile that starts at `tile` with `rows` rows left; rows beyond are zero
__device__ __forceinline__ void unit_load(Unit &un, const UnitPlan &p, const char *tile, int rows) {
    if (rows >= ATTN_ROWS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) un.r[i] = p.in ? *reinterpret_cast<const u32x4 *>(tile + (p.off + i * p.row_bytes)) : u32x4{0, 0, 0, 0};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            un.r[i] = p.in && 4 * p.grp + i < rows ? *reinterpret_cast<const u32x4 *>(tile + (p.off + i * p.row_bytes)) : u32x4{0, 0, 0, 0};
    }
}
// rows of padding (document id < 0) may hold anything: they are staged as zeros, so that a NaN among them does not send the
// whole tile down the careful path
struct UnitIds {
    int id[4];
};
__device__ __forceinline__ void unit_load_ids(UnitIds &ids, const UnitPlan &p, const int *tile, int rows) {
#pragma unroll
    for (int i = 0; i < 4; ++i) ids.id[i] = 4 * p.grp + i < rows ? tile[4 * p.grp + i] : -1;
}
__device__ __forceinline__ void unit_skip(Unit &un, const UnitIds &ids) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) un.r[i][w] = ids.id[i] >= 0 ? un.r[i][w] : 0u;
}

template <int TYPE, int DP, bool ROWMAJOR, bool TRANSPOSED>
__device__ __forceinline__ void unit_write(const Unit &un, int u, typename Elem<TYPE>::raw *tile, typename Elem<TYPE>::raw *tile_t) {
    typedef Shape<TYPE, DP> S;
    int grp, piece;
    unit_place<TYPE, DP>(u, grp, piece);
    if constexpr (ROWMAJOR || S::wide) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4 *>(tile + (4 * grp + i) * S::ld + piece * S::vec) = un.r[i];
    }
    if constexpr (TRANSPOSED && !S::wide) {
        const int t = grp >> 2, at = 32 * (t >> 1) + 8 * (grp & 3) + 4 * (t & 1);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            typename Elem<TYPE>::raw *p = tile_t + (piece * 8 + 2 * w) * S::ldt + at;
            *reinterpret_cast<u32x2 *>(p) = u32x2{__builtin_amdgcn_perm(un.r[1][w], un.r[0][w], 0x05040100u),
                                                  __builtin_amdgcn_perm(un.r[3][w], un.r[2][w], 0x05040100u)};
            *reinterpret_cast<u32x2 *>(p + S::ldt) = u32x2{__builtin_amdgcn_perm(un.r[1][w], un.r[0][w], 0x07060302u),
                                                           __builtin_amdgcn_perm(un.r[3][w], un.r[2][w], 0x07060302u)};
        }
    }
}

// 16-bit row-major tiles of heads below 32: the columns beyond the head size multiply zero operands and have to be finite
template <int TYPE, int DP> __device__ __forceinline__ void zero_padding(typename Elem<TYPE>::raw *tile) {
    typedef Shape<TYPE, DP> S;
    if constexpr (!S::wide && DP < 32) {
        for (int i = threadIdx.x; i < ATTN_ROWS * (32 - DP) / 8; i += blockDim.x) {
            const int per = (32 - DP) / 8;
            *reinterpret_cast<u32x4 *>(tile + (i / per) * S::ld + DP + 8 * (i % per)) = u32x4{0, 0, 0, 0};
        }
    }
}
