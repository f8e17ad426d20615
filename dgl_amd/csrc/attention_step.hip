// Attention of one new token per row over a paged key-value cache, and the cache's append.
//
// The rows of an instance (multi-starts x beams) and the query heads that share a key head all read the same keys, so one
// pass over a sequence serves them together: a wave holds NQ blocks of 16 (row, head) queries as matrix operands and walks
// over tiles of 32 keys, S^T = K Q^T and O^T += V^T P^T on the 16 x 16 matrix instructions with a running maximum and sum.
// With few queries the operation is bound by reading the cache once; the matrix instructions' idle columns cost nothing
// there.  Every operand goes from memory straight to registers, no LDS and no barrier in the loop:
//   K  lane (g, c) reads 16 bytes of key c: exactly a matrix operand;
//   V  lane (g, c) reads VW neighbouring elements of keys 4 g + r; the output row that a lane's element i stands for is
//      chosen to be d = VW c + i, so one wide load feeds VW products (16-bit types: eight keys are packed in registers).
// A sequence is cut into `splits` ranges (few sequences, long caches) and each range over the 8 waves of a workgroup; the
// waves join through LDS, the ranges through a second kernel.
//
// A masked key contributes nothing, whatever it holds: results that are not finite are recomputed key by key.
//
// Measured, per launch: 8 ragged caches up to 65536 tokens, 32 heads over 8 of 128, bf16, 295 us = 5.5 TB/s of live keys and
// values (a copy reaches 6.6 with its reads and writes), the join of the 8 ranges 11 us, the append of one token 5 us; 32
// instances of 1000 keys, 16 rows and 8 heads of 16 with coordinates and blocked bits, binary32, 16 us = 2.1 TB/s: four tiles a
// wave behind the lookups of length, page and keys; one row over 100 keys 6 us: the same chain alone.
#include "attention_tile.h"

#include <cfloat>

namespace {

#define STEP_WAVES 8
#define STEP_TILE 32

struct StepArgs {
    const char *q, *k, *v;
    char *out;
    float *lse;
    int64_t qs[2], os[2], ks[3], vs[3];
    int B, P, Hq, Hkv, G, D, M, chunks, splits, shift, max_pages, num_pages, bias;
    float scale, cap;
    const int *table, *lengths;
    int64_t ts;
    const float *slope, *pos_q, *pos_k;
    int pos_rows;
    int64_t pks;
    const unsigned *blocked;      // 32-bit halves of the words
    int halves;
    int64_t bs;
    float *part;                  // [B Hkv][splits][M][D + 2]: sum of p v, maximum, sum of p
};

// ---- operands straight from memory: binary32 on the binary32 matrix instructions (the operation waits for memory, and a
// split into bfloat16 terms would cost vector work), 16-bit types as they are ------------------------------------------
template <int TYPE, int DP> struct DirectShape {
    static constexpr bool wide = TYPE == ATTN_F32;
    static constexpr int chunks = wide ? DP / 16 : DP < 32 ? 1 : DP / 32;   // operand register sets over the head size
    static constexpr int dt = DP / 16;
};
template <int TYPE, int DP> struct Frag {
    u32x4 c[DirectShape<TYPE, DP>::chunks];
};
// lane (g, c) of a block whose row c starts at `row`: binary32 takes d = 16 k + 4 g + i, 16-bit d = 32 k + 8 g + i
template <int TYPE, int DP>
__device__ __forceinline__ void frag_from_global(Frag<TYPE, DP> &f, const typename Elem<TYPE>::raw *row, bool live, int D, int g) {
    typedef DirectShape<TYPE, DP> S;
#pragma unroll
    for (int k = 0; k < S::chunks; ++k) {
        const int d = S::wide ? 16 * k + 4 * g : 32 * k + 8 * g;
        f.c[k] = live && d < D ? *reinterpret_cast<const u32x4 *>(row + d) : u32x4{0, 0, 0, 0};
    }
}
template <int TYPE, int DP> __device__ __forceinline__ f32x4 dot_block(const Frag<TYPE, DP> &a, const Frag<TYPE, DP> &b) {
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < DirectShape<TYPE, DP>::chunks; ++k) {
        if constexpr (TYPE == ATTN_F32) {
            const f32x4 x = __builtin_bit_cast(f32x4, a.c[k]), y = __builtin_bit_cast(f32x4, b.c[k]);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], acc, 0, 0, 0);
        } else {
            acc = mfma32<TYPE>(a.c[k], b.c[k], acc);
        }
    }
    return acc;
}

__device__ __forceinline__ int live_length(const StepArgs &a, int b) {
    return max(0, min(a.lengths[b], a.max_pages << a.shift));
}

// one (row, head) key by key: the wave's lanes hold keys for the scores and dimensions for the sum
template <int TYPE> __device__ void careful_step_row(const StepArgs &a, int b, int hk, int m, float top, float total) {
    typedef typename Elem<TYPE>::raw raw;
    const int lane = threadIdx.x & 63, p = m / a.G, h = hk * a.G + m % a.G, n = live_length(a, b);
    const int64_t row = (int64_t)b * a.P + p;
    const ScoreParams sp = score_params(a.scale, a.cap, 0, nullptr, 0);
    const raw *q = reinterpret_cast<const raw *>(a.q) + row * a.qs[0] + h * a.qs[1];
    float acc0 = 0.0f, acc1 = 0.0f;
    for (int base = 0; base < n; base += 64) {
        const int j = base + lane;
        int page = j < n ? a.table[b * a.ts + (j >> a.shift)] : -1;
        bool ok = page >= 0 && page < a.num_pages;
        if (ok && a.blocked != nullptr && (j >> 5) < a.halves) ok = !((a.blocked[row * a.bs + (j >> 5)] >> (j & 31)) & 1);
        float w = 0.0f;
        if (ok) {
            const raw *k = reinterpret_cast<const raw *>(a.k) + page * a.ks[0] + hk * a.ks[1] + (j & ((1 << a.shift) - 1)) * a.ks[2];
            float dot = 0.0f;
            for (int d = 0; d < a.D; ++d) dot = fmaf(elem_to_float<TYPE>(q[d]), elem_to_float<TYPE>(k[d]), dot);
            float th, s = score_of(sp, dot, th);
            if (a.bias == 1) s = fmaf(-a.slope[h] * ATTN_LOG2E, (float)(n - 1 - j), s);
            if (a.bias == 2) {
                const int at = min(j, a.pos_rows - 1);
                const float dx = a.pos_q[2 * row] - a.pos_k[b * a.pks + 2 * (int64_t)at], dy = a.pos_q[2 * row + 1] - a.pos_k[b * a.pks + 2 * (int64_t)at + 1];
                s = fmaf(-a.slope[h] * ATTN_LOG2E, __builtin_amdgcn_sqrtf(fmaf(dx, dx, dy * dy)), s);
            }
            w = __builtin_amdgcn_exp2f(s - top);
        }
        for (unsigned long long bits = __ballot(ok); bits != 0; bits &= bits - 1) {
            const int jj = __ffsll((long long)bits) - 1;
            const float x = __shfl(w, jj);
            const int pg = __shfl(page, jj);
            const raw *v = reinterpret_cast<const raw *>(a.v) + pg * a.vs[0] + hk * a.vs[1] + ((base + jj) & ((1 << a.shift) - 1)) * a.vs[2];
            if (lane < a.D) acc0 = fmaf(x, elem_to_float<TYPE>(v[lane]), acc0);
            if (lane + 64 < a.D) acc1 = fmaf(x, elem_to_float<TYPE>(v[lane + 64]), acc1);
        }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    raw *o = reinterpret_cast<raw *>(a.out) + row * a.os[0] + h * a.os[1];
    for (int half = 0; half < 2; ++half) {
        const int d = lane + 64 * half;
        const float x = (half ? acc1 : acc0) * inv;
        if (d < a.D) {
            if constexpr (TYPE == ATTN_F32) o[d] = x;
            else if constexpr (TYPE == ATTN_F16) o[d] = __builtin_bit_cast(unsigned short, (_Float16)x);
            else o[d] = __builtin_bit_cast(unsigned short, (__bf16)x);
        }
    }
}

template <int TYPE, int DP> struct StepShape {
    typedef DirectShape<TYPE, DP> S;
    static constexpr int vw = S::wide ? (S::dt < 4 ? S::dt : 4) : (S::dt < 8 ? S::dt : 8);   // elements of V a lane reads at once
    static constexpr int vb = S::dt / vw;                                                     // such reads per key
    static constexpr int words = (vw * Elem<TYPE>::bytes + 3) / 4;                            // 32-bit registers of one
};

// keys and values of one tile of 32 keys, as loaded
template <int TYPE, int DP> struct StepTile {
    typedef StepShape<TYPE, DP> V;
    Frag<TYPE, DP> k[2];
    unsigned v[2][4][V::vb][V::words];
    bool live[2];                                // the page of each half tile exists
};

template <int TYPE, int DP>
__device__ __forceinline__ void step_load(StepTile<TYPE, DP> &t, const StepArgs &a, int b, int hk, int base, int n, int g, int c) {
    typedef typename Elem<TYPE>::raw raw;
    typedef StepShape<TYPE, DP> V;
    const int mask = (1 << a.shift) - 1;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int j0 = base + 16 * x;            // 16 keys lie in one page
        int page = j0 < n ? a.table[b * a.ts + (j0 >> a.shift)] : -1;
        page = __builtin_amdgcn_readfirstlane(page);
        t.live[x] = page >= 0 && page < a.num_pages;
        if (!t.live[x]) page = 0;                // (the page exists whatever it holds: its keys are masked)
        const raw *k = reinterpret_cast<const raw *>(a.k) + page * a.ks[0] + hk * a.ks[1] + (j0 & mask) * a.ks[2];
        const raw *v = reinterpret_cast<const raw *>(a.v) + page * a.vs[0] + hk * a.vs[1] + (j0 & mask) * a.vs[2];
        frag_from_global<TYPE, DP>(t.k[x], k + c * a.ks[2], true, a.D, g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const raw *row = v + (4 * g + r) * a.vs[2];
            const bool in = j0 + 4 * g + r < n;  // slots behind the last token may hold anything: they are taken as zero
#pragma unroll
            for (int y = 0; y < V::vb; ++y) {
                const int d = 16 * V::vw * y + V::vw * c;
                const bool get = in && d < a.D;
                if constexpr (V::words == 4) {
                    const u32x4 w = get ? *reinterpret_cast<const u32x4 *>(row + d) : u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int e = 0; e < 4; ++e) t.v[x][r][y][e] = w[e];
                } else if constexpr (V::words == 2) {
                    const u32x2 w = get ? *reinterpret_cast<const u32x2 *>(row + d) : u32x2{0, 0};
                    t.v[x][r][y][0] = w[0];
                    t.v[x][r][y][1] = w[1];
                } else if constexpr (V::vw * Elem<TYPE>::bytes == 4) {
                    t.v[x][r][y][0] = get ? *reinterpret_cast<const unsigned *>(row + d) : 0;
                } else {
                    t.v[x][r][y][0] = get ? (unsigned)*reinterpret_cast<const unsigned short *>(row + d) : 0;
                }
            }
        }
    }
}

// out[n][vw y + i] += V^T P^T of a tile
template <int TYPE, int DP, int NQ>
__device__ __forceinline__ void step_accumulate(f32x4 (&o)[NQ][DP / 16], const StepTile<TYPE, DP> &t, const f32x4 (&p)[2][NQ]) {
    typedef StepShape<TYPE, DP> V;
    if constexpr (TYPE == ATTN_F32) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int y = 0; y < V::vb; ++y)
#pragma unroll
                    for (int i = 0; i < V::vw; ++i)
#pragma unroll
                        for (int n = 0; n < NQ; ++n)
                            o[n][V::vw * y + i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(t.v[x][r][y][i]), p[x][n][r],
                                                                                       o[n][V::vw * y + i], 0, 0, 0);
    } else {
        u32x4 b[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            u32x2 lo, hi;
            if constexpr (TYPE == ATTN_F16) {
                lo = __builtin_bit_cast(u32x2, __builtin_convertvector(p[0][n], f16x4));
                hi = __builtin_bit_cast(u32x2, __builtin_convertvector(p[1][n], f16x4));
            } else {
                lo = __builtin_bit_cast(u32x2, __builtin_convertvector(p[0][n], bf16x4));
                hi = __builtin_bit_cast(u32x2, __builtin_convertvector(p[1][n], bf16x4));
            }
            b[n] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
#pragma unroll
        for (int y = 0; y < V::vb; ++y)
#pragma unroll
            for (int i = 0; i < V::vw; ++i) {
                const unsigned pick = i & 1 ? 0x07060302u : 0x05040100u;
                const int w = i >> 1;
                const u32x4 av = {__builtin_amdgcn_perm(t.v[0][1][y][w], t.v[0][0][y][w], pick),
                                  __builtin_amdgcn_perm(t.v[0][3][y][w], t.v[0][2][y][w], pick),
                                  __builtin_amdgcn_perm(t.v[1][1][y][w], t.v[1][0][y][w], pick),
                                  __builtin_amdgcn_perm(t.v[1][3][y][w], t.v[1][2][y][w], pick)};
#pragma unroll
                for (int n = 0; n < NQ; ++n) o[n][V::vw * y + i] = mfma32<TYPE>(av, b[n], o[n][V::vw * y + i]);
            }
    }
}

template <int TYPE, int DP, int NQ>
__global__ __launch_bounds__(64 * STEP_WAVES) void attn_step_kernel(StepArgs a) {
    typedef typename Elem<TYPE>::raw raw;
    typedef DirectShape<TYPE, DP> S;
    typedef StepShape<TYPE, DP> V;
    constexpr int LD = 16 * S::dt + 4;           // floats of one query's partial result in LDS (sum, maximum, sum of p)
    __shared__ __align__(16) float join[STEP_WAVES / 2][16 * NQ][LD];
    // ranges of one sequence and its chunks of queries follow each other on one XCD: chunks read the same keys
    const int work = (int)(blockIdx.x % 8) * (int)(gridDim.x / 8) + (int)(blockIdx.x / 8);
    if (work >= a.B * a.Hkv * a.splits * a.chunks) return;
    const int chunk = work % a.chunks, split = work / a.chunks % a.splits, bh = work / (a.chunks * a.splits);
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
    // (in a scalar register, so that the pages are looked up by scalar loads: a vector load among the tiles' would be waited for
    // with all the loads before it)
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n_keys = live_length(a, b);
    const int tiles = (n_keys + STEP_TILE - 1) / STEP_TILE, per = (tiles + a.splits - 1) / a.splits;
    const int end = min(tiles, (split + 1) * per);
    const ScoreParams sp = score_params(a.scale, a.cap, 0, nullptr, 0);

    Frag<TYPE, DP> qf[NQ];
    f32x4 o[NQ][S::dt];
    float m[NQ], l[NQ], slope2[NQ], qx[NQ], qy[NQ];
    int64_t mask_row[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int at = (chunk * NQ + n) * 16 + c;
        const bool live = at < a.M;
        const int p = live ? at / a.G : 0, h = hk * a.G + (live ? at % a.G : 0);
        const int64_t row = (int64_t)b * a.P + p;
        frag_from_global<TYPE, DP>(qf[n], reinterpret_cast<const raw *>(a.q) + row * a.qs[0] + h * a.qs[1], live, a.D, g);
        m[n] = -attn_inf();
        l[n] = 0.0f;
        slope2[n] = a.bias ? a.slope[h] * ATTN_LOG2E : 0.0f;
        qx[n] = a.bias == 2 ? a.pos_q[2 * row] : (float)(n_keys - 1);
        qy[n] = a.bias == 2 ? a.pos_q[2 * row + 1] : 0.0f;
        mask_row[n] = row * a.bs;
#pragma unroll
        for (int d = 0; d < S::dt; ++d) o[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    auto compute = [&](const StepTile<TYPE, DP> &t, int tile) {
        const int base = tile * STEP_TILE;
        unsigned bits[NQ];
        if (a.blocked != nullptr) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) bits[n] = tile < a.halves ? a.blocked[mask_row[n] + tile] >> (4 * g) : 0u;
        }
        f32x4 s[2][NQ];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int n = 0; n < NQ; ++n) s[x][n] = dot_block<TYPE, DP>(t.k[x], qf[n]);
        if (sp.cap == CAP_NONE) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int n = 0; n < NQ; ++n) s[x][n] = s[x][n] * sp.mul;
        } else if (sp.cap == CAP_FAST) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[x][n][r] = 2.0f * sp.cap2 * cap_h(s[x][n][r] * sp.mul2);
        } else {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[x][n][r] = sp.cap2 * attn_tanh(s[x][n][r] * sp.mul);
        }
        if (a.bias == 1) {
            const float k0 = (float)(base + 4 * g);
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[x][n][r] = fmaf(-slope2[n], qx[n] - (k0 + (float)(16 * x + r)), s[x][n][r]);
        } else if (a.bias == 2) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = min(base + 16 * x + 4 * g + r, a.pos_rows - 1);
                    const f32x2 at = *reinterpret_cast<const f32x2 *>(a.pos_k + b * a.pks + 2 * (int64_t)j);
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        const float dx = qx[n] - at[0], dy = qy[n] - at[1];
                        s[x][n][r] = fmaf(-slope2[n], __builtin_amdgcn_sqrtf(fmaf(dx, dx, dy * dy)), s[x][n][r]);
                    }
                }
        }
        if (base + STEP_TILE > n_keys || !t.live[0] || !t.live[1]) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        s[x][n][r] = t.live[x] && base + 16 * x + 4 * g + r < n_keys ? s[x][n][r] : -attn_inf();
        }
        if (a.blocked != nullptr) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[x][n][r] = (bits[n] >> (16 * x + r)) & 1 ? -attn_inf() : s[x][n][r];
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float top = fast_max(fast_max(fast_max(s[0][n][0], s[0][n][1]), fast_max(s[0][n][2], s[0][n][3])),
                                 fast_max(fast_max(s[1][n][0], s[1][n][1]), fast_max(s[1][n][2], s[1][n][3])));
            top = fast_max(group_max(top), m[n]);
            const float shift = top == -attn_inf() ? 0.0f : top;
            if (__any(top > m[n])) {
                const float f = __builtin_amdgcn_exp2f(m[n] - shift);
                l[n] *= f;
#pragma unroll
                for (int d = 0; d < S::dt; ++d) o[n][d] = o[n][d] * f;
                m[n] = top;
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[x][n][r] = __builtin_amdgcn_exp2f(s[x][n][r] - shift);
                    l[n] += s[x][n][r];
                }
        }
        step_accumulate<TYPE, DP, NQ>(o, t, s);
    };

    // two tiles in flight, the loads of one issued before the other is computed - where both fit the registers beside the
    // queries and sums (256 at two waves per SIMD); else one, and the other waves' loads cover the wait
    constexpr int tile_regs = 2 * 4 * S::chunks + 8 * V::vb * V::words, held_regs = NQ * (4 * S::chunks + 4 * S::dt + 32);
    if constexpr (2 * tile_regs + held_regs > 240) {
        StepTile<TYPE, DP> t;
        for (int tile = split * per + wave; tile < end; tile += STEP_WAVES) {
            step_load<TYPE, DP>(t, a, b, hk, tile * STEP_TILE, n_keys, g, c);
            compute(t, tile);
        }
    } else {
        StepTile<TYPE, DP> t0, t1;
        int tile = split * per + wave;
        if (tile < end) step_load<TYPE, DP>(t0, a, b, hk, tile * STEP_TILE, n_keys, g, c);
        while (tile < end) {
            const int next = tile + STEP_WAVES;
            if (next < end) step_load<TYPE, DP>(t1, a, b, hk, next * STEP_TILE, n_keys, g, c);
            compute(t0, tile);
            tile = next;
            if (tile >= end) break;
            const int after = tile + STEP_WAVES;
            if (after < end) step_load<TYPE, DP>(t0, a, b, hk, after * STEP_TILE, n_keys, g, c);
            compute(t1, tile);
            tile = after;
        }
    }

#pragma unroll
    for (int n = 0; n < NQ; ++n) l[n] = group_sum(l[n]);
    // the waves' results join in a fixed tree
    for (int half = STEP_WAVES / 2; half > 0; half >>= 1) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                float *to = join[wave - half][16 * n + c];
#pragma unroll
                for (int d = 0; d < S::dt; ++d) *reinterpret_cast<f32x4 *>(to + 16 * d + 4 * g) = o[n][d];
                if (g == 0) *reinterpret_cast<f32x2 *>(to + 16 * S::dt) = f32x2{m[n], l[n]};
            }
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const float *from = join[wave][16 * n + c];
                const f32x2 ml = *reinterpret_cast<const f32x2 *>(from + 16 * S::dt);
                const float top = fmaxf(m[n], ml[0]), shift = top == -attn_inf() ? 0.0f : top;
                const float f = __builtin_amdgcn_exp2f(m[n] - shift), e = __builtin_amdgcn_exp2f(ml[0] - shift);
                l[n] = fmaf(l[n], f, ml[1] * e);
                m[n] = top;
#pragma unroll
                for (int d = 0; d < S::dt; ++d) {
                    const f32x4 x = *reinterpret_cast<const f32x4 *>(from + 16 * d + 4 * g);
                    o[n][d] = o[n][d] * f + x * e;
                }
            }
        }
        __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int at = (chunk * NQ + n) * 16 + c;
        const bool live = at < a.M;
        const int p = at / a.G, h = hk * a.G + at % a.G;
        const int64_t row = (int64_t)b * a.P + p;
        const float shift = m[n] == -attn_inf() ? 0.0f : m[n], inv = l[n] == 0.0f ? 0.0f : 1.0f / l[n];
        if (a.splits > 1) {
            if (live) {
                float *to = a.part + (((int64_t)bh * a.splits + split) * a.M + at) * (a.D + 2);
#pragma unroll
                for (int y = 0; y < V::vb; ++y)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int i = 0; i < V::vw; ++i) {
                            const int d = 16 * V::vw * y + V::vw * (4 * g + r) + i;
                            if (d < a.D) to[d] = o[n][V::vw * y + i][r];
                        }
                if (g == 0) {
                    to[a.D] = m[n];
                    to[a.D + 1] = l[n];
                }
            }
            continue;
        }
        bool fine = true;
#pragma unroll
        for (int d = 0; d < S::dt; ++d) {
            const f32x4 &v = o[n][d];
            fine = fine && (v[0] * 0.0f + v[1] * 0.0f) + (v[2] * 0.0f + v[3] * 0.0f) == 0.0f;
        }
        if (live) {
            raw *to = reinterpret_cast<raw *>(a.out) + row * a.os[0] + h * a.os[1];
#pragma unroll
            for (int y = 0; y < V::vb; ++y)
#pragma unroll
                for (int e = 0; e < V::vw; ++e) {
                    // element 4 e + f of the lane's 4 vw consecutive ones is (r, i) = divmod(4 e + f, vw)
                    const int d = 16 * V::vw * y + 4 * V::vw * g + 4 * e;
                    f32x4 w;
#pragma unroll
                    for (int f = 0; f < 4; ++f) w[f] = o[n][V::vw * y + (4 * e + f) % V::vw][(4 * e + f) / V::vw] * inv;
                    if (d < a.D) store4<TYPE>(to + d, w);
                }
            if (a.lse != nullptr && g == 0)
                a.lse[row * a.Hq + h] = l[n] == 0.0f ? -attn_inf() : (shift + __builtin_amdgcn_logf(l[n])) * ATTN_LN2;
        }
        unsigned long long bad = __ballot(!fine && live);
        bad = (bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffff;
        for (; bad != 0; bad &= bad - 1) {
            const int cc = __ffsll((long long)bad) - 1;
            careful_step_row<TYPE>(a, b, hk, (chunk * NQ + n) * 16 + cc, __shfl(shift, cc), __shfl(l[n], cc));
        }
    }
}

// Joins the ranges of a sequence: one wave per (row, head), lanes over the head size, in the order of the ranges.
template <int TYPE> __global__ __launch_bounds__(256) void attn_step_join_kernel(StepArgs a) {
    typedef typename Elem<TYPE>::raw raw;
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= (int64_t)a.B * a.Hkv * a.M) return;
    const int64_t bh = at / a.M;
    const int m = (int)(at % a.M), b = (int)(bh / a.Hkv), hk = (int)(bh % a.Hkv);
    const float *from = a.part + (bh * a.splits * a.M + m) * (a.D + 2);
    const int64_t stride = (int64_t)a.M * (a.D + 2);
    float top = -attn_inf();
    for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, from[s * stride + a.D]);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float shift = top == -attn_inf() ? 0.0f : top;
    float total = 0.0f, acc0 = 0.0f, acc1 = 0.0f;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {             // (unrolled: the ranges' loads are in flight together)
        const float *x = from + s * stride;
        const float f = __builtin_amdgcn_exp2f(x[a.D] - shift);
        total = fmaf(x[a.D + 1], f, total);
        if (lane < a.D) acc0 = fmaf(x[lane], f, acc0);
        if (lane + 64 < a.D) acc1 = fmaf(x[lane + 64], f, acc1);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int h = hk * a.G + m % a.G;
    const int64_t row = (int64_t)b * a.P + m / a.G;
    raw *o = reinterpret_cast<raw *>(a.out) + row * a.os[0] + h * a.os[1];
    for (int half = 0; half < 2; ++half) {
        const int d = lane + 64 * half;
        const float x = (half ? acc1 : acc0) * inv;
        if (d < a.D) {
            if constexpr (TYPE == ATTN_F32) o[d] = x;
            else if constexpr (TYPE == ATTN_F16) o[d] = __builtin_bit_cast(unsigned short, (_Float16)x);
            else o[d] = __builtin_bit_cast(unsigned short, (__bf16)x);
        }
    }
    if (a.lse != nullptr && lane == 0) a.lse[row * a.Hq + h] = total == 0.0f ? -attn_inf() : (shift + __builtin_amdgcn_logf(total)) * ATTN_LN2;
    if (__any((acc0 + acc1) * 0.0f != 0.0f)) careful_step_row<TYPE>(a, b, hk, m, shift, total);
}

// ------------------------------------------------------------------------------------------------------------ append
struct AppendArgs {
    const char *k_new, *v_new;
    char *k, *v;
    int64_t kn[3], vn[3], ks[3], vs[3], ts;      // new tokens: batch, head, token; pages: page, head, slot (bytes)
    int B, Hkv, T, pieces, shift, max_pages, num_pages, blocks;
    const int *table, *start, *counts;
    int *lengths_out;
};
// The length after an append: the end of its tokens, or the first of them whose page is absent.  (A token that was not stored
// must not count: once the sequence gets the page, whatever lies there would be read as that token.)  Called by whole waves.
__device__ __forceinline__ int end_of_append(const AppendArgs &a, int b, int first, int count) {
    const int64_t capacity = (int64_t)a.max_pages << a.shift, stop = (int64_t)first + count;
    const int lo = max(first, 0), hi = (int)min(stop, capacity);
    const int lane = threadIdx.x & 63;
    for (int p = lo >> a.shift; lo < hi && p <= (hi - 1) >> a.shift; p += 64) {
        const int at = p + lane;
        const int page = at <= (hi - 1) >> a.shift ? a.table[b * a.ts + at] : 0;
        const unsigned long long absent = __ballot(page < 0 || page >= a.num_pages);
        if (absent != 0) return max(lo, (p + __ffsll((long long)absent) - 1) << a.shift);
    }
    return (int)max((int64_t)0, min(stop, capacity));
}
// `blocks` workgroups per sequence copy 16-byte pieces; one workgroup per sequence may also store the new length (it is
// the only one that reads the old one)
__global__ __launch_bounds__(256) void cache_append_kernel(AppendArgs a) {
    const int b = blockIdx.x / a.blocks, part = blockIdx.x % a.blocks;
    const int first = a.start[b];
    const int count = max(0, min(a.counts != nullptr ? a.counts[b] : a.T, a.T));
    const int64_t total = (int64_t)count * a.Hkv * a.pieces;
    const bool store = a.lengths_out != nullptr && a.blocks == 1;
    int end = 0;
    if (store && threadIdx.x < 64) end = end_of_append(a, b, first, count);
    for (int64_t x = (int64_t)part * 256 + threadIdx.x; x < total; x += (int64_t)a.blocks * 256) {
        const int piece = (int)(x % a.pieces), hk = (int)(x / a.pieces % a.Hkv), t = (int)(x / ((int64_t)a.pieces * a.Hkv));
        const int64_t at = (int64_t)first + t;
        if (at < 0 || at >= (int64_t)a.max_pages << a.shift) continue;
        const int page = a.table[b * a.ts + (at >> a.shift)];
        if (page < 0 || page >= a.num_pages) continue;
        const int64_t slot = at & ((1 << a.shift) - 1);
        *reinterpret_cast<u32x4 *>(a.k + page * a.ks[0] + hk * a.ks[1] + slot * a.ks[2] + 16 * piece) =
            *reinterpret_cast<const u32x4 *>(a.k_new + b * a.kn[0] + hk * a.kn[1] + t * a.kn[2] + 16 * piece);
        *reinterpret_cast<u32x4 *>(a.v + page * a.vs[0] + hk * a.vs[1] + slot * a.vs[2] + 16 * piece) =
            *reinterpret_cast<const u32x4 *>(a.v_new + b * a.vn[0] + hk * a.vn[1] + t * a.vn[2] + 16 * piece);
    }
    if (store) {
        __syncthreads();                         // every thread has read the old length
        if (threadIdx.x == 0) a.lengths_out[b] = end;
    }
}
__global__ __launch_bounds__(256) void cache_lengths_kernel(AppendArgs a) {      // one wave per sequence
    const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= a.B) return;
    const int count = max(0, min(a.counts != nullptr ? a.counts[b] : a.T, a.T));
    const int end = end_of_append(a, b, a.start[b], count);
    if ((threadIdx.x & 63) == 0) a.lengths_out[b] = end;
}

// ------------------------------------------------------------------------------------------------------------ launch
bool aligned16(const int64_t *s, int n, const void *p, int bytes) {
    if ((reinterpret_cast<uintptr_t>(p) & 15) != 0) return false;
    for (int i = 0; i < n; ++i)
        if ((s[i] * bytes) % 16 != 0 || s[i] < 0) return false;
    return true;
}
int log2_of(int x) {
    int s = 0;
    while ((1 << s) < x) ++s;
    return s;
}

int check_cache(const dgl_kv_cache_t *c) {
    DGL_CHECK_ARG(c != nullptr, "NULL argument");
    DGL_CHECK_ARG(c->dtype >= DGL_DTYPE_F32 && c->dtype <= DGL_DTYPE_BF16, "unknown element type %d", c->dtype);
    DGL_CHECK_ARG(c->B >= 1 && c->Hkv >= 1, "B=%d Hkv=%d", c->B, c->Hkv);
    DGL_CHECK_ARG(c->D >= 8 && c->D <= 128 && c->D % 8 == 0, "head size %d (a multiple of 8, at most 128)", c->D);
    DGL_CHECK_ARG(c->page_size >= 16 && c->page_size <= (1 << 20) && (c->page_size & (c->page_size - 1)) == 0,
                  "page size %d (a power of two from 16 on)", c->page_size);
    DGL_CHECK_ARG(c->num_pages >= 1 && c->max_pages >= 1 && (int64_t)c->max_pages * c->page_size <= DGL_CACHE_MAX_TOKENS,
                  "%d pages, %d per sequence of %d tokens", c->num_pages, c->max_pages, c->page_size);
    DGL_CHECK_ARG(c->k_pages != nullptr && c->v_pages != nullptr && c->table != nullptr && c->lengths != nullptr, "NULL in the cache");
    DGL_CHECK_ARG(c->table_stride >= 0, "table stride %lld", (long long)c->table_stride);
    const int bytes = c->dtype == DGL_DTYPE_F32 ? 4 : 2;
    DGL_CHECK_ARG(aligned16(c->k_stride, 3, c->k_pages, bytes) && aligned16(c->v_stride, 3, c->v_pages, bytes),
                  "pages: 16-byte aligned pointers and strides");
    return DGL_OK;
}
int check_step(const dgl_attention_step_t *p) {
    DGL_CHECK_ARG(p != nullptr, "NULL argument");
    if (int e = check_cache(&p->cache)) return e;
    DGL_CHECK_ARG(p->rows_per_instance >= 1 && p->Hq >= 1 && p->Hq % p->cache.Hkv == 0, "rows %d, %d query heads over %d key heads",
                  p->rows_per_instance, p->Hq, p->cache.Hkv);
    DGL_CHECK_ARG(score_params_fit(p->scale, p->cap), "scale %g, cap %g", (double)p->scale, (double)p->cap);
    DGL_CHECK_ARG(p->q != nullptr && p->out != nullptr, "q or out is NULL");
    DGL_CHECK_ARG((p->pos_q == nullptr) == (p->pos_k == nullptr), "coordinates of one side only");
    DGL_CHECK_ARG(p->pos_q == nullptr || (p->slope != nullptr && p->pos_rows >= 1), "coordinates without a slope or without rows");
    DGL_CHECK_ARG(p->pos_q == nullptr || ((reinterpret_cast<uintptr_t>(p->pos_k) & 7) == 0 && p->pos_k_stride % 2 == 0),
                  "coordinates: 8-byte aligned");
    DGL_CHECK_ARG(p->blocked == nullptr || (p->words >= 0 && p->blocked_stride >= 0), "words %d", p->words);
    const int bytes = p->cache.dtype == DGL_DTYPE_F32 ? 4 : 2;
    DGL_CHECK_ARG(aligned16(p->q_stride, 2, p->q, bytes) && aligned16(p->o_stride, 2, p->out, bytes), "q, out: 16-byte aligned pointers and strides");
    const int64_t queries = (int64_t)p->cache.B * p->rows_per_instance * p->Hq;
    DGL_CHECK_ARG(queries < (1ll << 29) && (int64_t)p->rows_per_instance * p->Hq < (1ll << 26), "too many rows");
    return DGL_OK;
}

int padded_size(int D) { return D <= 16 ? 16 : D <= 32 ? 32 : D <= 64 ? 64 : 128; }

struct StepPlan {
    int nq, chunks, splits;
};
// the most blocks of 16 queries whose operands and sums fit a wave's registers
constexpr int most_blocks(int dtype, int DP) { return DP <= 32 ? 4 : DP == 128 && dtype == ATTN_F32 ? 1 : 2; }
// Queries of one key head are taken 16 NQ at a time (two blocks per wave from 17 queries on, four for small heads from 33
// on: the cache is read once per chunk).  A sequence is cut so that the workgroups cover the 256 compute units twice, but
// a range keeps at least four tiles for each of its 8 waves - below that the second launch costs more than it brings.
StepPlan step_plan(const dgl_attention_step_t *p) {
    StepPlan s;
    const int M = p->rows_per_instance * (p->Hq / p->cache.Hkv), DP = padded_size(p->cache.D);
    const int wanted = M <= 16 ? 1 : M <= 32 ? 2 : 4, most_nq = most_blocks(p->cache.dtype, DP);
    s.nq = wanted < most_nq ? wanted : most_nq;
    s.chunks = (M + 16 * s.nq - 1) / (16 * s.nq);
    const int64_t units = (int64_t)p->cache.B * p->cache.Hkv * s.chunks;
    const int64_t tiles = ((int64_t)p->cache.max_pages * p->cache.page_size + STEP_TILE - 1) / STEP_TILE;
    int64_t want = units >= 512 ? 1 : (512 + units - 1) / units;
    const int64_t most = tiles / (4 * STEP_WAVES);
    if (want > most) want = most;
    s.splits = want < 1 ? 1 : want > 256 ? 256 : (int)want;
    return s;
}

template <int T, int DP, int NQ = most_blocks(T, DP)> void launch_blocks(const StepArgs &a, int nq, hipStream_t s) {
    if constexpr (NQ > 1)
        if (nq < NQ) return launch_blocks<T, DP, NQ / 2>(a, nq, s);
    const int64_t work = (int64_t)a.B * a.Hkv * a.splits * a.chunks;
    hipLaunchKernelGGL((attn_step_kernel<T, DP, NQ>), dim3((unsigned)((work + 7) / 8 * 8)), dim3(64 * STEP_WAVES), 0, s, a);
}
template <int T, int DP> int launch_step(const StepArgs &a, int nq, hipStream_t s) {
    launch_blocks<T, DP>(a, nq, s);
    DGL_CHECK_LAUNCH("dgl_attention_step");
    if (a.splits > 1) {
        const int64_t rows = (int64_t)a.B * a.Hkv * a.M;
        hipLaunchKernelGGL((attn_step_join_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
        DGL_CHECK_LAUNCH("dgl_attention_step (join)");
    }
    return DGL_OK;
}

}  // namespace

extern "C" int64_t dgl_attention_step_workspace_floats(const dgl_attention_step_t *p) {
    if (check_step(p) != DGL_OK) return -1;
    const StepPlan s = step_plan(p);
    if (s.splits == 1) return 0;
    return (int64_t)p->cache.B * s.splits * p->rows_per_instance * p->Hq * (p->cache.D + 2);
}

extern "C" int dgl_attention_step(const dgl_attention_step_t *p, float *ws, dgl_stream_t stream) {
    if (int e = check_step(p)) return e;
    const StepPlan plan = step_plan(p);
    DGL_CHECK_ARG(plan.splits == 1 || ws != nullptr, "a workspace is needed");
    const dgl_kv_cache_t &c = p->cache;
    StepArgs a{};
    a.q = (const char *)p->q; a.k = (const char *)c.k_pages; a.v = (const char *)c.v_pages; a.out = (char *)p->out; a.lse = p->lse;
    for (int i = 0; i < 2; ++i) { a.qs[i] = p->q_stride[i]; a.os[i] = p->o_stride[i]; }
    for (int i = 0; i < 3; ++i) { a.ks[i] = c.k_stride[i]; a.vs[i] = c.v_stride[i]; }
    a.B = c.B; a.P = p->rows_per_instance; a.Hq = p->Hq; a.Hkv = c.Hkv; a.G = p->Hq / c.Hkv; a.D = c.D; a.M = a.P * a.G;
    a.chunks = plan.chunks; a.splits = plan.splits; a.shift = log2_of(c.page_size); a.max_pages = c.max_pages; a.num_pages = c.num_pages;
    a.bias = p->slope == nullptr ? 0 : p->pos_q == nullptr ? 1 : 2;
    a.scale = p->scale; a.cap = p->cap; a.table = c.table; a.lengths = c.lengths; a.ts = c.table_stride;
    a.slope = p->slope; a.pos_q = p->pos_q; a.pos_k = p->pos_k; a.pos_rows = p->pos_rows; a.pks = p->pos_k_stride;
    a.blocked = (const unsigned *)p->blocked; a.halves = 2 * p->words; a.bs = 2 * p->blocked_stride; a.part = ws;
    hipStream_t s = (hipStream_t)stream;
#define STEP_CASE(T, DPV) \
    if (c.dtype == T && padded_size(c.D) == DPV) return launch_step<T, DPV>(a, plan.nq, s);
    STEP_CASE(ATTN_F32, 16) STEP_CASE(ATTN_F32, 32) STEP_CASE(ATTN_F32, 64) STEP_CASE(ATTN_F32, 128)
    STEP_CASE(ATTN_F16, 16) STEP_CASE(ATTN_F16, 32) STEP_CASE(ATTN_F16, 64) STEP_CASE(ATTN_F16, 128)
    STEP_CASE(ATTN_BF16, 16) STEP_CASE(ATTN_BF16, 32) STEP_CASE(ATTN_BF16, 64) STEP_CASE(ATTN_BF16, 128)
#undef STEP_CASE
    return dgl_set_error(DGL_ERR_INVALID_ARGUMENT, "unknown element type %d", c.dtype);
}

extern "C" int dgl_cache_append(const dgl_kv_cache_t *c, const void *k_new, const void *v_new, const int64_t *k_new_stride,
                                const int64_t *v_new_stride, int32_t T, const int32_t *start, const int32_t *counts,
                                int32_t *lengths_out, dgl_stream_t stream) {
    if (int e = check_cache(c)) return e;
    DGL_CHECK_ARG(T >= 0 && T <= DGL_CACHE_MAX_TOKENS, "T=%d", T);
    if (T == 0 && lengths_out == nullptr) return DGL_OK;
    const int bytes = c->dtype == DGL_DTYPE_F32 ? 4 : 2;
    DGL_CHECK_ARG(start != nullptr && k_new_stride != nullptr && v_new_stride != nullptr && (T == 0 || (k_new != nullptr && v_new != nullptr)), "NULL argument");
    DGL_CHECK_ARG(aligned16(k_new_stride, 3, k_new, bytes) && aligned16(v_new_stride, 3, v_new, bytes), "new tokens: 16-byte aligned pointers and strides");
    AppendArgs a{};
    a.k_new = (const char *)k_new; a.v_new = (const char *)v_new; a.k = (char *)c->k_pages; a.v = (char *)c->v_pages;
    for (int i = 0; i < 3; ++i) {
        a.kn[i] = k_new_stride[i] * bytes; a.vn[i] = v_new_stride[i] * bytes;
        a.ks[i] = c->k_stride[i] * bytes; a.vs[i] = c->v_stride[i] * bytes;
    }
    a.ts = c->table_stride; a.B = c->B; a.Hkv = c->Hkv; a.T = T; a.pieces = c->D * bytes / 16; a.shift = log2_of(c->page_size);
    a.max_pages = c->max_pages; a.num_pages = c->num_pages; a.table = c->table; a.start = start; a.counts = counts;
    a.lengths_out = lengths_out;
    // one workgroup per sequence up to 8 pieces a thread, then as many as that takes
    const int64_t pieces = (int64_t)T * a.Hkv * a.pieces, blocks = (pieces + 2047) / 2048;
    a.blocks = blocks < 1 ? 1 : blocks > 4096 ? 4096 : (int)blocks;
    DGL_CHECK_ARG((int64_t)a.B * a.blocks < (1ll << 31), "too many sequences");
    hipLaunchKernelGGL(cache_append_kernel, dim3((unsigned)(a.B * a.blocks)), dim3(256), 0, (hipStream_t)stream, a);
    DGL_CHECK_LAUNCH("dgl_cache_append");
    if (lengths_out != nullptr && a.blocks > 1) {
        hipLaunchKernelGGL(cache_lengths_kernel, dim3((a.B + 3) / 4), dim3(256), 0, (hipStream_t)stream, a);
        DGL_CHECK_LAUNCH("dgl_cache_append (lengths)");
    }
    return DGL_OK;
}
