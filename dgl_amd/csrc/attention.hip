// Attention over nodes or sequence positions, forward and backward.
//
//   s_ij = cap tanh(scale q_i . k_j / cap) - slope_h dist(i, j)          (cap = 0: no tanh; slope = NULL: no bias)
//   p_ij = softmax over the allowed j;   o_i = sum_j p_ij v_j;   lse_i = log sum_j exp(s_ij)
//   dp = do v^T;  ds = p (dp - do . o);  dslope = - sum ds dist;  du = ds (1 - tanh^2);
//   dq = scale du k;  dk = scale du^T q;  dv = p^T do
//
// dist is the Euclidean distance of 2-D coordinates, or |i + Lk - Lq - j|; a pair is allowed when both sides carry the same
// document id >= 0 and, under `causal`, j <= i + Lk - Lq or j < prefix.  A row without an allowed pair gives zeros.
//
// One pass over the keys with a running maximum and sum (scores never leave registers); the backward pass recomputes the
// scores from lse in two kernels - one owns query rows (dq, delta, dslope), one owns key rows (dk, dv, summed over the
// query heads that share them) - so no gradient needs atomics and every call gives the same bits.
//
// A pair that is masked contributes nothing, whatever its operands hold: the products of the matrix instructions would
// carry a NaN or infinity of a masked row into its tile neighbours (0 * NaN), so a result that is not finite at the end is
// recomputed pair by pair (careful_*), which costs nothing where all is finite.
//
// Bound by vector instructions, not by memory (a head's keys are read by all its row blocks from L2): a pair of
// a forward pass takes 18 simple operations and 4 of exp / rcp / sqrt with a cap and coordinates in binary32 (a third of the
// simple ones split probabilities into terms), 7 and 3 with a cap in 16 bits, and the 16-bit matrix instructions hold the
// vector unit back for two thirds of their 17 cycles.  Their issue fills the binary32 forward pass (vector unit busy 1.00 of its
// cycles).  Heads of 128 leave both units free (vector 0.57, matrix 0.26): two waves a SIMD wait for each other's results a third of
// the time.  The backward kernels and documents have 1.2-1.9 waves a SIMD on average, their blocks being uneven (vector 0.25-0.6,
// matrix 0.09-0.15).  Measured, per launch:
//   forward, 64 x 8 heads of 16, 1000 nodes, cap and coordinates, binary32                431 us  76 TFLOP/s
//   forward, 32 heads over 8 of 128, 8192 causal rows, cap, bf16                           860 us  640 TFLOP/s
//   2 x 16 heads over 4 of 64, 2047 causal rows behind a prefix, slopes, bf16     forward 71, rows 86, keys 111 + 13 us
//   8 heads of 64, 6000 rows in 9 documents, fp16                                 forward 88, rows 117, keys 162 us
//   8 x 8 heads of 16, 1001 rows in 4 documents, cap and coordinates, binary32    forward 89, rows 114, keys 120 us
#include "attention_tile.h"

#include <cfloat>

namespace {

#define ATTN_THREADS 256
#define ATTN_MAX_TILES 4096      // tiles whose document overlap is looked up before the pass; later ones are all visited

struct AttnArgs {
    const char *q, *k, *v;                       // element pointers
    char *out;
    char *rest;                                  // what out's rounding left off (out's strides), or nullptr
    float *lse;
    int64_t qs[3], ks[3], vs[3], os[3];          // strides: batch, head, token (elements)
    int B, Hq, Hkv, G, Lq, Lk, D, causal, bias;  // bias: 0 none, 1 positions, 2 coordinates
    float scale, cap;
    const float *slope, *pos_q, *pos_k;
    int64_t pqs, pks;
    const int *doc_q, *doc_k;
    int64_t dqs, dks;
    const int *prefix;
    int tiles;                                   // row blocks per (batch, head)
    int splits;                                  // forward: ranges of keys per row block; backward: ranges of rows per key block
    float *part;                                 // results of the ranges
    // backward
    const char *dout;
    char *dq, *dk, *dv;
    int64_t dos[3], dqst[3], dkst[3], dvst[3];
    float *delta, *rowscale, *dslope_part, *dslope;
    int *many;                                   // per row: all ones, or 0 where it sees a single key
    int head_parts;                              // key kernel: parts of the heads that share a key head
};

// Blocks are dealt to the 8 XCDs in turn; giving every XCD a contiguous range of the work keeps the row blocks of one
// head, which read the same keys and values, on one L2.
__device__ __forceinline__ int xcd_work() { return (int)(blockIdx.x % 8) * (int)(gridDim.x / 8) + (int)(blockIdx.x / 8); }

// The workgroup's unit (a head, or a part of one) and the rank of its block among the unit's `tiles`, longest first.  Blocks of
// a causal call differ in length: there the longest blocks of all the heads of an XCD start before any shorter one, or the last
// head's long blocks would run on a chip that is otherwise idle (32 heads of 128, 8192 rows: 883 -> 856 us; 2 x 16 heads of 64, 2047
// rows: forward 78 -> 72, query rows' gradients 96 -> 86.  The keys' gradients, cut finer, gain nothing and keep their order).
struct Work {
    int unit, rank;                              // rank >= tiles: nothing to do
};
__device__ __forceinline__ Work deal(bool uneven, int units, int tiles) {
    const int i = blockIdx.x;
    if (!uneven) {
        const int work = xcd_work();
        return {work / tiles, work < units * tiles ? work % tiles : tiles};
    }
    if (units % 8 != 0) return {i % units, i / units};
    const int per = units / 8, l = i / 8;
    return {i % 8 * per + l % per, l / per};
}

// keys a query row sees: j < limit (and the document test)
__device__ __forceinline__ int row_limit(const AttnArgs &a, int b, int i) {
    if (i >= a.Lq) return 0;
    if (!a.causal) return a.Lk;
    int lim = i + a.Lk - a.Lq + 1;
    if (a.prefix != nullptr) lim = max(lim, a.prefix[b]);
    return max(0, min(lim, a.Lk));
}
// document ids with the padding of either side made unequal to everything
__device__ __forceinline__ int doc_of_query(const AttnArgs &a, int b, int i) {
    const int id = i < a.Lq ? a.doc_q[b * a.dqs + i] : -1;
    return id < 0 ? -2 : id;
}
__device__ __forceinline__ int doc_of_key(const AttnArgs &a, int b, int j) {
    const int id = j < a.Lk ? a.doc_k[b * a.dks + j] : -1;
    return id < 0 ? -1 : id;
}

__device__ __forceinline__ float pair_distance(const AttnArgs &a, int b, int i, int j) {
    if (a.bias == 1) return fabsf((float)(i + a.Lk - a.Lq - j));
    const float *x = a.pos_q + b * a.pqs + 2 * (int64_t)i, *y = a.pos_k + b * a.pks + 2 * (int64_t)j;
    const float dx = x[0] - y[0], dy = x[1] - y[1];
    return __builtin_amdgcn_sqrtf(fmaf(dx, dx, dy * dy));
}

// one pair for the careful path: its score (log2 units) and tanh
template <int TYPE>
__device__ float pair_score(const AttnArgs &a, const ScoreParams &sp, int b, int i, int j, const typename Elem<TYPE>::raw *q,
                            const typename Elem<TYPE>::raw *k, float &th) {
    float dot = 0.0f;
    for (int d = 0; d < a.D; ++d) dot = fmaf(elem_to_float<TYPE>(q[d]), elem_to_float<TYPE>(k[d]), dot);
    const float s = score_of(sp, dot, th);
    return sp.bias ? fmaf(-sp.slope2, pair_distance(a, b, i, j), s) : s;
}
__device__ __forceinline__ bool pair_allowed(const AttnArgs &a, int b, int i, int j, int limit) {
    if (j >= limit) return false;
    return a.doc_q == nullptr || doc_of_query(a, b, i) == doc_of_key(a, b, j);
}

// Which 64-row tiles of the other side hold a document of this block's rows: bit set = visit; second word = every pair
// of the tile is in one document (no test per pair).
struct TileMap {
    unsigned long long any[ATTN_MAX_TILES / 64], same[ATTN_MAX_TILES / 64];
    int lo, hi, uniform;
};
__device__ void build_tile_map(TileMap &m, const int *own, int own_base, int own_rows, int own_n, const int *other, int other_n) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid == 0) {
        m.lo = INT_MAX;
        m.hi = -1;
        m.uniform = 1;
    }
    for (int w = tid; w < ATTN_MAX_TILES / 64; w += ATTN_THREADS) m.any[w] = m.same[w] = 0;
    __syncthreads();
    for (int i = tid; i < own_rows; i += ATTN_THREADS) {
        if (own_base + i >= own_n) break;
        const int id = own[own_base + i];
        if (id >= 0) {
            atomicMin(&m.lo, id);
            atomicMax(&m.hi, id);
        } else {
            m.uniform = 0;
        }
    }
    __syncthreads();
    const int lo = m.lo, hi = m.hi;
    const bool one = m.uniform && lo == hi;
    const int tiles = min(ATTN_MAX_TILES, (other_n + ATTN_ROWS - 1) / ATTN_ROWS);
    for (int t = wave; t < tiles; t += ATTN_THREADS / 64) {
        const int j = t * ATTN_ROWS + lane;
        const int id = j < other_n ? other[j] : -1;
        const unsigned long long in = __ballot(id >= 0 && id >= lo && id <= hi), eq = __ballot(id == lo);
        if (lane == 0 && in != 0) {
            atomicOr(&m.any[t / 64], 1ull << (t % 64));
            if (one && eq == ~0ull) atomicOr(&m.same[t / 64], 1ull << (t % 64));
        }
    }
    __syncthreads();
}
// first tile >= t to visit, or `end`
__device__ __forceinline__ int next_tile(const TileMap *m, int t, int end) {
    if (m == nullptr) return t;
    while (t < end && t < ATTN_MAX_TILES) {
        const unsigned long long w = m->any[t / 64] >> (t % 64);
        if (w != 0) return min(end, t + __ffsll((long long)w) - 1);
        t = (t / 64 + 1) * 64;
    }
    return min(t, end);
}
__device__ __forceinline__ bool tile_same(const TileMap *m, int t) {
    return m == nullptr || (t < ATTN_MAX_TILES && ((m->same[t / 64] >> (t % 64)) & 1));
}

__device__ __forceinline__ bool finite4(const f32x4 &v) {
    const float t = (v[0] * 0.0f + v[1] * 0.0f) + (v[2] * 0.0f + v[3] * 0.0f);
    return t == 0.0f;
}

// --------------------------------------------------------------------------------------------------------- forward
// One workgroup = 4 waves x NQ blocks of 16 queries of one (batch, head); keys and values pass through LDS in tiles of 64,
// the next tile's loads in flight while the current one is computed.  Lane (g, c) holds query c of its blocks and, per
// 16 keys, the scores against keys 4 g + r.
//
// The running maximum follows the scores only when one rises 2^SOFTMAX_RISE above it: sums and probabilities are binary32,
// or have room for 2^8 in 16 bits, and a row's sums are rescaled a few times instead of at every new maximum.  Scores come
// out of the cap (or the scaling) relative to it, which saves the subtraction.
#define SOFTMAX_RISE 8.0f
template <int TYPE> __device__ __forceinline__ void store_wide(typename Elem<TYPE>::raw *o, int d, float x) {
    if constexpr (TYPE == ATTN_F32) o[d] = x;
    else if constexpr (TYPE == ATTN_F16) o[d] = __builtin_bit_cast(unsigned short, (_Float16)x);
    else o[d] = __builtin_bit_cast(unsigned short, (__bf16)x);
}
// An output value and, where a backward pass is to come, what its rounding to 16 bits left off: dout . (out + rest) is the
// delta that the unrounded output would give.  (With bfloat16 outputs alone the error of delta was as large as that of the
// rounded score gradients where few keys carry a row: dq of 16 heads, 2047 causal rows with slopes, 0.0027 relative, now 0.0024.)
template <int TYPE> __device__ __forceinline__ void store_out(const AttnArgs &a, int64_t at, float x) {
    typedef typename Elem<TYPE>::raw raw;
    raw *o = reinterpret_cast<raw *>(a.out) + at;
    store_wide<TYPE>(o, 0, x);
    if constexpr (TYPE != ATTN_F32)
        if (a.rest != nullptr) store_wide<TYPE>(reinterpret_cast<raw *>(a.rest) + at, 0, x - elem_to_float<TYPE>(*o));
}
template <int TYPE> __device__ __forceinline__ void store_out4(const AttnArgs &a, int64_t at, f32x4 x) {
    typedef typename Elem<TYPE>::raw raw;
    store4<TYPE>(reinterpret_cast<raw *>(a.out) + at, x);
    if constexpr (TYPE != ATTN_F32)
        if (a.rest != nullptr) store4<TYPE>(reinterpret_cast<raw *>(a.rest) + at, x - rounded4<TYPE>(x));
}
template <int TYPE> __device__ void careful_forward_row(const AttnArgs &a, const ScoreParams &sp, int b, int h, int i) {
    typedef typename Elem<TYPE>::raw raw;
    const int lane = threadIdx.x & 63, hk = h / a.G, limit = row_limit(a, b, i);
    const raw *q = reinterpret_cast<const raw *>(a.q) + b * a.qs[0] + h * a.qs[1] + i * a.qs[2];
    const raw *k = reinterpret_cast<const raw *>(a.k) + b * a.ks[0] + hk * a.ks[1];
    const raw *v = reinterpret_cast<const raw *>(a.v) + b * a.vs[0] + hk * a.vs[1];
    float m = -attn_inf(), l = 0.0f, acc0 = 0.0f, acc1 = 0.0f, th;
    for (int j = lane; j < limit; j += 64)
        if (pair_allowed(a, b, i, j, limit)) m = fmaxf(m, pair_score<TYPE>(a, sp, b, i, j, q, k + j * a.ks[2], th));
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    if (m == -attn_inf()) m = 0.0f;
    for (int base = 0; base < limit; base += 64) {
        const int j = base + lane;
        const bool ok = pair_allowed(a, b, i, j, limit);
        float p = 0.0f;
        if (ok) p = __builtin_amdgcn_exp2f(pair_score<TYPE>(a, sp, b, i, j, q, k + j * a.ks[2], th) - m);
        l += p;
        for (unsigned long long w = __ballot(ok); w != 0; w &= w - 1) {
            const int jj = __ffsll((long long)w) - 1;
            const float pj = __shfl(p, jj);
            const raw *vr = v + (int64_t)(base + jj) * a.vs[2];
            if (lane < a.D) acc0 = fmaf(pj, elem_to_float<TYPE>(vr[lane]), acc0);
            if (lane + 64 < a.D) acc1 = fmaf(pj, elem_to_float<TYPE>(vr[lane + 64]), acc1);
        }
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) l += __shfl_xor(l, x);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t o = b * a.os[0] + h * a.os[1] + i * a.os[2] + lane;
    if (lane < a.D) store_out<TYPE>(a, o, acc0 * inv);
    if (lane + 64 < a.D) store_out<TYPE>(a, o + 64, acc1 * inv);
    if (a.lse != nullptr && lane == 0)
        a.lse[((int64_t)b * a.Hq + h) * a.Lq + i] = l == 0.0f ? -attn_inf() : (m + __builtin_amdgcn_logf(l)) * ATTN_LN2;
}

template <int TYPE, int DP, int NQ>
__global__ __launch_bounds__(ATTN_THREADS, TYPE == ATTN_F32 && DP == 128 ? 1 : 2) void attn_fwd_kernel(AttnArgs a) {
    typedef Shape<TYPE, DP> S;
    typedef typename Elem<TYPE>::raw raw;
    // KB: blocks of 16 keys whose scores are held at once.  Two where that fits another wave on a SIMD: heads of 128 (256
    // registers for two waves) and binary32 heads of 16 (168 for three: 14 % less for nodes of 1000)
    constexpr int ROWS = 64 * NQ, KB = DP == 128 || (TYPE == ATTN_F32 && DP <= 32) ? 2 : 4;
    __shared__ __align__(16) char Kt[S::bytes], Vt[S::bytes];
    __shared__ __align__(16) float key_pos[2 * ATTN_ROWS];
    __shared__ __align__(16) int key_doc[ATTN_ROWS];
    __shared__ TileMap map_store;
    const Work work = deal(a.causal, a.B * a.Hq * a.splits, a.tiles);
    if (work.rank >= a.tiles) return;
    const int split = work.unit % a.splits, bh = work.unit / a.splits, qt = a.tiles - 1 - work.rank;      // (the last rows see most)
    const int b = bh / a.Hq, h = bh % a.Hq, hk = h / a.G;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
    const int row0 = qt * ROWS, wrow0 = row0 + wave * 16 * NQ;
    const raw *q = reinterpret_cast<const raw *>(a.q) + b * a.qs[0] + h * a.qs[1];
    const char *k = a.k + (b * a.ks[0] + hk * a.ks[1]) * Elem<TYPE>::bytes;
    const char *v = a.v + (b * a.vs[0] + hk * a.vs[1]) * Elem<TYPE>::bytes;
    const int *docs = a.doc_k != nullptr ? a.doc_k + b * a.dks : nullptr;
    const ScoreParams sp = score_params(a.scale, a.cap, a.bias, a.slope, h);

    TileMap *map = nullptr;
    if (docs != nullptr) {
        map = &map_store;
        build_tile_map(map_store, a.doc_q + b * a.dqs, row0, ROWS, a.Lq, docs, a.Lk);
    }
    
    ColFrag<TYPE, DP> qf[NQ];
    f32x4 o[NQ][S::dt];
    float w[NQ], rise[NQ], l[NQ], qx[NQ], qy[NQ];     // what scores are taken relative to, and how far above it they may be
    int limit[NQ], doc[NQ];
    int wave_limit = 0, wave_full = INT_MAX;          // keys some row / every row of the wave sees
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int i = wrow0 + 16 * n + c;
        Eight<TYPE> q8[S::chunks];
#pragma unroll
        for (int k8 = 0; k8 < S::chunks; ++k8) q8[k8] = load_eight<TYPE>(q + (int64_t)i * a.qs[2], frag_d<DP>(k8, g), i < a.Lq && frag_d<DP>(k8, g) < a.D);
        col_frag<TYPE, DP>(qf[n], q8, g, score_factor(sp));
        w[n] = 0.0f;
        rise[n] = -attn_inf();
        l[n] = 0.0f;
        limit[n] = row_limit(a, b, i);
        doc[n] = map != nullptr ? doc_of_query(a, b, i) : 0;
        qx[n] = qy[n] = 0.0f;
        if (a.bias == 1) qx[n] = (float)(i + a.Lk - a.Lq);
        if (a.bias == 2 && i < a.Lq) {
            qx[n] = a.pos_q[b * a.pqs + 2 * (int64_t)i];
            qy[n] = a.pos_q[b * a.pqs + 2 * (int64_t)i + 1];
        }
#pragma unroll
        for (int d = 0; d < S::dt; ++d) o[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if (wrow0 < a.Lq) {
        wave_limit = row_limit(a, b, min(wrow0 + 16 * NQ, a.Lq) - 1);        // limits rise with the row
        wave_full = row_limit(a, b, wrow0);
    }
    const int tiles = (row_limit(a, b, min(row0 + ROWS, a.Lq) - 1) + ATTN_ROWS - 1) / ATTN_ROWS;
    const int per = (tiles + a.splits - 1) / a.splits, end = min(tiles, (split + 1) * per);

    Stager<TYPE, DP> stage;
    stage.init(a.ks[2], a.vs[2], a.D);
    float stage_pos = 0.0f;
    int stage_doc = -1;
    auto load = [&](int tile) {
        const int base = tile * ATTN_ROWS, left = a.Lk - base;
        const char *kt = k + base * a.ks[2] * Elem<TYPE>::bytes, *vt = v + base * a.vs[2] * Elem<TYPE>::bytes;
        stage.load(kt, vt, left, map != nullptr ? docs + base : nullptr);
        if (a.bias == 2 && tid < 2 * ATTN_ROWS) stage_pos = tid < 2 * left ? a.pos_k[b * a.pks + 2 * (int64_t)base + tid] : 0.0f;
        if (map != nullptr && tid < ATTN_ROWS) stage_doc = doc_of_key(a, b, base + tid);
    };
    int tile = next_tile(map, split * per, end);
    if (tile < end) load(tile);
    while (tile < end) {
        __syncthreads();
        stage.write(Kt, Vt, map != nullptr);
        if (a.bias == 2 && tid < 2 * ATTN_ROWS) key_pos[tid] = stage_pos;
        if (map != nullptr && tid < ATTN_ROWS) key_doc[tid] = stage_doc;
        const int here = tile, base = here * ATTN_ROWS;
        tile = next_tile(map, here + 1, end);
        if (tile < end) load(tile);
        __syncthreads();
        if (base >= wave_limit) continue;
        const bool by_doc = !tile_same(map, here), by_limit = base + ATTN_ROWS > wave_full;

#pragma unroll
        for (int kb = 0; kb < 4; kb += KB) {
            f32x4 s[KB][NQ];
#pragma unroll
            for (int t = 0; t < KB; ++t) {
                RowFrag<TYPE, DP> kf;
                row_frag<TYPE, DP>(kf, Kt, 16 * (kb + t) + c, g);
#pragma unroll
                for (int n = 0; n < NQ; ++n) s[t][n] = dot_block<TYPE, DP>(kf, qf[n]);
            }
            if (sp.cap == CAP_NONE) {
#pragma unroll
                for (int t = 0; t < KB; ++t)
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][n][r] = TYPE == ATTN_F32 ? s[t][n][r] - w[n] : fmaf(s[t][n][r], sp.mul, -w[n]);
            } else if (sp.cap == CAP_FAST) {
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const float high = sp.cap2 - w[n];
#pragma unroll
                    for (int t = 0; t < KB; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][n][r] = TYPE == ATTN_F32 ? fmaf(2.0f * sp.cap2, cap_h(s[t][n][r]), -w[n])
                                                          : fmaf(-2.0f * sp.cap2, cap_r(s[t][n][r] * sp.mul2), high);
                }
            } else {
#pragma unroll
                for (int t = 0; t < KB; ++t)
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][n][r] = fmaf(sp.cap2, attn_tanh(scaled<TYPE>(s[t][n][r], sp.mul)), -w[n]);
            }
            if (sp.bias == 1) {
                const float k0 = (float)(base + 16 * kb + 4 * g);
#pragma unroll
                for (int t = 0; t < KB; ++t)
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][n][r] = fmaf(-sp.slope2, fabsf((qx[n] - k0) - (float)(16 * t + r)), s[t][n][r]);
            } else if (sp.bias == 2) {
#pragma unroll
                for (int t = 0; t < KB; ++t) {
                    const float *at = key_pos + 2 * (16 * (kb + t) + 4 * g);
                    const f32x4 p0 = *reinterpret_cast<const f32x4 *>(at), p1 = *reinterpret_cast<const f32x4 *>(at + 4);
                    const float kx[4] = {p0[0], p0[2], p1[0], p1[2]}, ky[4] = {p0[1], p0[3], p1[1], p1[3]};
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float dx = qx[n] - kx[r], dy = qy[n] - ky[r];
                            s[t][n][r] = fmaf(-sp.slope2, __builtin_amdgcn_sqrtf(fmaf(dx, dx, dy * dy)), s[t][n][r]);
                        }
                }
            }
            if (by_limit) {
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const int left = limit[n] - (base + 16 * kb + 4 * g);
#pragma unroll
                    for (int t = 0; t < KB; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][n][r] = keep_or(mask_below(16 * t + r, left), s[t][n][r], -attn_inf());
                }
            }
            if (by_doc) {
#pragma unroll
                for (int t = 0; t < KB; ++t) {
                    const i32x4 kd = *reinterpret_cast<const i32x4 *>(key_doc + 16 * (kb + t) + 4 * g);
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][n][r] = keep_or(mask_equal(kd[r], doc[n]), s[t][n][r], -attn_inf());
                }
            }
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                float top = s[0][n][0];
#pragma unroll
                for (int t = 0; t < KB; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) top = fast_max(top, s[t][n][r]);
                if (__any(top > rise[n])) {
                    top = group_max(top);
                    const bool up = top > rise[n];
                    const float next = up ? w[n] + top : w[n], by = next - w[n];
                    const float f = rise[n] == -attn_inf() ? 1.0f : __builtin_amdgcn_exp2f(-by);     // (nothing summed yet: 1)
                    l[n] *= f;
#pragma unroll
                    for (int d = 0; d < S::dt; ++d) o[n][d] = o[n][d] * f;
                    w[n] = next;
                    if (up) rise[n] = SOFTMAX_RISE;
#pragma unroll
                    for (int t = 0; t < KB; ++t) s[t][n] = s[t][n] - f32x4{by, by, by, by};
                }
#pragma unroll
                for (int t = 0; t < KB; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[t][n][r] = __builtin_amdgcn_exp2f(s[t][n][r]);
                        l[n] += s[t][n][r];
                    }
            }
#pragma unroll
            for (int t = 0; t < KB; t += 2) accumulate<TYPE, DP, NQ>(o, Vt, (kb + t) / 2, s[t], s[t + 1], g, c);
        }
    }

#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int i = wrow0 + 16 * n + c;
        const float total = group_sum(l[n]);
        if (a.splits > 1) {
            if (i < a.Lq) {
                float *to = a.part + (((int64_t)bh * a.splits + split) * a.Lq + i) * (a.D + 4);
#pragma unroll
                for (int d = 0; d < S::dt; ++d)
                    if (16 * d + 4 * g < a.D) *reinterpret_cast<f32x4 *>(to + 16 * d + 4 * g) = o[n][d];
                if (g == 0) *reinterpret_cast<f32x2 *>(to + a.D) = f32x2{rise[n] == -attn_inf() ? -attn_inf() : w[n], total};
            }
            continue;
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        bool fine = true;
#pragma unroll
        for (int d = 0; d < S::dt; ++d) fine = fine && finite4(o[n][d]);
        if (i < a.Lq) {
            const int64_t out = b * a.os[0] + h * a.os[1] + (int64_t)i * a.os[2] + 4 * g;
#pragma unroll
            for (int d = 0; d < S::dt; ++d)
                if (16 * d + 4 * g < a.D) store_out4<TYPE>(a, out + 16 * d, o[n][d] * inv);
            if (a.lse != nullptr && g == 0)
                a.lse[((int64_t)b * a.Hq + h) * a.Lq + i] = total == 0.0f ? -attn_inf() : (w[n] + __builtin_amdgcn_logf(total)) * ATTN_LN2;
        }
        unsigned long long bad = __ballot(!fine && i < a.Lq);
        bad = (bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffff;
        for (; bad != 0; bad &= bad - 1) {
            careful_forward_row<TYPE>(a, sp, b, h, wrow0 + 16 * n + __ffsll((long long)bad) - 1);
        }
    }
}

// Joins the ranges of keys: one wave per row, lanes over the head size, in the order of the ranges.
template <int TYPE> __global__ __launch_bounds__(ATTN_THREADS) void attn_fwd_join_kernel(AttnArgs a) {
    typedef typename Elem<TYPE>::raw raw;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * (ATTN_THREADS / 64) + (threadIdx.x >> 6);
    if (row >= (int64_t)a.B * a.Hq * a.Lq) return;
    const int64_t bh = row / a.Lq;
    const int i = (int)(row % a.Lq), b = (int)(bh / a.Hq), h = (int)(bh % a.Hq);
    const float *from = a.part + (bh * a.splits * a.Lq + i) * (a.D + 4);
    const int64_t stride = (int64_t)a.Lq * (a.D + 4);
    float top = -attn_inf();
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, from[s * stride + a.D]);
    const float shift = top == -attn_inf() ? 0.0f : top;
    float total = 0.0f, acc0 = 0.0f, acc1 = 0.0f;
    for (int s = 0; s < a.splits; ++s) {
        const float *x = from + s * stride;
        const float f = __builtin_amdgcn_exp2f(x[a.D] - shift);
        total = fmaf(x[a.D + 1], f, total);
        if (lane < a.D) acc0 = fmaf(x[lane], f, acc0);
        if (lane + 64 < a.D) acc1 = fmaf(x[lane + 64], f, acc1);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int64_t o = b * a.os[0] + h * a.os[1] + i * a.os[2] + lane;
    if (lane < a.D) store_out<TYPE>(a, o, acc0 * inv);
    if (lane + 64 < a.D) store_out<TYPE>(a, o + 64, acc1 * inv);
    if (a.lse != nullptr && lane == 0) a.lse[row] = total == 0.0f ? -attn_inf() : (shift + __builtin_amdgcn_logf(total)) * ATTN_LN2;
    if (__any((acc0 + acc1) * 0.0f != 0.0f))
        careful_forward_row<TYPE>(a, score_params(a.scale, a.cap, a.bias, a.slope, h), b, h, i);
}

// ---------------------------------------------------------------------------------------------------------- backward
// The scalar part of the backward pass on the pairs of 2 x N blocks of 16 x 16, phase by phase: each phase is one uniform
// branch around 8 N independent chains a lane (a branch per block left too few to hide the latency of exp and rcp).
//   in   s = q.k,  dp = do.v - delta (the subtraction is the matrix instruction's initial accumulator), e = lse in units of
//        log2 (infinite for rows without a key), dist
//   out  s = p,  dp = ds = p (dp - delta)
// slack is 1 - tanh^2 = 4 (r - r^2) without its 4 (undo_factor).  FOLD: it goes into dp (which then ends as du); else it is
// returned, undefined without a cap (the slope's gradient needs ds itself).
template <int TYPE, int N, bool FOLD>
__device__ __forceinline__ void pair_probability(const ScoreParams &sp, f32x4 (&s)[2][N], f32x4 (&dp)[2][N], f32x4 (&slack)[2][N],
                                                 const f32x4 (&dist)[2][N], const f32x4 (&e)[2][N]) {
    if (sp.cap == CAP_NONE) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                f32x4 x = s[t][n];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = TYPE == ATTN_F32 ? x[r] - e[t][n][r] : fmaf(x[r], sp.mul, -e[t][n][r]);
                s[t][n] = x;
            }
    } else if (sp.cap == CAP_FAST) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                f32x4 x = s[t][n], k = x;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (TYPE == ATTN_F32) {
                        const float y = cap_h(x[r]);
                        x[r] = fmaf(2.0f * sp.cap2, y, -e[t][n][r]);
                        k[r] = fmaf(-y, y, 0.25f);
                    } else {
                        const float y = cap_r(x[r] * sp.mul2);
                        x[r] = fmaf(-2.0f * sp.cap2, y, sp.cap2 - e[t][n][r]);
                        k[r] = fmaf(-y, y, y);
                    }
                }
                s[t][n] = x;
                if constexpr (FOLD) dp[t][n] = dp[t][n] * k;
                else slack[t][n] = k;
            }
    } else {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                f32x4 x = s[t][n], k = x;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float th = attn_tanh(scaled<TYPE>(x[r], sp.mul));
                    x[r] = fmaf(sp.cap2, th, -e[t][n][r]);
                    k[r] = 0.25f * fmaf(-th, th, 1.0f);
                }
                s[t][n] = x;
                if constexpr (FOLD) dp[t][n] = dp[t][n] * k;
                else slack[t][n] = k;
            }
    }
    if (sp.bias) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                f32x4 x = s[t][n];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = fmaf(-sp.slope2, dist[t][n][r], x[r]);
                s[t][n] = x;
            }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int n = 0; n < N; ++n) {
            f32x4 x = s[t][n];
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = __builtin_amdgcn_exp2f(x[r]);
            s[t][n] = x;
            dp[t][n] = x * dp[t][n];
        }
}
__device__ __forceinline__ float undo_factor(const AttnArgs &a) { return a.cap > 0.0f ? 4.0f * a.scale : a.scale; }

// Half precision keeps 2^-24 at the least: score gradients of rows with a small do would vanish.  They are scaled by a
// power of two that brings the row's largest |do| to 8..16 (undone exactly in the result).
__device__ __forceinline__ int gradient_exponent(float amax) {
    if (!(amax > 0.0f) || !(amax < 3.0e38f)) return 0;
    return max(-100, min(100, 3 - ((int)(__float_as_uint(amax) >> 23) - 127)));
}
__device__ __forceinline__ float exp2_of(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }
// The scale of a row whose score gradients are zero - no gradient of its own, no key or a single one - or not finite, which the
// careful path deals with: larger than every other, so that it never is the least
#define NO_SCALE 0x1p127f

// ---- query rows: dq of NQ x 16 rows per wave, with delta_i = do_i . o_i on the way (kept for the kernel that owns the
// keys) and the rows' share of dslope.  sum_j ds_ij is zero by definition; what it is with the delta at hand (o may have
// been rounded to 16 bits, and its rest not kept) is measured and its part of the slope's gradient taken out again.
template <int TYPE>
__device__ void careful_dq_row(const AttnArgs &a, const ScoreParams &sp, int b, int h, int i, float lse2, float delta) {
    typedef typename Elem<TYPE>::raw raw;
    const int lane = threadIdx.x & 63, hk = h / a.G, limit = row_limit(a, b, i);
    const raw *q = reinterpret_cast<const raw *>(a.q) + b * a.qs[0] + h * a.qs[1] + i * a.qs[2];
    const raw *o = reinterpret_cast<const raw *>(a.dout) + b * a.dos[0] + h * a.dos[1] + i * a.dos[2];
    const raw *k = reinterpret_cast<const raw *>(a.k) + b * a.ks[0] + hk * a.ks[1];
    const raw *v = reinterpret_cast<const raw *>(a.v) + b * a.vs[0] + hk * a.vs[1];
    float acc0 = 0.0f, acc1 = 0.0f;
    for (int base = 0; base < limit; base += 64) {
        const int j = base + lane;
        const bool ok = pair_allowed(a, b, i, j, limit);
        float ds = 0.0f, th;
        if (ok) {
            const float p = __builtin_amdgcn_exp2f(pair_score<TYPE>(a, sp, b, i, j, q, k + j * a.ks[2], th) - lse2);
            float dp = 0.0f;
            for (int d = 0; d < a.D; ++d) dp = fmaf(elem_to_float<TYPE>(o[d]), elem_to_float<TYPE>(v[j * a.vs[2] + d]), dp);
            ds = p * (dp - delta) * fmaf(-th, th, 1.0f);
        }
        for (unsigned long long w = __ballot(ok); w != 0; w &= w - 1) {
            const int jj = __ffsll((long long)w) - 1;
            const float x = __shfl(ds, jj);
            const raw *kr = k + (int64_t)(base + jj) * a.ks[2];
            if (lane < a.D) acc0 = fmaf(x, elem_to_float<TYPE>(kr[lane]), acc0);
            if (lane + 64 < a.D) acc1 = fmaf(x, elem_to_float<TYPE>(kr[lane + 64]), acc1);
        }
    }
    raw *out = reinterpret_cast<raw *>(a.dq) + b * a.dqst[0] + h * a.dqst[1] + i * a.dqst[2];
    if (lane < a.D) store_wide<TYPE>(out, lane, acc0 * a.scale);
    if (lane + 64 < a.D) store_wide<TYPE>(out, lane + 64, acc1 * a.scale);
}

template <int TYPE, int DP, int NQ>
__global__ __launch_bounds__(ATTN_THREADS, DP <= 64 ? 2 : 1) void attn_bwd_q_kernel(AttnArgs a) {
    typedef Shape<TYPE, DP> S;
    typedef typename Elem<TYPE>::raw raw;
    constexpr int ROWS = 64 * NQ, HALVES = DP <= 32 ? 2 : 1;     // (unrolled, the halves of a tile of wide heads spill)
    __shared__ __align__(16) char Kt[S::bytes], Vt[S::bytes];
    __shared__ __align__(16) float key_pos[2 * ATTN_ROWS];
    __shared__ __align__(16) int key_doc[ATTN_ROWS];
    __shared__ TileMap map_store;
    __shared__ float part[4];
    const Work work = deal(a.causal, a.B * a.Hq, a.tiles);
    if (work.rank >= a.tiles) return;
    const int bh = work.unit, qt = a.tiles - 1 - work.rank;
    const int b = bh / a.Hq, h = bh % a.Hq, hk = h / a.G;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
    const int row0 = qt * ROWS, wrow0 = row0 + wave * 16 * NQ;
    const raw *q = reinterpret_cast<const raw *>(a.q) + b * a.qs[0] + h * a.qs[1];
    const char *k = a.k + (b * a.ks[0] + hk * a.ks[1]) * Elem<TYPE>::bytes;
    const char *v = a.v + (b * a.vs[0] + hk * a.vs[1]) * Elem<TYPE>::bytes;
    const raw *go = reinterpret_cast<const raw *>(a.dout) + b * a.dos[0] + h * a.dos[1];
    const raw *fo = reinterpret_cast<const raw *>(a.out) + b * a.os[0] + h * a.os[1];
    const raw *fr = a.rest != nullptr ? reinterpret_cast<const raw *>(a.rest) + b * a.os[0] + h * a.os[1] : nullptr;
    const int *docs = a.doc_k != nullptr ? a.doc_k + b * a.dks : nullptr;
    const ScoreParams sp = score_params(a.scale, a.cap, a.bias, a.slope, h);

    TileMap *map = nullptr;
    if (docs != nullptr) {
        map = &map_store;
        build_tile_map(map_store, a.doc_q + b * a.dqs, row0, ROWS, a.Lq, docs, a.Lk);
    }
    
    ColFrag<TYPE, DP> qf[NQ], of[NQ];
    f32x4 dq[NQ][S::dt];
    float lse2[NQ], delta[NQ], rs[NQ], qx[NQ], qy[NQ], excess[NQ], pd[NQ], dsl[NQ];
    int limit[NQ], doc[NQ], seen[NQ];            // seen: how many of the lane's keys the row sees
    int wave_limit = 0, wave_full = INT_MAX;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int i = wrow0 + 16 * n + c;
        const bool live = i < a.Lq;
        Eight<TYPE> q8[S::chunks], g8[S::chunks];
        float dot = 0.0f, amax = 0.0f;
#pragma unroll
        for (int k8 = 0; k8 < S::chunks; ++k8) {
            const int d = frag_d<DP>(k8, g);
            q8[k8] = load_eight<TYPE>(q + (int64_t)i * a.qs[2], d, live && d < a.D);
            g8[k8] = load_eight<TYPE>(go + (int64_t)i * a.dos[2], d, live && d < a.D);
            const Eight<TYPE> o8 = load_eight<TYPE>(fo + (int64_t)i * a.os[2], d, live && d < a.D && frag_counts<DP>(g));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = eight_at<TYPE>(g8[k8], e);
                if (frag_counts<DP>(g)) dot = fmaf(x, eight_at<TYPE>(o8, e), dot);
                amax = fmaxf(amax, fabsf(x));
            }
            if (TYPE != ATTN_F32 && fr != nullptr && frag_counts<DP>(g)) {
                const Eight<TYPE> r8 = load_eight<TYPE>(fr + (int64_t)i * a.os[2], d, live && d < a.D);
#pragma unroll
                for (int e = 0; e < 8; ++e) dot = fmaf(eight_at<TYPE>(g8[k8], e), eight_at<TYPE>(r8, e), dot);
            }
        }
        col_frag<TYPE, DP>(qf[n], q8, g, score_factor(sp));
        col_frag<TYPE, DP>(of[n], g8, g);
        delta[n] = group_sum(dot);
        const int64_t at = ((int64_t)b * a.Hq + h) * a.Lq + i;
        const float lse = live ? a.lse[at] : -attn_inf();
        lse2[n] = lse == -attn_inf() ? attn_inf() : lse * ATTN_LOG2E;
        rs[n] = 1.0f;
        float key_scale = NO_SCALE;
        if constexpr (TYPE == ATTN_F16) {          // probabilities carry the row's scale through their exponent
            amax = group_max(amax);
            const int e = gradient_exponent(amax);
            rs[n] = exp2_of(e);
            if (amax > 0.0f && amax < attn_inf() && lse2[n] != attn_inf()) key_scale = rs[n];
            lse2[n] -= (float)e;
        }
        if (live && g == 0) {
            a.delta[at] = delta[n];
            if (TYPE == ATTN_F16) a.rowscale[at] = key_scale;
        }
        limit[n] = row_limit(a, b, i);
        doc[n] = map != nullptr ? doc_of_query(a, b, i) : 0;
        qx[n] = qy[n] = excess[n] = pd[n] = dsl[n] = 0.0f;
        seen[n] = 0;
        if (a.bias == 1) qx[n] = (float)(i + a.Lk - a.Lq);
        if (a.bias == 2 && live) {
            qx[n] = a.pos_q[b * a.pqs + 2 * (int64_t)i];
            qy[n] = a.pos_q[b * a.pqs + 2 * (int64_t)i + 1];
        }
#pragma unroll
        for (int d = 0; d < S::dt; ++d) dq[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if (wrow0 < a.Lq) {
        wave_limit = row_limit(a, b, min(wrow0 + 16 * NQ, a.Lq) - 1);
        wave_full = row_limit(a, b, wrow0);
    }
    const int end = (row_limit(a, b, min(row0 + ROWS, a.Lq) - 1) + ATTN_ROWS - 1) / ATTN_ROWS;
    const bool want_slope = a.dslope_part != nullptr;

    Stager<TYPE, DP> stage;
    stage.init(a.ks[2], a.vs[2], a.D);
    float stage_pos = 0.0f;
    int stage_doc = -1;
    auto load = [&](int tile) {
        const int base = tile * ATTN_ROWS, left = a.Lk - base;
        const char *kt = k + base * a.ks[2] * Elem<TYPE>::bytes, *vt = v + base * a.vs[2] * Elem<TYPE>::bytes;
        stage.load(kt, vt, left, map != nullptr ? docs + base : nullptr);
        if (a.bias == 2 && tid < 2 * ATTN_ROWS) stage_pos = tid < 2 * left ? a.pos_k[b * a.pks + 2 * (int64_t)base + tid] : 0.0f;
        if (map != nullptr && tid < ATTN_ROWS) stage_doc = doc_of_key(a, b, base + tid);
    };
    int tile = next_tile(map, 0, end);
    if (tile < end) load(tile);
    while (tile < end) {
        __syncthreads();
        stage.write(Kt, Vt, map != nullptr);
        if (a.bias == 2 && tid < 2 * ATTN_ROWS) key_pos[tid] = stage_pos;
        if (map != nullptr && tid < ATTN_ROWS) key_doc[tid] = stage_doc;
        const int here = tile, base = here * ATTN_ROWS;
        tile = next_tile(map, here + 1, end);
        if (tile < end) load(tile);
        __syncthreads();
        if (base >= wave_limit) continue;
        const bool by_doc = !tile_same(map, here), masked = by_doc || base + ATTN_ROWS > wave_full;

#pragma unroll HALVES
        for (int tp = 0; tp < 2; ++tp) {
            f32x4 s[2][NQ], dp[2][NQ], slack[2][NQ] = {}, dist[2][NQ] = {};
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                RowFrag<TYPE, DP> f;
                row_frag<TYPE, DP>(f, Kt, 32 * tp + 16 * t + c, g);
#pragma unroll
                for (int n = 0; n < NQ; ++n) s[t][n] = dot_block<TYPE, DP>(f, qf[n]);
                row_frag<TYPE, DP>(f, Vt, 32 * tp + 16 * t + c, g);
#pragma unroll
                for (int n = 0; n < NQ; ++n) dp[t][n] = dot_block<TYPE, DP>(f, of[n], f32x4{-delta[n], -delta[n], -delta[n], -delta[n]});
            }
            if (sp.bias == 1) {
                const float k0 = (float)(base + 32 * tp + 4 * g);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) dist[t][n][r] = fabsf((qx[n] - k0) - (float)(16 * t + r));
            } else if (sp.bias == 2) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const float *at = key_pos + 2 * (32 * tp + 16 * t + 4 * g);
                    const f32x4 p0 = *reinterpret_cast<const f32x4 *>(at), p1 = *reinterpret_cast<const f32x4 *>(at + 4);
                    const float kx[4] = {p0[0], p0[2], p1[0], p1[2]}, ky[4] = {p0[1], p0[3], p1[1], p1[3]};
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float dx = qx[n] - kx[r], dy = qy[n] - ky[r];
                            dist[t][n][r] = __builtin_amdgcn_sqrtf(fmaf(dx, dx, dy * dy));
                        }
                }
            }
            f32x4 e[2][NQ];
#pragma unroll
            for (int n = 0; n < NQ; ++n) e[0][n] = e[1][n] = f32x4{lse2[n], lse2[n], lse2[n], lse2[n]};
            pair_probability<TYPE, NQ, false>(sp, s, dp, slack, dist, e);
            if (masked) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    i32x4 kd = {0, 0, 0, 0};
                    if (by_doc) kd = *reinterpret_cast<const i32x4 *>(key_doc + 32 * tp + 16 * t + 4 * g);
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        const int left = limit[n] - (base + 32 * tp + 4 * g), own = by_doc ? doc[n] : 0;
                        f32x4 p = s[t][n], ds = dp[t][n], away = dist[t][n];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const unsigned ok = mask_below(16 * t + r, left) & mask_equal(kd[r], own);
                            seen[n] -= (int)ok;
                            p[r] = keep_or_zero(ok, p[r]);
                            ds[r] = keep_or_zero(ok, ds[r]);
                            away[r] = keep_or_zero(ok, away[r]);             // (a masked key's coordinates may be NaN)
                        }
                        s[t][n] = p;
                        dp[t][n] = ds;
                        dist[t][n] = away;
                    }
                }
            } else {
#pragma unroll
                for (int n = 0; n < NQ; ++n) seen[n] += 8;
            }
            if (want_slope) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            excess[n] += dp[t][n][r];
                            pd[n] = fmaf(s[t][n][r], dist[t][n][r], pd[n]);
                            dsl[n] = fmaf(dp[t][n][r], dist[t][n][r], dsl[n]);
                        }
            }
            if (sp.cap) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int n = 0; n < NQ; ++n) dp[t][n] = dp[t][n] * slack[t][n];
            }
            accumulate<TYPE, DP, NQ>(dq, Kt, tp, dp[0], dp[1], g, c);
        }
    }

    float slope_sum = 0.0f;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int i = wrow0 + 16 * n + c;
        const bool live = i < a.Lq;
        bool fine = true;
        const float inv_rs = 1.0f / rs[n], undo = undo_factor(a) * inv_rs;
#pragma unroll
        for (int d = 0; d < S::dt; ++d) fine = fine && finite4(dq[n][d]);
        unsigned long long bad = __ballot(!fine && live);
        bad = (bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffff;
        // A single key has the probability 1 whatever its score: the row's score gradients are zero, and not what the rounding
        // of dp and delta leaves of their difference.  (Such a row is never in a tile without masks, here or below.)
        const bool single = group_sum((float)min(seen[n], 64)) == 1.0f && (bad >> c & 1) == 0;
        if (live) {
            raw *out = reinterpret_cast<raw *>(a.dq) + b * a.dqst[0] + h * a.dqst[1] + (int64_t)i * a.dqst[2];
#pragma unroll
            for (int d = 0; d < S::dt; ++d)
                if (16 * d + 4 * g < a.D) store4<TYPE>(out + 16 * d + 4 * g, single ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : dq[n][d] * undo);
            if (g == 0) {
                a.many[((int64_t)b * a.Hq + h) * a.Lq + i] = single ? 0 : -1;
                if (TYPE == ATTN_F16 && single) a.rowscale[((int64_t)b * a.Hq + h) * a.Lq + i] = NO_SCALE;
            }
        }
        for (; bad != 0; bad &= bad - 1) {
            const int cc = __ffsll((long long)bad) - 1;
            const int64_t at = ((int64_t)b * a.Hq + h) * a.Lq + wrow0 + 16 * n + cc;
            careful_dq_row<TYPE>(a, sp, b, h, wrow0 + 16 * n + cc, a.lse[at] * ATTN_LOG2E, __shfl(delta[n], cc));
        }
        if (want_slope) {
            const float e = group_sum(excess[n]) * inv_rs, x = group_sum(pd[n]) * inv_rs, y = group_sum(dsl[n]) * inv_rs;
            slope_sum += live && !single ? fmaf(-e, x, y) : 0.0f;
        }
    }
    if (want_slope) {
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) slope_sum += __shfl_xor(slope_sum, x);
        if (lane == 0) part[wave] = slope_sum;
        __syncthreads();
        if (tid == 0) a.dslope_part[(int64_t)bh * a.tiles + qt] = (part[0] + part[1]) + (part[2] + part[3]);
    }
}

// dslope[h] = - sum over batch entries and row blocks, in a fixed order, in binary64
__global__ __launch_bounds__(256) void attn_dslope_kernel(AttnArgs a) {
    __shared__ double sums[256];
    const int h = blockIdx.x, tid = threadIdx.x;
    double s = 0.0;
    for (int64_t x = tid; x < (int64_t)a.B * a.tiles; x += 256)
        s += (double)a.dslope_part[((x / a.tiles) * a.Hq + h) * a.tiles + x % a.tiles];
    sums[tid] = s;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if (tid < w) sums[tid] += sums[tid + w];
        __syncthreads();
    }
    if (tid == 0) a.dslope[h] = (float)-sums[0];
}

// ---- key rows: dk and dv of NK x 16 keys per wave, over the query rows of the heads that share them.  Lane (g, c) holds key
// c and, per 16 queries, the pairs with queries 4 g + r.  Where key blocks alone do not fill the chip, the heads of a group
// and the query rows are dealt to several workgroups (head_parts x splits), whose binary32 sums a second kernel adds.
template <int TYPE>
__device__ void careful_dkv_row(const AttnArgs &a, int b, int hk, int j) {
    typedef typename Elem<TYPE>::raw raw;
    const int lane = threadIdx.x & 63;
    const raw *k = reinterpret_cast<const raw *>(a.k) + b * a.ks[0] + hk * a.ks[1] + j * a.ks[2];
    const raw *v = reinterpret_cast<const raw *>(a.v) + b * a.vs[0] + hk * a.vs[1] + j * a.vs[2];
    float gk0 = 0.0f, gk1 = 0.0f, gv0 = 0.0f, gv1 = 0.0f;
    for (int h = hk * a.G; h < (hk + 1) * a.G; ++h) {
        const ScoreParams sp = score_params(a.scale, a.cap, a.bias, a.slope, h);
        const raw *q = reinterpret_cast<const raw *>(a.q) + b * a.qs[0] + h * a.qs[1];
        const raw *o = reinterpret_cast<const raw *>(a.dout) + b * a.dos[0] + h * a.dos[1];
        for (int base = 0; base < a.Lq; base += 64) {
            const int i = base + lane;
            const bool ok = i < a.Lq && pair_allowed(a, b, i, j, row_limit(a, b, i));
            float p = 0.0f, ds = 0.0f, th;
            if (ok) {
                const int64_t at = ((int64_t)b * a.Hq + h) * a.Lq + i;
                p = __builtin_amdgcn_exp2f(pair_score<TYPE>(a, sp, b, i, j, q + i * a.qs[2], k, th) - a.lse[at] * ATTN_LOG2E);
                float dp = 0.0f;
                for (int d = 0; d < a.D; ++d) dp = fmaf(elem_to_float<TYPE>(o[i * a.dos[2] + d]), elem_to_float<TYPE>(v[d]), dp);
                ds = p * (dp - a.delta[at]) * fmaf(-th, th, 1.0f);
            }
            for (unsigned long long w = __ballot(ok); w != 0; w &= w - 1) {
                const int ii = __ffsll((long long)w) - 1;
                const float x = __shfl(ds, ii), y = __shfl(p, ii);
                const raw *qr = q + (int64_t)(base + ii) * a.qs[2], *orow = o + (int64_t)(base + ii) * a.dos[2];
                if (lane < a.D) {
                    gk0 = fmaf(x, elem_to_float<TYPE>(qr[lane]), gk0);
                    gv0 = fmaf(y, elem_to_float<TYPE>(orow[lane]), gv0);
                }
                if (lane + 64 < a.D) {
                    gk1 = fmaf(x, elem_to_float<TYPE>(qr[lane + 64]), gk1);
                    gv1 = fmaf(y, elem_to_float<TYPE>(orow[lane + 64]), gv1);
                }
            }
        }
    }
    raw *outk = reinterpret_cast<raw *>(a.dk) + b * a.dkst[0] + hk * a.dkst[1] + j * a.dkst[2];
    raw *outv = reinterpret_cast<raw *>(a.dv) + b * a.dvst[0] + hk * a.dvst[1] + j * a.dvst[2];
    if (lane < a.D) {
        store_wide<TYPE>(outk, lane, gk0 * a.scale);
        store_wide<TYPE>(outv, lane, gv0);
    }
    if (lane + 64 < a.D) {
        store_wide<TYPE>(outk, lane + 64, gk1 * a.scale);
        store_wide<TYPE>(outv, lane + 64, gv1);
    }
}

#define F16_P_EXPONENT 10        // probabilities (<= 1) are rounded to binary16 times 2^10: those of long rows stay normal

template <int TYPE, int DP, int NK>
__global__ __launch_bounds__(ATTN_THREADS, DP <= 64 ? 2 : 1) void attn_bwd_kv_kernel(AttnArgs a) {
    typedef Shape<TYPE, DP> S;
    typedef typename Elem<TYPE>::raw raw;
    constexpr int ROWS = 64 * NK, HALVES = DP <= 32 ? 2 : 1;
    __shared__ __align__(16) char Qt[S::bytes], Ot[S::bytes];
    __shared__ __align__(16) float row_lse[ATTN_ROWS], row_delta[ATTN_ROWS], row_x[ATTN_ROWS], row_y[ATTN_ROWS];
    __shared__ __align__(16) int row_lim[ATTN_ROWS], row_doc[ATTN_ROWS], row_many[ATTN_ROWS];
    __shared__ TileMap map_store;
    __shared__ unsigned least_scale;
    const int parts = a.head_parts * a.splits;
    int work = xcd_work();
    if (work >= a.B * a.Hkv * a.tiles * parts) return;
    const int part = work % parts;
    work /= parts;
    const int bh = work / a.tiles, kt = work % a.tiles;          // (causal: the first keys are seen by the most rows)
    const int b = bh / a.Hkv, hk = bh % a.Hkv;
    const int hper = (a.G + a.head_parts - 1) / a.head_parts, h0 = hk * a.G + part / a.splits * hper;
    const int h1 = min(h0 + hper, (hk + 1) * a.G), split = part % a.splits;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
    const int row0 = kt * ROWS, wrow0 = row0 + wave * 16 * NK;
    const raw *k = reinterpret_cast<const raw *>(a.k) + b * a.ks[0] + hk * a.ks[1];
    const raw *v = reinterpret_cast<const raw *>(a.v) + b * a.vs[0] + hk * a.vs[1];
    const int *docs = a.doc_q != nullptr ? a.doc_q + b * a.dqs : nullptr;

    TileMap *map = nullptr;
    if (docs != nullptr) {
        map = &map_store;
        build_tile_map(map_store, a.doc_k + b * a.dks, row0, ROWS, a.Lk, docs, a.Lq);
    }

    const float factor = score_factor(score_params(a.scale, a.cap, 0, nullptr, 0));      // (the same for all heads)
    ColFrag<TYPE, DP> kf[NK], vf[NK];
    f32x4 dk[NK][S::dt], dv[NK][S::dt];
    float kx[NK], ky[NK];
    int doc[NK];
#pragma unroll
    for (int n = 0; n < NK; ++n) {
        const int j = wrow0 + 16 * n + c;
        const bool live = j < a.Lk;
        Eight<TYPE> k8[S::chunks], v8[S::chunks];
#pragma unroll
        for (int x = 0; x < S::chunks; ++x) {
            const int d = frag_d<DP>(x, g);
            k8[x] = load_eight<TYPE>(k + (int64_t)j * a.ks[2], d, live && d < a.D);
            v8[x] = load_eight<TYPE>(v + (int64_t)j * a.vs[2], d, live && d < a.D);
        }
        col_frag<TYPE, DP>(kf[n], k8, g, factor);
        col_frag<TYPE, DP>(vf[n], v8, g);
        doc[n] = map != nullptr ? doc_of_key(a, b, j) : 0;
        kx[n] = ky[n] = 0.0f;
        if (a.bias == 1) kx[n] = (float)j;
        if (a.bias == 2 && live) {
            kx[n] = a.pos_k[b * a.pks + 2 * (int64_t)j];
            ky[n] = a.pos_k[b * a.pks + 2 * (int64_t)j + 1];
        }
#pragma unroll
        for (int d = 0; d < S::dt; ++d) dk[n][d] = dv[n][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // the first query row that sees the first key of this block / of this wave
    int first = 0;
    if (a.causal && (a.prefix == nullptr || row0 >= a.prefix[b])) first = max(0, row0 - (a.Lk - a.Lq));
    const int all_begin = min(first, a.Lq) / ATTN_ROWS, all_end = (a.Lq + ATTN_ROWS - 1) / ATTN_ROWS;
    const int per = (all_end - all_begin + a.splits - 1) / a.splits;
    const int begin = all_begin + split * per, end = min(all_end, begin + per);
    int wave_first = 0;                              // rows before it see no key of the wave
    if (a.causal && (a.prefix == nullptr || wrow0 >= a.prefix[b])) wave_first = max(0, wrow0 - (a.Lk - a.Lq));
    const int wave_all = a.causal ? wrow0 + 16 * NK - 1 - (a.Lk - a.Lq) : 0;   // rows from here on see all keys of the wave
    const bool tail = wrow0 + 16 * NK > a.Lk;

    float gscale = 1.0f;
    if constexpr (TYPE == ATTN_F16) {               // one scale for all rows: that of the largest gradient among them
        const unsigned none = __float_as_uint(NO_SCALE);
        unsigned least = none;
        for (int h = h0; h < h1; ++h)
            for (int x = tid; x < a.Lq; x += ATTN_THREADS) least = min(least, __float_as_uint(a.rowscale[((int64_t)b * a.Hq + h) * a.Lq + x]));
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) least = min(least, (unsigned)__shfl_xor((int)least, x));
        if (tid == 0) least_scale = none;
        __syncthreads();
        if (lane == 0) atomicMin(&least_scale, least);
        __syncthreads();
        gscale = least_scale == none ? 1.0f : __uint_as_float(least_scale);
    }
    const float gmul = TYPE == ATTN_F16 ? gscale * exp2_of(-F16_P_EXPONENT) : 1.0f;

    Stager<TYPE, DP> stage;
    stage.init(a.qs[2], a.dos[2], a.D);
    for (int h = h0; h < h1; ++h) {
        const char *q = a.q + (b * a.qs[0] + h * a.qs[1]) * Elem<TYPE>::bytes;
        const char *go = a.dout + (b * a.dos[0] + h * a.dos[1]) * Elem<TYPE>::bytes;
        const float *lse = a.lse + ((int64_t)b * a.Hq + h) * a.Lq, *del = a.delta + ((int64_t)b * a.Hq + h) * a.Lq;
        const int *many = a.many + ((int64_t)b * a.Hq + h) * a.Lq;
        const ScoreParams sp = score_params(a.scale, a.cap, a.bias, a.slope, h);
        float st_lse = 0.0f, st_delta = 0.0f, st_x = 0.0f, st_y = 0.0f;
        int st_lim = 0, st_doc = -2, st_many = 0;
        auto load = [&](int tile) {
            const int base = tile * ATTN_ROWS, left = a.Lq - base;
            const char *qt = q + base * a.qs[2] * Elem<TYPE>::bytes, *ot = go + base * a.dos[2] * Elem<TYPE>::bytes;
            stage.load(qt, ot, left, map != nullptr ? docs + base : nullptr);
            if (tid < ATTN_ROWS) {
                const int i = base + tid;
                const bool live = i < a.Lq;
                const float e = live ? lse[i] : -attn_inf();
                st_lse = e == -attn_inf() ? attn_inf() : e * ATTN_LOG2E;
                if (TYPE == ATTN_F16) st_lse -= (float)F16_P_EXPONENT;
                st_delta = live ? -del[i] : 0.0f;
                st_many = live ? many[i] : 0;
                st_lim = row_limit(a, b, i);
                if (map != nullptr) st_doc = doc_of_query(a, b, i);
                if (a.bias == 1) st_x = (float)(i + a.Lk - a.Lq);
                if (a.bias == 2 && live) {
                    st_x = a.pos_q[b * a.pqs + 2 * (int64_t)i];
                    st_y = a.pos_q[b * a.pqs + 2 * (int64_t)i + 1];
                }
            }
        };
        int tile = next_tile(map, begin, end);
        if (tile < end) load(tile);
        while (tile < end) {
            __syncthreads();
            stage.write(Qt, Ot, map != nullptr);
            if (tid < ATTN_ROWS) {
                row_lse[tid] = st_lse;
                row_delta[tid] = st_delta;
                row_lim[tid] = st_lim;
                row_doc[tid] = st_doc;
                row_many[tid] = st_many;
                row_x[tid] = st_x;
                row_y[tid] = st_y;
            }
            const int here = tile, base = here * ATTN_ROWS;
            tile = next_tile(map, here + 1, end);
            if (tile < end) load(tile);
            __syncthreads();
            if (base + ATTN_ROWS <= wave_first || wrow0 >= a.Lk) continue;
            const bool by_doc = !tile_same(map, here), masked = by_doc || tail || base < wave_all || base + ATTN_ROWS > a.Lq;

#pragma unroll HALVES
            for (int tp = 0; tp < 2; ++tp) {
                f32x4 s[2][NK], dp[2][NK], slack[2][NK] = {}, dist[2][NK] = {}, e[2][NK];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int at = 32 * tp + 16 * t;
                    RowFrag<TYPE, DP> f;
                    row_frag<TYPE, DP>(f, Qt, at + c, g);
#pragma unroll
                    for (int n = 0; n < NK; ++n) s[t][n] = dot_block<TYPE, DP>(f, kf[n]);
                    const f32x4 minus_delta = *reinterpret_cast<const f32x4 *>(row_delta + at + 4 * g);
                    row_frag<TYPE, DP>(f, Ot, at + c, g);
#pragma unroll
                    for (int n = 0; n < NK; ++n) dp[t][n] = dot_block<TYPE, DP>(f, vf[n], minus_delta);
                    const f32x4 lse2 = *reinterpret_cast<const f32x4 *>(row_lse + at + 4 * g);
#pragma unroll
                    for (int n = 0; n < NK; ++n) e[t][n] = lse2;
                }
                if (sp.bias) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const f32x4 qx = *reinterpret_cast<const f32x4 *>(row_x + 32 * tp + 16 * t + 4 * g);
                        if (sp.bias == 1) {
#pragma unroll
                            for (int n = 0; n < NK; ++n)
#pragma unroll
                                for (int r = 0; r < 4; ++r) dist[t][n][r] = fabsf(qx[r] - kx[n]);
                        } else {
                            const f32x4 qy = *reinterpret_cast<const f32x4 *>(row_y + 32 * tp + 16 * t + 4 * g);
#pragma unroll
                            for (int n = 0; n < NK; ++n)
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    const float dx = qx[r] - kx[n], dy = qy[r] - ky[n];
                                    dist[t][n][r] = __builtin_amdgcn_sqrtf(fmaf(dx, dx, dy * dy));
                                }
                        }
                    }
                }
                pair_probability<TYPE, NK, true>(sp, s, dp, slack, dist, e);
                if (masked) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const i32x4 lim = *reinterpret_cast<const i32x4 *>(row_lim + 32 * tp + 16 * t + 4 * g);
                        const i32x4 more = *reinterpret_cast<const i32x4 *>(row_many + 32 * tp + 16 * t + 4 * g);
                        i32x4 qd = {0, 0, 0, 0};
                        if (by_doc) qd = *reinterpret_cast<const i32x4 *>(row_doc + 32 * tp + 16 * t + 4 * g);
#pragma unroll
                        for (int n = 0; n < NK; ++n) {
                            const int j = wrow0 + 16 * n + c, own = by_doc ? doc[n] : 0;
                            f32x4 p = s[t][n], ds = dp[t][n];
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const unsigned ok = mask_below(j, lim[r]) & mask_equal(qd[r], own);
                                p[r] = keep_or_zero(ok, p[r]);
                                ds[r] = keep_or_zero(ok & (unsigned)more[r], ds[r]);
                            }
                            s[t][n] = p;
                            dp[t][n] = ds;
                        }
                    }
                }
                accumulate<TYPE, DP, NK>(dv, Ot, tp, s[0], s[1], g, c);
                if (TYPE == ATTN_F16) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int n = 0; n < NK; ++n) dp[t][n] = dp[t][n] * gmul;
                }
                accumulate<TYPE, DP, NK>(dk, Qt, tp, dp[0], dp[1], g, c);
            }
        }
    }

    const float undo = undo_factor(a) / gscale, undo_v = TYPE == ATTN_F16 ? exp2_of(-F16_P_EXPONENT) : 1.0f;
#pragma unroll
    for (int n = 0; n < NK; ++n) {
        const int j = wrow0 + 16 * n + c;
        const bool live = j < a.Lk;
        if (parts > 1) {
            if (live) {
                float *to = a.part + (((int64_t)part * a.B * a.Hkv + bh) * a.Lk + j) * 2 * a.D;
#pragma unroll
                for (int d = 0; d < S::dt; ++d)
                    if (16 * d + 4 * g < a.D) {
                        *reinterpret_cast<f32x4 *>(to + 16 * d + 4 * g) = dk[n][d] * undo;
                        *reinterpret_cast<f32x4 *>(to + a.D + 16 * d + 4 * g) = dv[n][d] * undo_v;
                    }
            }
            continue;
        }
        bool fine = true;
#pragma unroll
        for (int d = 0; d < S::dt; ++d) fine = fine && finite4(dk[n][d]) && finite4(dv[n][d]);
        if (live) {
            raw *outk = reinterpret_cast<raw *>(a.dk) + b * a.dkst[0] + hk * a.dkst[1] + (int64_t)j * a.dkst[2];
            raw *outv = reinterpret_cast<raw *>(a.dv) + b * a.dvst[0] + hk * a.dvst[1] + (int64_t)j * a.dvst[2];
#pragma unroll
            for (int d = 0; d < S::dt; ++d)
                if (16 * d + 4 * g < a.D) {
                    store4<TYPE>(outk + 16 * d + 4 * g, dk[n][d] * undo);
                    store4<TYPE>(outv + 16 * d + 4 * g, dv[n][d] * undo_v);
                }
        }
        unsigned long long bad = __ballot(!fine && live);
        bad = (bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffff;
        for (; bad != 0; bad &= bad - 1) careful_dkv_row<TYPE>(a, b, hk, wrow0 + 16 * n + __ffsll((long long)bad) - 1);
    }
}

// Adds the parts of dk and dv, in order: one wave per key row.
template <int TYPE> __global__ __launch_bounds__(ATTN_THREADS) void attn_bwd_kv_join_kernel(AttnArgs a) {
    typedef typename Elem<TYPE>::raw raw;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * (ATTN_THREADS / 64) + (threadIdx.x >> 6), rows = (int64_t)a.B * a.Hkv * a.Lk;
    if (row >= rows) return;
    const int64_t bh = row / a.Lk;
    const int j = (int)(row % a.Lk), b = (int)(bh / a.Hkv), hk = (int)(bh % a.Hkv), parts = a.head_parts * a.splits;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};                  // dk, dv together are 2 D <= 256 values
    for (int p = 0; p < parts; ++p) {
        const float *from = a.part + (p * rows + row) * 2 * a.D;
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (lane + 64 * x < 2 * a.D) sum[x] += from[lane + 64 * x];
    }
    raw *outk = reinterpret_cast<raw *>(a.dk) + b * a.dkst[0] + hk * a.dkst[1] + j * a.dkst[2];
    raw *outv = reinterpret_cast<raw *>(a.dv) + b * a.dvst[0] + hk * a.dvst[1] + j * a.dvst[2];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const int d = lane + 64 * x;
        if (d < a.D) store_wide<TYPE>(outk, d, sum[x]);
        else if (d < 2 * a.D) store_wide<TYPE>(outv, d - a.D, sum[x]);
    }
    if (__any((sum[0] + sum[1] + sum[2] + sum[3]) * 0.0f != 0.0f)) careful_dkv_row<TYPE>(a, b, hk, j);
}

// ------------------------------------------------------------------------------------------------------------ launch
bool aligned_strides(const int64_t *s, const void *p, int bytes) {
    if ((reinterpret_cast<uintptr_t>(p) & 15) != 0) return false;
    for (int i = 0; i < 3; ++i)
        if ((s[i] * bytes) % 16 != 0 || s[i] < 0) return false;
    return s[2] * bytes < (1 << 26);             // a tile's rows are addressed by 32-bit offsets
}

int check_attention(const dgl_attention_t *p) {
    DGL_CHECK_ARG(p != nullptr, "NULL argument");
    DGL_CHECK_ARG(p->dtype >= DGL_DTYPE_F32 && p->dtype <= DGL_DTYPE_BF16, "unknown element type %d", p->dtype);
    DGL_CHECK_ARG(p->B >= 1 && p->Hq >= 1 && p->Hkv >= 1 && p->Lq >= 0 && p->Lk >= 0, "B=%d Hq=%d Hkv=%d Lq=%d Lk=%d", p->B, p->Hq,
                  p->Hkv, p->Lq, p->Lk);
    DGL_CHECK_ARG(p->Hq % p->Hkv == 0, "%d query heads over %d key heads", p->Hq, p->Hkv);
    DGL_CHECK_ARG(p->D >= 8 && p->D <= 128 && p->D % 8 == 0, "head size %d (a multiple of 8, at most 128)", p->D);
    DGL_CHECK_ARG(p->Lq <= DGL_ATTENTION_MAX_LENGTH && p->Lk <= DGL_ATTENTION_MAX_LENGTH, "length above %d", DGL_ATTENTION_MAX_LENGTH);
    DGL_CHECK_ARG(score_params_fit(p->scale, p->cap), "scale %g, cap %g", (double)p->scale, (double)p->cap);
    DGL_CHECK_ARG((p->pos_q == nullptr) == (p->pos_k == nullptr), "coordinates of one side only");
    DGL_CHECK_ARG(p->pos_q == nullptr || p->slope != nullptr, "coordinates without a slope");
    DGL_CHECK_ARG((p->doc_q == nullptr) == (p->doc_k == nullptr), "document ids of one side only");
    DGL_CHECK_ARG(p->prefix == nullptr || p->causal, "a prefix belongs to a causal mask");
    DGL_CHECK_ARG((int64_t)p->B * p->Hq * (((p->Lq > p->Lk ? p->Lq : p->Lk) + 63) / 64) < (1ll << 30), "too many rows");
    const int bytes = p->dtype == DGL_DTYPE_F32 ? 4 : 2;
    DGL_CHECK_ARG(p->Lq == 0 || (p->q != nullptr && p->out != nullptr), "q or out is NULL");
    DGL_CHECK_ARG(p->Lk == 0 || (p->k != nullptr && p->v != nullptr), "k or v is NULL");
    DGL_CHECK_ARG(aligned_strides(p->q_stride, p->q, bytes) && aligned_strides(p->k_stride, p->k, bytes) &&
                      aligned_strides(p->v_stride, p->v, bytes) && aligned_strides(p->o_stride, p->out, bytes),
                  "q, k, v, out: 16-byte aligned pointers and strides, tokens less than 64 MiB apart");
    DGL_CHECK_ARG(p->out_rest == nullptr || (p->dtype != DGL_DTYPE_F32 && (reinterpret_cast<uintptr_t>(p->out_rest) & 15) == 0),
                  "out_rest belongs to a 16-bit type, 16-byte aligned");
    return DGL_OK;
}

AttnArgs attention_args(const dgl_attention_t *p) {
    AttnArgs a{};
    a.q = (const char *)p->q; a.k = (const char *)p->k; a.v = (const char *)p->v; a.out = (char *)p->out;
    a.rest = (char *)p->out_rest; a.lse = p->lse;
    for (int i = 0; i < 3; ++i) { a.qs[i] = p->q_stride[i]; a.ks[i] = p->k_stride[i]; a.vs[i] = p->v_stride[i]; a.os[i] = p->o_stride[i]; }
    a.B = p->B; a.Hq = p->Hq; a.Hkv = p->Hkv; a.G = p->Hq / p->Hkv; a.Lq = p->Lq; a.Lk = p->Lk; a.D = p->D;
    a.causal = p->causal != 0; a.scale = p->scale; a.cap = p->cap;
    a.bias = p->slope == nullptr ? 0 : p->pos_q == nullptr ? 1 : 2;
    a.slope = p->slope; a.pos_q = p->pos_q; a.pos_k = p->pos_k; a.pqs = p->pos_q_stride; a.pks = p->pos_k_stride;
    a.doc_q = p->doc_q; a.doc_k = p->doc_k; a.dqs = p->doc_q_stride; a.dks = p->doc_k_stride; a.prefix = p->prefix;
    return a;
}

unsigned xcd_grid(int64_t work) { return (unsigned)((work + 7) / 8 * 8); }
int padded(int D) { return D <= 16 ? 16 : D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// Two blocks of 16 rows per wave halve the LDS reads per pair.  Two where the operands and sums of both fit the 256 registers
// of two waves per SIMD, and one where two would leave compute units idle (fewer than two workgroups for each of the 256).
enum { KERNEL_FWD, KERNEL_BWD_Q, KERNEL_BWD_KV };
constexpr bool two_fit(int kernel, int type, int DP) {
    return kernel == KERNEL_FWD ? !(type == ATTN_F32 && DP == 128) : DP <= (type == ATTN_F32 ? 32 : 64);
}
bool two_blocks(int kernel, int dtype, const AttnArgs &a, int rows, int heads) {
    return two_fit(kernel, dtype, padded(a.D)) && (int64_t)a.B * heads * ((rows + 127) / 128) >= 512;
}

// A long side is cut into ranges where the blocks of the other side are too few for the chip (512 workgroups wanted), as
// long as a range keeps eight tiles: below that the second launch costs more than the idle units.
int ranges(int64_t blocks, int length) {
    const int64_t want = blocks >= 512 ? 1 : (512 + blocks - 1) / blocks, most = (length + 511) / 512;
    return (int)(want < most ? want : most < 1 ? 1 : most);
}
void plan_forward(AttnArgs &a, int dtype, int &n) {
    n = two_blocks(KERNEL_FWD, dtype, a, a.Lq, a.Hq) ? 2 : 1;
    a.tiles = (a.Lq + 64 * n - 1) / (64 * n);
    a.splits = a.tiles > 0 ? ranges((int64_t)a.B * a.Hq * a.tiles, a.Lk) : 1;
}
void plan_keys(AttnArgs &a, int dtype, int &n) {
    // The heads of a group and ranges of 512 query rows can be dealt out as well, so two blocks of keys fill the chip earlier.
    // Not with documents: a range of rows may hold none of the block's documents, and the work is badly dealt (8 heads of 64
    // numbers, 6000 rows in 9 documents, fp16: 168 us with one block and no ranges, 237 us with two and ranges; 2 x 16 heads over
    // 4 of 64 numbers, 2047 causal rows behind a prefix, bf16: 146 us and 130 us).
    const int64_t pairs = (int64_t)a.B * a.Hq * ((a.Lk + 127) / 128) * ((a.Lq + 511) / 512);
    const bool two = a.doc_k != nullptr ? two_blocks(KERNEL_BWD_KV, dtype, a, a.Lk, a.Hkv)
                                        : two_fit(KERNEL_BWD_KV, dtype, padded(a.D)) && pairs >= 512;
    n = two ? 2 : 1;
    a.tiles = (a.Lk + 64 * n - 1) / (64 * n);
    const int64_t blocks = (int64_t)a.B * a.Hkv * (a.tiles > 0 ? a.tiles : 1);
    const int64_t want = blocks >= 768 ? 1 : (768 + blocks - 1) / blocks;       // (two or three workgroups fit a unit)
    const int heads = (int)((a.G + (want < a.G ? want : a.G) - 1) / (want < a.G ? want : a.G));
    a.head_parts = (a.G + heads - 1) / heads;
    a.splits = ranges(blocks * a.head_parts, a.Lq);
}
int64_t forward_floats(AttnArgs a, int dtype) {
    int n;
    plan_forward(a, dtype, n);
    return a.splits > 1 ? (int64_t)a.B * a.Hq * a.splits * a.Lq * (a.D + 4) : 0;
}
int64_t keys_floats(AttnArgs a, int dtype) {
    int n;
    plan_keys(a, dtype, n);
    const int64_t parts = (int64_t)a.head_parts * a.splits;
    return parts > 1 ? parts * a.B * a.Hkv * a.Lk * 2 * a.D : 0;
}

template <template <int, int, int> class Launch> int by_type(const AttnArgs &a, int dtype, int n, hipStream_t s) {
#define ATTN_CASE(T, DPV) \
    if (dtype == T && padded(a.D) == DPV) { \
        if constexpr (two_fit(Launch<T, DPV, 1>::kernel, T, DPV)) { \
            if (n == 2) return Launch<T, DPV, 2>::go(a, s); \
        } \
        return Launch<T, DPV, 1>::go(a, s); \
    }
    ATTN_CASE(ATTN_F32, 16) ATTN_CASE(ATTN_F32, 32) ATTN_CASE(ATTN_F32, 64) ATTN_CASE(ATTN_F32, 128)
    ATTN_CASE(ATTN_F16, 16) ATTN_CASE(ATTN_F16, 32) ATTN_CASE(ATTN_F16, 64) ATTN_CASE(ATTN_F16, 128)
    ATTN_CASE(ATTN_BF16, 16) ATTN_CASE(ATTN_BF16, 32) ATTN_CASE(ATTN_BF16, 64) ATTN_CASE(ATTN_BF16, 128)
#undef ATTN_CASE
    return dgl_set_error(DGL_ERR_INVALID_ARGUMENT, "unknown element type %d", dtype);
}
template <int T, int DP, int N> struct LaunchFwd {
    static constexpr int kernel = KERNEL_FWD;
    static int go(const AttnArgs &a, hipStream_t s) {
        hipLaunchKernelGGL((attn_fwd_kernel<T, DP, N>), dim3(xcd_grid((int64_t)a.B * a.Hq * a.tiles * a.splits)), dim3(ATTN_THREADS), 0, s, a);
        DGL_CHECK_LAUNCH("dgl_attention_forward");
        if (a.splits > 1) {
            const int64_t rows = (int64_t)a.B * a.Hq * a.Lq;
            hipLaunchKernelGGL((attn_fwd_join_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(ATTN_THREADS), 0, s, a);
            DGL_CHECK_LAUNCH("dgl_attention_forward (join)");
        }
        return DGL_OK;
    }
};
template <int T, int DP, int N> struct LaunchBwdQ {
    static constexpr int kernel = KERNEL_BWD_Q;
    static int go(const AttnArgs &a, hipStream_t s) {
        hipLaunchKernelGGL((attn_bwd_q_kernel<T, DP, N>), dim3(xcd_grid((int64_t)a.B * a.Hq * a.tiles)), dim3(ATTN_THREADS), 0, s, a);
        DGL_CHECK_LAUNCH("dgl_attention_backward (query rows)");
        return DGL_OK;
    }
};
template <int T, int DP, int N> struct LaunchBwdKv {
    static constexpr int kernel = KERNEL_BWD_KV;
    static int go(const AttnArgs &a, hipStream_t s) {
        const int64_t blocks = (int64_t)a.B * a.Hkv * a.tiles * a.head_parts * a.splits;
        hipLaunchKernelGGL((attn_bwd_kv_kernel<T, DP, N>), dim3(xcd_grid(blocks)), dim3(ATTN_THREADS), 0, s, a);
        DGL_CHECK_LAUNCH("dgl_attention_backward (key rows)");
        if (a.head_parts * a.splits > 1) {
            const int64_t rows = (int64_t)a.B * a.Hkv * a.Lk;
            hipLaunchKernelGGL((attn_bwd_kv_join_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(ATTN_THREADS), 0, s, a);
            DGL_CHECK_LAUNCH("dgl_attention_backward (join)");
        }
        return DGL_OK;
    }
};

}  // namespace

extern "C" int64_t dgl_attention_forward_workspace_floats(const dgl_attention_t *p) {
    return check_attention(p) != DGL_OK ? -1 : forward_floats(attention_args(p), p->dtype);
}

extern "C" int dgl_attention_forward(const dgl_attention_t *p, float *ws, dgl_stream_t stream) {
    if (int e = check_attention(p)) return e;
    if (p->Lq == 0) return DGL_OK;
    AttnArgs a = attention_args(p);
    int n;
    plan_forward(a, p->dtype, n);
    DGL_CHECK_ARG(a.splits == 1 || (ws != nullptr && (reinterpret_cast<uintptr_t>(ws) & 15) == 0), "a 16-byte aligned workspace is needed");
    a.part = ws;
    return by_type<LaunchFwd>(a, p->dtype, n, (hipStream_t)stream);
}

// Workspace of the backward pass: delta, (half precision) the row scales, the rows' flags, the slopes' partial sums, the parts of dk / dv
int64_t backward_rows(const dgl_attention_t *p) { return ((int64_t)p->B * p->Hq * p->Lq + 3) / 4 * 4; }
int64_t backward_slopes(const dgl_attention_t *p) { return ((int64_t)p->B * p->Hq * ((p->Lq + 63) / 64) + 3) / 4 * 4; }

extern "C" int64_t dgl_attention_backward_workspace_floats(const dgl_attention_t *p) {
    if (check_attention(p) != DGL_OK) return -1;
    return 3 * backward_rows(p) + backward_slopes(p) + keys_floats(attention_args(p), p->dtype) + 4;
}

extern "C" int dgl_attention_backward(const dgl_attention_t *p, const dgl_attention_grad_t *g, float *ws, dgl_stream_t stream) {
    if (int e = check_attention(p)) return e;
    DGL_CHECK_ARG(g != nullptr && ws != nullptr && (reinterpret_cast<uintptr_t>(ws) & 15) == 0, "NULL argument or misaligned workspace");
    DGL_CHECK_ARG((p->Lq == 0 || (g->dout != nullptr && g->dq != nullptr && p->lse != nullptr)) &&
                      (p->Lk == 0 || (g->dk != nullptr && g->dv != nullptr)), "dout, dq, dk, dv or lse is NULL");
    DGL_CHECK_ARG(g->dslope == nullptr || p->slope != nullptr, "dslope without a slope");
    const int bytes = p->dtype == DGL_DTYPE_F32 ? 4 : 2;
    DGL_CHECK_ARG(aligned_strides(g->dout_stride, g->dout, bytes) && aligned_strides(g->dq_stride, g->dq, bytes) &&
                      aligned_strides(g->dk_stride, g->dk, bytes) && aligned_strides(g->dv_stride, g->dv, bytes),
                  "dout, dq, dk, dv: 16-byte aligned pointers and strides, tokens less than 64 MiB apart");
    AttnArgs a = attention_args(p);
    a.dout = (const char *)g->dout; a.dq = (char *)g->dq; a.dk = (char *)g->dk; a.dv = (char *)g->dv; a.dslope = g->dslope;
    for (int i = 0; i < 3; ++i) {
        a.dos[i] = g->dout_stride[i]; a.dqst[i] = g->dq_stride[i]; a.dkst[i] = g->dk_stride[i]; a.dvst[i] = g->dv_stride[i];
    }
    a.delta = ws;
    a.rowscale = ws + backward_rows(p);
    a.many = reinterpret_cast<int *>(ws + 2 * backward_rows(p));
    a.dslope_part = g->dslope != nullptr ? ws + 3 * backward_rows(p) : nullptr;
    a.part = ws + 3 * backward_rows(p) + backward_slopes(p);
    hipStream_t s = (hipStream_t)stream;
    if (p->Lq > 0) {
        const int n = two_blocks(KERNEL_BWD_Q, p->dtype, a, a.Lq, a.Hq) ? 2 : 1;
        a.tiles = (a.Lq + 64 * n - 1) / (64 * n);
        if (int e = by_type<LaunchBwdQ>(a, p->dtype, n, s)) return e;
    }
    if (a.dslope != nullptr) {                       // (without rows: the empty sum)
        hipLaunchKernelGGL(attn_dslope_kernel, dim3(a.Hq), dim3(256), 0, s, a);
        DGL_CHECK_LAUNCH("dgl_attention_backward (slopes)");
    }
    if (p->Lk > 0) {
        int n;
        plan_keys(a, p->dtype, n);
        return by_type<LaunchBwdKv>(a, p->dtype, n, s);
    }
    return DGL_OK;
}
