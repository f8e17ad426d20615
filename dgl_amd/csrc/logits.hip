// Logits to log-probabilities: penalties for actions in a row's history, biases, temperature, blocked actions, the
// log-softmax of what is left and its greedy pick.
//
//   c = occurrences of a in the history;  c > 0:  x = (x > 0 ? x / repetition : x repetition) - presence - frequency c
//   x = (x + bias) / temperature;  blocked: x = -inf;   log_prob = x - log sum exp x;   pick = lowest index of the maximum
//
// Bound by reading the logits and writing the log-probabilities once.  Up to 24576 actions a row stays in the registers of
// one workgroup between the two (the policy's rows up to CVRP-12000 do); longer rows are cut into tiles of
// 8192 actions, one launch for the tiles' maxima and sums, a second one that computes the values again - reading the
// logits twice costs less than writing and reading back binary32 values in between.
// Occurrences are counted in LDS per row (or tile), with integer atomics: their order does not matter.
//
// Measured, per launch: 512 rows x 1000 with blocked bits 3.9 us; 512 x 20002 with bits shared by two moves, biases, penalties
// and a temperature, binary32, 25 us = 3.3 TB/s (14 us = 5.9 TB/s without controls); 256 x 131072, bf16, bits, penalties over a
// history of 2048, temperature: 44 us for the statistics and 47 us for the values (27 and 27 without controls, of which
// writing the result takes 20), 12 of each for counting the history once more per tile.
#include "common.h"

#include <cfloat>

namespace {

#define LOGITS_TILE 8192
#define LOGITS_TILE_THREADS 512

struct LogitsArgs {
    const void *logits;
    int64_t ls;
    const unsigned *blocked;          // 32-bit halves of the words
    int64_t bs;
    int halves, period;
    unsigned inv_period;
    const float *bias;
    int64_t bias_s;
    const int *history, *history_len;
    int64_t hs;
    int cols;
    const float *rep, *pres, *freq;
    float rep_all, pres_all, freq_all, temperature, inv_temperature;
    float *out;
    int64_t os;
    int *selected;
    int R, A, tiles;
    float *part;                      // [R][tiles][4]: maximum, sum, pick (bits), unused
};

template <int TYPE> struct LogitElem { typedef unsigned short raw; };
template <> struct LogitElem<0> { typedef float raw; };
template <int TYPE> __device__ __forceinline__ float logit_float(typename LogitElem<TYPE>::raw x) {
    if constexpr (TYPE == 0) return x;
    else if constexpr (TYPE == 1) return (float)__builtin_bit_cast(_Float16, x);
    else return __uint_as_float((unsigned)x << 16);
}

// V consecutive values by one access
template <int TYPE, int V> __device__ __forceinline__ void load_logits(float (&x)[V], const typename LogitElem<TYPE>::raw *p) {
    typedef typename LogitElem<TYPE>::raw raw;
    struct alignas(sizeof(raw) * V) Pack { raw e[V]; };
    const Pack v = *reinterpret_cast<const Pack *>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = logit_float<TYPE>(v.e[e]);
}

struct RowParams {
    float rep, pres, freq;
};
__device__ __forceinline__ RowParams row_params(const LogitsArgs &a, int r) {
    RowParams p;
    p.rep = a.rep != nullptr ? a.rep[r] : a.rep_all;
    p.pres = a.pres != nullptr ? a.pres[r] : a.pres_all;
    p.freq = a.freq != nullptr ? a.freq[r] : a.freq_all;
    return p;
}
// a mod period by a multiplication with floor(2^32 / period): at most two too low
__device__ __forceinline__ unsigned bit_of(const LogitsArgs &a, unsigned act) {
    if (act < (unsigned)a.period) return act;
    unsigned r = act - __umulhi(act, a.inv_period) * (unsigned)a.period;
    if (r >= (unsigned)a.period) r -= (unsigned)a.period;
    if (r >= (unsigned)a.period) r -= (unsigned)a.period;
    return r;
}
// The value of an action that occurs c > 0 times in the history
__device__ __forceinline__ float penalised(const RowParams &p, float x, unsigned c) {
    const float y = __fsub_rn(x > 0.0f ? __fdiv_rn(x, p.rep) : __fmul_rn(x, p.rep), p.pres);
    return __fsub_rn(y, __fmul_rn(p.freq, (float)c));
}

// Occurrences in LDS, two 16-bit fields to a word while a history has fewer than 65536 entries (a CVRP-10000 row's fields
// then leave room for several workgroups), else one 32-bit counter.
struct Counts {
    unsigned *word;
    bool narrow;
    __device__ __forceinline__ unsigned at(int i) const { return narrow ? (word[i >> 1] >> (16 * (i & 1))) & 0xffffu : word[i]; }
};
// Counts the actions first .. first + n - 1 in row r's history.  (Computing the penalised values here, by the threads that
// hold history entries, so that the values' owners only look them up, was 9 us slower at 256 x 131072 with 2048 entries.)
template <int THREADS> __device__ __forceinline__ void count_history(const Counts &c, const LogitsArgs &a, int r, int first, int n, int tid) {
    constexpr int EARLY = 4;                     // entries requested before the fields are cleared
    const int words = c.narrow ? (n + 1) / 2 : n;
    const int *h = a.history + r * a.hs;
    int early[EARLY];
#pragma unroll
    for (int k = 0; k < EARLY; ++k) early[k] = tid + k * THREADS < a.cols ? h[tid + k * THREADS] : -1;
    const int len = min(a.history_len != nullptr ? a.history_len[r] : a.cols, a.cols);
    for (int i = tid; i < words; i += THREADS) c.word[i] = 0;
    __syncthreads();
    auto add = [&](int action) {
        const int x = action - first;
        if (x >= 0 && x < n) atomicAdd(&c.word[c.narrow ? x >> 1 : x], c.narrow ? 1u << (16 * (x & 1)) : 1u);
    };
#pragma unroll
    for (int k = 0; k < EARLY; ++k)
        if (tid + k * THREADS < len) add(early[k]);
    for (int i = tid + EARLY * THREADS; i < len; i += THREADS) add(h[i]);
    __syncthreads();
}

// Blocked bits in LDS, one per action from `first` on, whatever the period: 32 of them are gathered from two neighbouring words
// (more only where the period ends among them).  The first ones are requested before the logits.  (Words read from memory for each
// thread's actions, after the logits: 22 us in place of 16 at 512 x 20002 with odd periods, where two words were needed per action.)
struct Window {
    unsigned bit, lo, hi;
};
__device__ __forceinline__ unsigned bits_at(const LogitsArgs &a, const unsigned *bits, int i) { return i < a.halves ? bits[i] : 0u; }
__device__ __forceinline__ Window request_bits(const LogitsArgs &a, int r, int first, int n, int w) {
    Window x = {0, 0, 0};
    if (32 * w >= n) return x;
    const unsigned *bits = a.blocked + r * a.bs;
    x.bit = bit_of(a, (unsigned)(first + 32 * w));
    x.lo = bits_at(a, bits, (int)(x.bit >> 5));
    x.hi = bits_at(a, bits, (int)(x.bit >> 5) + 1);
    return x;
}
__device__ __forceinline__ unsigned gather_bits(const LogitsArgs &a, int r, const Window &x) {
    unsigned v = __builtin_amdgcn_alignbit(x.hi, x.lo, x.bit & 31), filled = (unsigned)a.period - x.bit;
    const unsigned *bits = a.blocked + r * a.bs;
    while (filled < 32) {                        // the period starts again
        v &= (1u << filled) - 1;
        const unsigned next = __builtin_amdgcn_alignbit(bits_at(a, bits, 1), bits_at(a, bits, 0), 0);
        v |= next << filled;
        filled += min((unsigned)a.period, 32u);
    }
    return v;
}

__device__ __forceinline__ float shifted_exp(float x, float shift) { return __builtin_amdgcn_exp2f((x - shift) * 1.4426950408889634f); }

// Exchanges inside a wave by lane permutations of the vector unit: a shuffle takes the LDS pipe, and 18 of them per wave took
// 2 of 54 us at 256 x 131072 bf16 without controls.
template <int CTRL> __device__ __forceinline__ float permuted(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
#define DPP_SWAP_1 0xb1            // quad_perm(1, 0, 3, 2)
#define DPP_SWAP_2 0x4e            // quad_perm(2, 3, 0, 1)
#define DPP_HALF_MIRROR 0x141
#define DPP_MIRROR 0x140
template <typename F> __device__ __forceinline__ float wave_reduce(float x, F f) {
    x = f(x, permuted<DPP_SWAP_1>(x));
    x = f(x, permuted<DPP_SWAP_2>(x));
    x = f(x, permuted<DPP_HALF_MIRROR>(x));
    x = f(x, permuted<DPP_MIRROR>(x));
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(p[0]), __uint_as_float(p[1]));
    p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
// maximum / sum over the workgroup, in every thread; `slots` of each are their own
template <int THREADS> __device__ __forceinline__ float block_max(float v, float *slots, int tid) {
    v = wave_reduce(v, [](float x, float y) { return fmaxf(x, y); });
    if constexpr (THREADS > 64) {
        if ((tid & 63) == 0) slots[tid >> 6] = v;
        __syncthreads();
        v = slots[0];
#pragma unroll
        for (int w = 1; w < THREADS / 64; ++w) v = fmaxf(v, slots[w]);
    }
    return v;
}
// The sum, and the lowest of the indexes that threads have put into *index before (behind a barrier that set it to INT_MAX)
template <int THREADS> __device__ __forceinline__ float block_sum(float v, float *slots, int tid) {
    v = wave_reduce(v, [](float x, float y) { return x + y; });
    if ((tid & 63) == 0) slots[tid >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) v += slots[w];
    return v;
}

// Values of chunks tid, tid + THREADS, ... of V actions each from action `first` on, at most N chunks; dead places are -inf.
// Returns the thread's maximum.  The logits are requested first and arrive while the history is counted.  One uniform branch
// per control around all of a thread's values; every operation rounds once, as the header writes it.  Selections are bit
// operations on masks: a comparison into a scalar register and a v_cndmask from it cost five times as much here.
template <int TYPE, int THREADS, int N, int V>
__device__ __forceinline__ float load_values(float (&x)[N][V], const LogitsArgs &a, int r, int first, int n, unsigned *words, int tid) {
    typedef typename LogitElem<TYPE>::raw raw;
    unsigned *blocked_words = words, *count_words = words + (a.blocked != nullptr ? (n + 31) / 32 : 0);
    Window window = {0, 0, 0};
    if (a.blocked != nullptr) window = request_bits(a, r, first, n, tid);
    const raw *row = reinterpret_cast<const raw *>(a.logits) + r * a.ls + first;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int at = (k * THREADS + tid) * V;
        if (at < n) load_logits<TYPE, V>(x[k], row + at);
        else
#pragma unroll
            for (int e = 0; e < V; ++e) x[k][e] = -__builtin_inff();
    }
    if (a.blocked != nullptr) {
        if (32 * tid < n) blocked_words[tid] = gather_bits(a, r, window);
        for (int w = tid + THREADS; 32 * w < n; w += THREADS) blocked_words[w] = gather_bits(a, r, request_bits(a, r, first, n, w));
        if (a.history == nullptr) __syncthreads();
    }
    if (a.history != nullptr) {
        const Counts count = {count_words, a.cols < 65536};
        count_history<THREADS>(count, a, r, first, n, tid);
        const RowParams p = row_params(a, r);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int at = (k * THREADS + tid) * V;
            if (at >= n) continue;
            unsigned c[V], some = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) some |= c[e] = count.at(at + e);
            if (some == 0) continue;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c[e] != 0) x[k][e] = penalised(p, x[k][e], c[e]);
        }
    }
    if (a.bias != nullptr) {
        const float *b = a.bias + r * a.bias_s + first;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int at = (k * THREADS + tid) * V;
            if (at >= n) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) x[k][e] = __fadd_rn(x[k][e], b[at + e]);
        }
    }
    if (a.temperature != 1.0f) {
        // x / t, correctly rounded: with y the rounded reciprocal, q = x y is within an ulp, x - q t is exact, and one more
        // multiply-add rounds correctly (Markstein) while nothing over- or underflows.  A thread with a value outside 1e-15 ..
        // 1e15 (dead places apart), and every temperature outside that or with a significand of ones, divides.
        float small = 1.0f, large = 1.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if ((k * THREADS + tid) * V >= n) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                small = fminf(small, fabsf(x[k][e]));
                large = fmaxf(large, fabsf(x[k][e]));
            }
        }
        if (a.inv_temperature != 0.0f && small > 1.0e-15f && large < 1.0e15f) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                if ((k * THREADS + tid) * V >= n) continue;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float q = x[k][e] * a.inv_temperature;
                    x[k][e] = fmaf(fmaf(-q, a.temperature, x[k][e]), a.inv_temperature, q);
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) x[k][e] = __fdiv_rn(x[k][e], a.temperature);
        }
    }
    if (a.blocked != nullptr) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int at = (k * THREADS + tid) * V;
            if (at >= n) continue;
            const unsigned word = blocked_words[at >> 5] >> (at & 31);       // (V divides 32)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const unsigned mask = (unsigned)((int)(word << (31 - e)) >> 31);
                x[k][e] = __uint_as_float((__float_as_uint(x[k][e]) & ~mask) | (0xff800000u & mask));
            }
        }
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) top = fmaxf(top, x[k][e]);
    return top;
}
// the lowest index of the maximum among a thread's values
template <int THREADS, int N, int V> __device__ __forceinline__ int lowest_index(const float (&x)[N][V], float top, int first, int tid) {
    int index = INT_MAX;
#pragma unroll
    for (int k = N - 1; k >= 0; --k)
#pragma unroll
        for (int e = V - 1; e >= 0; --e)
            if (x[k][e] == top) index = first + (k * THREADS + tid) * V + e;
    return index;
}
template <int THREADS, int N, int V>
__device__ __forceinline__ void store_values(const float (&x)[N][V], float lse, float *row, int n, int tid) {
    const bool finite = lse - lse == 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int at = (k * THREADS + tid) * V;
        if (at >= n) continue;
        float y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            y[e] = x[k][e] - lse;
            if (!finite && x[k][e] == -__builtin_inff()) y[e] = x[k][e];      // (a row of NaN: what is blocked stays -inf)
        }
        struct alignas(4 * V) Pack { float e[V]; };
        Pack w;
#pragma unroll
        for (int e = 0; e < V; ++e) w.e[e] = y[e];
        *reinterpret_cast<Pack *>(row + at) = w;
    }
}

// one workgroup per row, the row in registers
template <int TYPE, int THREADS, int N, int V> __global__ __launch_bounds__(THREADS) void logits_row_kernel(LogitsArgs a) {
    extern __shared__ unsigned words[];
    __shared__ float max_slots[THREADS / 64], sum_slots[THREADS / 64];
    __shared__ int index;
    const int r = blockIdx.x, tid = threadIdx.x;
    float x[N][V];
    if (tid == 0) index = INT_MAX;
    const float own = load_values<TYPE, THREADS, N, V>(x, a, r, 0, a.A, words, tid);
    const float top = block_max<THREADS>(own, max_slots, tid), shift = top == -__builtin_inff() ? 0.0f : top;
    if (own == top && top != -__builtin_inff()) atomicMin(&index, lowest_index<THREADS, N, V>(x, top, 0, tid));
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) sum += shifted_exp(x[k][e], shift);
    sum = block_sum<THREADS>(sum, sum_slots, tid);
    if (a.selected != nullptr && tid == 0) a.selected[r] = index == INT_MAX ? -1 : index;
    if (a.out != nullptr) store_values<THREADS, N, V>(x, top == -__builtin_inff() ? 0.0f : shift + logf(sum), a.out + r * a.os, a.A, tid);
}

// long rows: one workgroup per tile; WRITE = second launch
template <int TYPE, int V, bool WRITE> __global__ __launch_bounds__(LOGITS_TILE_THREADS) void logits_tile_kernel(LogitsArgs a) {
    constexpr int THREADS = LOGITS_TILE_THREADS, N = LOGITS_TILE / THREADS / V;
    extern __shared__ unsigned words[];
    __shared__ float max_slots[THREADS / 64], sum_slots[THREADS / 64];
    __shared__ int index;
    const int r = blockIdx.x / a.tiles, t = blockIdx.x % a.tiles, tid = threadIdx.x;
    const int first = t * LOGITS_TILE, n = min(LOGITS_TILE, a.A - first);
    float x[N][V];
    if (tid == 0) index = INT_MAX;
    if constexpr (WRITE) {
        // the row's maximum and sum from its tiles', in a fixed order
        const float *p = a.part + (int64_t)r * a.tiles * 4;
        float top = -__builtin_inff();
        for (int i = tid; i < a.tiles; i += THREADS) top = fmaxf(top, p[4 * i]);
        top = block_max<THREADS>(top, max_slots, tid);
        const float shift = top == -__builtin_inff() ? 0.0f : top;
        float sum = 0.0f;
        for (int i = tid; i < a.tiles; i += THREADS) {
            const float m = p[4 * i];
            sum = fmaf(p[4 * i + 1], m == -__builtin_inff() ? 1.0f : shifted_exp(m, shift), sum);
            if (m == top) atomicMin(&index, __float_as_int(p[4 * i + 2]));
        }
        sum = block_sum<THREADS>(sum, sum_slots, tid);
        const float lse = top == -__builtin_inff() ? 0.0f : shift + logf(sum);
        if (a.selected != nullptr && t == 0 && tid == 0) a.selected[r] = index == INT_MAX ? -1 : index;
        if (a.out == nullptr) return;
        load_values<TYPE, THREADS, N, V>(x, a, r, first, n, words, tid);
        store_values<THREADS, N, V>(x, lse, a.out + r * a.os + first, n, tid);
    } else {
        const float own = load_values<TYPE, THREADS, N, V>(x, a, r, first, n, words, tid);
        const float top = block_max<THREADS>(own, max_slots, tid), shift = top == -__builtin_inff() ? 0.0f : top;
        if (own == top && top != -__builtin_inff()) atomicMin(&index, lowest_index<THREADS, N, V>(x, top, first, tid));
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) sum += shifted_exp(x[k][e], shift);
        sum = block_sum<THREADS>(sum, sum_slots, tid);
        if (tid == 0) {
            float *p = a.part + ((int64_t)r * a.tiles + t) * 4;
            p[0] = top;
            p[1] = sum;
            p[2] = __int_as_float(index);
        }
    }
}

int check_logits(const dgl_logits_t *p) {
    DGL_CHECK_ARG(p != nullptr, "NULL argument");
    DGL_CHECK_ARG(p->dtype >= DGL_DTYPE_F32 && p->dtype <= DGL_DTYPE_BF16, "unknown element type %d", p->dtype);
    DGL_CHECK_ARG(p->R >= 0 && p->A >= 1 && p->A <= (1 << 30), "R=%d rows of A=%d actions", p->R, p->A);
    DGL_CHECK_ARG(p->logits_stride >= 0 && p->out_stride >= 0 && p->bias_stride >= 0 && p->blocked_stride >= 0 && p->history_stride >= 0, "negative stride");
    DGL_CHECK_ARG(p->logits != nullptr && (p->log_probs != nullptr || p->selected != nullptr), "logits or every output is NULL");
    DGL_CHECK_ARG(p->log_probs == nullptr || p->out_stride >= p->A || p->R <= 1, "rows of the output overlap");
    DGL_CHECK_ARG(p->temperature > 0.0f && p->temperature < 3.0e38f, "temperature %g", (double)p->temperature);
    DGL_CHECK_ARG(p->blocked == nullptr || (p->period >= 1 && p->A % p->period == 0 && p->words >= 0), "A=%d actions share %d bits", p->A, p->period);
    DGL_CHECK_ARG(p->history == nullptr || p->history_cols >= 0, "history of %d", p->history_cols);
    DGL_CHECK_ARG(p->history == nullptr || p->repetition != nullptr || p->repetition_all > 0.0f, "repetition %g", (double)p->repetition_all);
    return DGL_OK;
}
#define LOGITS_ROW_MAX 24576           // 512 threads x 48 values
bool in_tiles(const dgl_logits_t *p) { return p->A > LOGITS_ROW_MAX; }

// LDS of n actions: blocked bits, then counters
int word_bytes(const LogitsArgs &a, int n) {
    return (a.blocked == nullptr ? 0 : (n + 31) / 32 * 4) + (a.history == nullptr ? 0 : a.cols < 65536 ? (n + 1) / 2 * 4 : n * 4);
}
template <int TYPE, int THREADS, int N, int V> void launch_row(const LogitsArgs &a, hipStream_t s) {
    const int lds = word_bytes(a, a.A);
    if (lds > 48 * 1024) dgl_max_dynamic_lds(reinterpret_cast<const void *>(&logits_row_kernel<TYPE, THREADS, N, V>), LOGITS_ROW_MAX * 4 + LOGITS_ROW_MAX / 8);
    hipLaunchKernelGGL((logits_row_kernel<TYPE, THREADS, N, V>), dim3(a.R), dim3(THREADS), lds, s, a);
}
// The smallest workgroup that holds a row at 4 to 48 values a thread; several share a compute unit, so that one row's loads
// run beside another's reductions and stores
template <int TYPE, int V> int launch_logits(const LogitsArgs &a, hipStream_t s) {
    if (a.A <= 256) launch_row<TYPE, 64, 4 / V, V>(a, s);
    else if (a.A <= 1024) launch_row<TYPE, 256, 4 / V, V>(a, s);
    else if (a.A <= 4096) launch_row<TYPE, 256, 16 / V, V>(a, s);
    else if (a.A <= 8192) launch_row<TYPE, 512, 16 / V, V>(a, s);
    else if (a.A <= 16384) launch_row<TYPE, 512, 32 / V, V>(a, s);
    else if (a.A <= LOGITS_ROW_MAX) launch_row<TYPE, 512, 48 / V, V>(a, s);
    else {
        const int lds = word_bytes(a, LOGITS_TILE);
        const dim3 grid((unsigned)((int64_t)a.R * a.tiles));
        hipLaunchKernelGGL((logits_tile_kernel<TYPE, V, false>), grid, dim3(LOGITS_TILE_THREADS), lds, s, a);
        DGL_CHECK_LAUNCH("dgl_logits_process (statistics)");
        hipLaunchKernelGGL((logits_tile_kernel<TYPE, V, true>), grid, dim3(LOGITS_TILE_THREADS), lds, s, a);
    }
    DGL_CHECK_LAUNCH("dgl_logits_process");
    return DGL_OK;
}

}  // namespace

extern "C" int64_t dgl_logits_workspace_floats(const dgl_logits_t *p) {
    if (check_logits(p) != DGL_OK) return -1;
    return in_tiles(p) ? (int64_t)p->R * ((p->A + LOGITS_TILE - 1) / LOGITS_TILE) * 4 : 0;
}

extern "C" int dgl_logits_process(const dgl_logits_t *p, float *ws, dgl_stream_t stream) {
    if (int e = check_logits(p)) return e;
    if (p->R == 0) return DGL_OK;
    LogitsArgs a{};
    a.logits = p->logits; a.ls = p->logits_stride; a.blocked = (const unsigned *)p->blocked; a.bs = 2 * p->blocked_stride;
    a.halves = 2 * p->words; a.period = p->period > 0 ? p->period : p->A;
    a.inv_period = a.period == 1 ? 0xffffffffu : (unsigned)((1ull << 32) / (unsigned)a.period);
    a.bias = p->bias; a.bias_s = p->bias_stride; a.history = p->history; a.history_len = p->history_len; a.hs = p->history_stride;
    a.cols = p->history_cols; a.rep = p->repetition; a.pres = p->presence; a.freq = p->frequency;
    a.rep_all = p->repetition_all; a.pres_all = p->presence_all; a.freq_all = p->frequency_all; a.temperature = p->temperature;
    a.out = p->log_probs; a.os = p->out_stride; a.selected = p->selected; a.R = p->R; a.A = p->A;
    a.tiles = (p->A + LOGITS_TILE - 1) / LOGITS_TILE; a.part = ws;
    DGL_CHECK_ARG(!in_tiles(p) || ws != nullptr, "a workspace is needed");
    DGL_CHECK_ARG((int64_t)a.R * a.tiles < (1ll << 31), "too many rows");
    // penalties that change nothing need no counts
    if (a.rep == nullptr && a.pres == nullptr && a.freq == nullptr && a.rep_all == 1.0f && a.pres_all == 0.0f && a.freq_all == 0.0f) a.history = nullptr;
    const bool all_ones = (__builtin_bit_cast(unsigned, a.temperature) & 0x7fffffu) == 0x7fffffu;
    a.inv_temperature = all_ones || a.temperature < 1.0e-15f || a.temperature > 1.0e15f ? 0.0f : 1.0f / a.temperature;
    // the widest access that every row of the logits and of the result can take
    const int bytes = p->dtype == DGL_DTYPE_F32 ? 4 : 2;
    auto fits = [&](int v) {
        return p->A % v == 0 && p->logits_stride % v == 0 && p->out_stride % v == 0 &&
               (reinterpret_cast<uintptr_t>(p->logits) & (v * bytes - 1)) == 0 && (reinterpret_cast<uintptr_t>(p->log_probs) & (4 * v - 1)) == 0;
    };
    const int v = fits(4) ? 4 : fits(2) ? 2 : 1;
    hipStream_t s = (hipStream_t)stream;
#define LOGITS_CASE(T) \
    if (p->dtype == T) return v == 4 ? launch_logits<T, 4>(a, s) : v == 2 ? launch_logits<T, 2>(a, s) : launch_logits<T, 1>(a, s);
    LOGITS_CASE(0) LOGITS_CASE(1) LOGITS_CASE(2)
#undef LOGITS_CASE
    return dgl_set_error(DGL_ERR_INVALID_ARGUMENT, "unknown element type %d", p->dtype);
}
