// Logits to log-probabilities: penalties for actions in a row's history, biases, temperature, blocked actions, the
// log-softmax of what is left and its greedy pick.
//
//   c = occurrences of a in the history;  c > 0:  x = (x > 0 ? x / repetition : x repetition) - presence - frequency c
//   x = (x + bias) / temperature;  blocked: x = -inf;   log_prob = x - log sum exp x;   pick = lowest index of the maximum
//
// Bound by reading the logits and writing the log-probabilities once.  Up to 32 values per thread a row stays in the
// registers of one workgroup between the two (a row of the policy's actions always does); longer rows are cut into tiles of
// 8192 actions, one launch for the tiles' maxima and sums, a second one that computes the values again - reading the
// logits twice costs less than writing and reading back binary32 values in between.
// Occurrences are counted in LDS per row (or tile), with integer atomics: their order does not matter.
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
    float rep_all, pres_all, freq_all, temperature;
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

// V consecutive values (V = 4: one access of 16 or 8 bytes)
template <int TYPE, int V> __device__ __forceinline__ void load_logits(float (&x)[V], const typename LogitElem<TYPE>::raw *p) {
    if constexpr (V == 1) {
        x[0] = logit_float<TYPE>(p[0]);
    } else if constexpr (TYPE == 0) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
        const ushort4 v = *reinterpret_cast<const ushort4 *>(p);
        x[0] = logit_float<TYPE>(v.x); x[1] = logit_float<TYPE>(v.y); x[2] = logit_float<TYPE>(v.z); x[3] = logit_float<TYPE>(v.w);
    }
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
// the value of action `act` of row r; count: its occurrences (0 without a history).  Every operation rounds once, as written
__device__ __forceinline__ float process(const LogitsArgs &a, const RowParams &p, int r, int act, float x, unsigned count) {
    if (count != 0) {
        x = __fsub_rn(x > 0.0f ? __fdiv_rn(x, p.rep) : __fmul_rn(x, p.rep), p.pres);
        x = __fsub_rn(x, __fmul_rn(p.freq, (float)count));
    }
    if (a.bias != nullptr) x = __fadd_rn(x, a.bias[r * a.bias_s + act]);
    if (a.temperature != 1.0f) x = __fdiv_rn(x, a.temperature);
    if (a.blocked != nullptr) {
        const unsigned bit = bit_of(a, (unsigned)act);
        if ((int)(bit >> 5) < a.halves && ((a.blocked[r * a.bs + (bit >> 5)] >> (bit & 31)) & 1)) x = -__builtin_inff();
    }
    return x;
}

// counts of the actions first .. first + n - 1 of row r, by THREADS threads (a barrier on either side for more than a wave)
template <int THREADS> __device__ __forceinline__ void count_history(unsigned *count, const LogitsArgs &a, int r, int first, int n, int tid) {
    for (int i = tid; i < n; i += THREADS) count[i] = 0;
    __syncthreads();
    const int len = min(a.history_len != nullptr ? a.history_len[r] : a.cols, a.cols);
    const int *h = a.history + r * a.hs;
    for (int i = tid; i < len; i += THREADS) {
        const int x = h[i] - first;
        if (x >= 0 && x < n) atomicAdd(&count[x], 1u);
    }
    __syncthreads();
}

struct Best {
    float value;
    int index;                                   // INT_MAX: none
};
__device__ __forceinline__ Best better(Best a, Best b) { return b.value > a.value || (b.value == a.value && b.index < a.index) ? b : a; }
__device__ __forceinline__ float shifted_exp(float x, float shift) { return __builtin_amdgcn_exp2f((x - shift) * 1.4426950408889634f); }

// maximum with its lowest index over the workgroup, in every thread
template <int THREADS> __device__ __forceinline__ Best block_best(Best v, Best *slots, int tid) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = better(v, Best{__shfl_xor(v.value, d), __shfl_xor(v.index, d)});
    if constexpr (THREADS > 64) {
        if ((tid & 63) == 0) slots[tid >> 6] = v;
        __syncthreads();
        v = slots[0];
#pragma unroll
        for (int w = 1; w < THREADS / 64; ++w) v = better(v, slots[w]);
    }
    return v;
}
template <int THREADS> __device__ __forceinline__ float block_sum(float v, float *slots, int tid) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    if constexpr (THREADS > 64) {
        if ((tid & 63) == 0) slots[tid >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) v += slots[w];
    }
    return v;
}

// values of chunks tid, tid + THREADS, ... of V actions each from action `first` on, at most N chunks; dead places are -inf
// and their index INT_MAX
template <int TYPE, int THREADS, int N, int V>
__device__ __forceinline__ Best load_values(float (&x)[N][V], const LogitsArgs &a, int r, int first, int n, const unsigned *count, int tid) {
    typedef typename LogitElem<TYPE>::raw raw;
    const raw *row = reinterpret_cast<const raw *>(a.logits) + r * a.ls + first;
    const RowParams p = row_params(a, r);
    Best best = {-__builtin_inff(), INT_MAX};
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int at = (k * THREADS + tid) * V;
        if (at < n) load_logits<TYPE, V>(x[k], row + at);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int at = (k * THREADS + tid) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (at >= n) {
                x[k][e] = -__builtin_inff();
                continue;
            }
            x[k][e] = process(a, p, r, first + at + e, x[k][e], count != nullptr ? count[at + e] : 0u);
            if (x[k][e] > best.value) best = Best{x[k][e], first + at + e};
        }
    }
    return best;
}
template <int THREADS, int N, int V>
__device__ __forceinline__ void store_values(const float (&x)[N][V], float lse, float *row, int n, int tid) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int at = (k * THREADS + tid) * V;
        if (at >= n) continue;
        float y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = x[k][e] == -__builtin_inff() ? x[k][e] : x[k][e] - lse;
        if constexpr (V == 4) *reinterpret_cast<float4 *>(row + at) = float4{y[0], y[1], y[2], y[3]};
        else row[at] = y[0];
    }
}

// one workgroup per row, the row in registers
template <int TYPE, int THREADS, int N, int V> __global__ __launch_bounds__(THREADS) void logits_row_kernel(LogitsArgs a) {
    extern __shared__ unsigned count[];
    __shared__ Best best_slots[THREADS / 64];
    __shared__ float sum_slots[THREADS / 64];
    const int r = blockIdx.x, tid = threadIdx.x;
    if (a.history != nullptr) count_history<THREADS>(count, a, r, 0, a.A, tid);
    float x[N][V];
    Best best = load_values<TYPE, THREADS, N, V>(x, a, r, 0, a.A, a.history != nullptr ? count : nullptr, tid);
    best = block_best<THREADS>(best, best_slots, tid);
    const float shift = best.value == -__builtin_inff() ? 0.0f : best.value;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) sum += shifted_exp(x[k][e], shift);
    sum = block_sum<THREADS>(sum, sum_slots, tid);
    if (a.selected != nullptr && tid == 0) a.selected[r] = best.index == INT_MAX ? -1 : best.index;
    if (a.out != nullptr) store_values<THREADS, N, V>(x, shift + logf(sum), a.out + r * a.os, a.A, tid);
}

// long rows: one workgroup per tile; `write` = second launch
template <int TYPE, int V, bool WRITE> __global__ __launch_bounds__(LOGITS_TILE_THREADS) void logits_tile_kernel(LogitsArgs a) {
    constexpr int THREADS = LOGITS_TILE_THREADS, N = LOGITS_TILE / THREADS / V;
    extern __shared__ unsigned count[];
    __shared__ Best best_slots[THREADS / 64];
    __shared__ float sum_slots[THREADS / 64];
    const int r = blockIdx.x / a.tiles, t = blockIdx.x % a.tiles, tid = threadIdx.x;
    const int first = t * LOGITS_TILE, n = min(LOGITS_TILE, a.A - first);
    float lse = 0.0f;
    if constexpr (WRITE) {
        // the row's maximum and sum from its tiles', in a fixed order
        const float *p = a.part + (int64_t)r * a.tiles * 4;
        Best best = {-__builtin_inff(), INT_MAX};
        for (int i = tid; i < a.tiles; i += THREADS) best = better(best, Best{p[4 * i], __float_as_int(p[4 * i + 2])});
        best = block_best<THREADS>(best, best_slots, tid);
        const float shift = best.value == -__builtin_inff() ? 0.0f : best.value;
        float sum = 0.0f;
        for (int i = tid; i < a.tiles; i += THREADS) sum = fmaf(p[4 * i + 1], shifted_exp(p[4 * i] == -__builtin_inff() ? shift : p[4 * i], shift), sum);
        sum = block_sum<THREADS>(sum, sum_slots, tid);
        lse = shift + logf(sum);
        if (a.selected != nullptr && t == 0 && tid == 0) a.selected[r] = best.index == INT_MAX ? -1 : best.index;
        if (a.out == nullptr) return;
    }
    if (a.history != nullptr) count_history<THREADS>(count, a, r, first, n, tid);
    float x[N][V];
    Best best = load_values<TYPE, THREADS, N, V>(x, a, r, first, n, a.history != nullptr ? count : nullptr, tid);
    if constexpr (WRITE) {
        store_values<THREADS, N, V>(x, lse, a.out + r * a.os + first, n, tid);
    } else {
        best = block_best<THREADS>(best, best_slots, tid);
        const float shift = best.value == -__builtin_inff() ? 0.0f : best.value;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) sum += shifted_exp(x[k][e], shift);
        sum = block_sum<THREADS>(sum, sum_slots, tid);
        if (tid == 0) {
            float *p = a.part + ((int64_t)r * a.tiles + t) * 4;
            p[0] = best.value;
            p[1] = sum;
            p[2] = __int_as_float(best.index);
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
#define LOGITS_ROW_MAX 32768           // 1024 threads x 32 values
bool in_tiles(const dgl_logits_t *p) { return p->A > LOGITS_ROW_MAX; }

template <int TYPE, int THREADS, int N, int V> void launch_row(const LogitsArgs &a, hipStream_t s) {
    const int lds = a.history != nullptr ? a.A * 4 : 0;
    if (lds > 48 * 1024) dgl_max_dynamic_lds(reinterpret_cast<const void *>(&logits_row_kernel<TYPE, THREADS, N, V>), LOGITS_ROW_MAX * 4);
    hipLaunchKernelGGL((logits_row_kernel<TYPE, THREADS, N, V>), dim3(a.R), dim3(THREADS), lds, s, a);
}
// The smallest workgroup that holds a row at 4 to 32 values a thread (V = 1: rows that 16-byte accesses cannot take)
template <int TYPE, int V> int launch_logits(const LogitsArgs &a, hipStream_t s) {
    if (a.A <= 256) launch_row<TYPE, 64, 4 / V, V>(a, s);
    else if (a.A <= 1024) launch_row<TYPE, 256, 4 / V, V>(a, s);
    else if (a.A <= 4096) launch_row<TYPE, 256, 16 / V, V>(a, s);
    else if (a.A <= 8192) launch_row<TYPE, 1024, 8 / V, V>(a, s);
    else if (a.A <= 16384) launch_row<TYPE, 1024, 16 / V, V>(a, s);
    else if (a.A <= LOGITS_ROW_MAX) launch_row<TYPE, 1024, 32 / V, V>(a, s);
    else {
        const int lds = a.history != nullptr ? LOGITS_TILE * 4 : 0;
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
    const int bytes = p->dtype == DGL_DTYPE_F32 ? 4 : 2;
    const bool four = p->A % 4 == 0 && p->logits_stride % 4 == 0 && p->out_stride % 4 == 0 &&
                      (reinterpret_cast<uintptr_t>(p->logits) & (4 * bytes - 1)) == 0 && (reinterpret_cast<uintptr_t>(p->log_probs) & 15) == 0;
    hipStream_t s = (hipStream_t)stream;
    if (p->dtype == DGL_DTYPE_F32) return four ? launch_logits<0, 4>(a, s) : launch_logits<0, 1>(a, s);
    if (p->dtype == DGL_DTYPE_F16) return four ? launch_logits<1, 4>(a, s) : launch_logits<1, 1>(a, s);
    return four ? launch_logits<2, 4>(a, s) : launch_logits<2, 1>(a, s);
}
