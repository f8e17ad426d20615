// Document ids of 64 bits to the 32-bit ones that the attention kernels compare (dgl_attention_t): the id of a document is the
// first position at which a key of the sequence has it, so equal and different stay equal and different whatever the values, and
// packed documents keep ascending ids (the kernels skip tiles by the range of a block's ids).
//
// One hash table per sequence, twice as many slots as keys, probed linearly: the keys' ids go in by compare-and-swap - only
// from the first token of a run of equal ids, where a first position has to be - and the least position of each by an integer
// minimum, so the result does not depend on the order.  Then both sides look theirs up.  No value returns to the host.  Bound by
// three launches: 15-16 us a call, from 6000 ids to 64 x 1001 and 200000 on either side.
#include "common.h"

namespace {

#define IDS_THREADS 256
#define IDS_NONE (-1ll)              // (negative ids are padding and never enter the table)

struct IdsArgs {
    const long long *doc_q, *doc_k;
    int64_t qs, ks;
    int B, Lq, Lk, log_slots;
    int *ids_q, *ids_k;
    unsigned long long *keys;        // [B][slots]
    int *first;                      // [B][slots]
};

__device__ __forceinline__ unsigned slot_of(unsigned long long id, int log_slots) {
    id ^= id >> 32;                  // (ids may differ in any of their bits)
    id *= 0x9E3779B97F4A7C15ull;     // odd, 2^64 / golden ratio
    id ^= id >> 29;
    id *= 0x9E3779B97F4A7C15ull;
    return (unsigned)(id >> (64 - log_slots));
}

__global__ __launch_bounds__(IDS_THREADS) void ids_clear_kernel(IdsArgs a) {
    const int64_t at = (int64_t)blockIdx.x * IDS_THREADS + threadIdx.x;
    if (at >= (int64_t)a.B << a.log_slots) return;
    a.keys[at] = (unsigned long long)IDS_NONE;
    a.first[at] = INT_MAX;
}

__global__ __launch_bounds__(IDS_THREADS) void ids_insert_kernel(IdsArgs a) {
    const int64_t at = (int64_t)blockIdx.x * IDS_THREADS + threadIdx.x;
    if (at >= (int64_t)a.B * a.Lk) return;
    const int64_t b = at / a.Lk;
    const int j = (int)(at % a.Lk);
    const long long *doc = a.doc_k + b * a.ks;
    const long long id = doc[j];
    if (id < 0 || (j > 0 && doc[j - 1] == id)) return;
    const unsigned mask = (1u << a.log_slots) - 1;
    unsigned long long *keys = a.keys + (b << a.log_slots);
    unsigned slot = slot_of((unsigned long long)id, a.log_slots);
    for (unsigned probe = 0; probe <= mask; ++probe, slot = (slot + 1) & mask) {     // (half of the slots stay empty)
        const unsigned long long was = atomicCAS(&keys[slot], (unsigned long long)IDS_NONE, (unsigned long long)id);
        if (was != (unsigned long long)IDS_NONE && was != (unsigned long long)id) continue;
        atomicMin(&a.first[(b << a.log_slots) + slot], j);
        return;
    }
}

__global__ __launch_bounds__(IDS_THREADS) void ids_look_up_kernel(IdsArgs a) {
    int64_t at = (int64_t)blockIdx.x * IDS_THREADS + threadIdx.x;
    const bool key = at < (int64_t)a.B * a.Lk;
    if (!key) at -= (int64_t)a.B * a.Lk;
    const int n = key ? a.Lk : a.Lq;
    if (!key && at >= (int64_t)a.B * a.Lq) return;
    const int64_t b = at / n;
    const long long id = key ? a.doc_k[b * a.ks + at % n] : a.doc_q[b * a.qs + at % n];
    int found = -1;
    if (id >= 0) {
        const unsigned mask = (1u << a.log_slots) - 1;
        const unsigned long long *keys = a.keys + (b << a.log_slots);
        unsigned slot = slot_of((unsigned long long)id, a.log_slots);
        for (unsigned probe = 0; probe <= mask; ++probe, slot = (slot + 1) & mask) {
            const unsigned long long k = keys[slot];
            if (k == (unsigned long long)id) found = a.first[(b << a.log_slots) + slot];
            if (k == (unsigned long long)id || k == (unsigned long long)IDS_NONE) break;
        }
    }
    (key ? a.ids_k : a.ids_q)[at] = found;
}

int log_slots_of(int Lk) {
    int s = 6;
    while ((1ll << s) < 2ll * Lk) ++s;
    return s;
}
int check_ids(int32_t B, int32_t Lq, int32_t Lk) {
    DGL_CHECK_ARG(B >= 1 && Lq >= 0 && Lk >= 0 && Lq <= DGL_ATTENTION_MAX_LENGTH && Lk <= DGL_ATTENTION_MAX_LENGTH, "B=%d Lq=%d Lk=%d", B, Lq, Lk);
    DGL_CHECK_ARG(((int64_t)B * ((int64_t)Lq + Lk) + ((int64_t)B << log_slots_of(Lk))) / IDS_THREADS < (1ll << 30), "too many rows");
    return DGL_OK;
}

}  // namespace

extern "C" int64_t dgl_document_ids_workspace_floats(int32_t B, int32_t Lk) {
    return check_ids(B, 0, Lk) != DGL_OK ? -1 : ((int64_t)B << log_slots_of(Lk)) * 3;
}

extern "C" int dgl_document_ids(int32_t B, int32_t Lq, int32_t Lk, const int64_t *doc_q, int64_t doc_q_stride, const int64_t *doc_k,
                                int64_t doc_k_stride, int32_t *ids_q, int32_t *ids_k, float *ws, dgl_stream_t stream) {
    if (int e = check_ids(B, Lq, Lk)) return e;
    DGL_CHECK_ARG((Lq == 0 || (doc_q != nullptr && ids_q != nullptr)) && (Lk == 0 || (doc_k != nullptr && ids_k != nullptr)), "NULL argument");
    DGL_CHECK_ARG(doc_q_stride >= 0 && doc_k_stride >= 0, "negative stride");
    DGL_CHECK_ARG(ws != nullptr && (reinterpret_cast<uintptr_t>(ws) & 7) == 0, "an 8-byte aligned workspace is needed");
    IdsArgs a{};
    a.doc_q = (const long long *)doc_q; a.doc_k = (const long long *)doc_k; a.qs = doc_q_stride; a.ks = doc_k_stride;
    a.B = B; a.Lq = Lq; a.Lk = Lk; a.log_slots = log_slots_of(Lk); a.ids_q = ids_q; a.ids_k = ids_k;
    const int64_t slots = (int64_t)B << a.log_slots;
    a.keys = reinterpret_cast<unsigned long long *>(ws);
    a.first = reinterpret_cast<int *>(a.keys + slots);
    hipStream_t s = (hipStream_t)stream;
    auto grid = [](int64_t n) { return dim3((unsigned)((n + IDS_THREADS - 1) / IDS_THREADS)); };
    hipLaunchKernelGGL(ids_clear_kernel, grid(slots), dim3(IDS_THREADS), 0, s, a);
    DGL_CHECK_LAUNCH("dgl_document_ids (clear)");
    if (Lk > 0) {
        hipLaunchKernelGGL(ids_insert_kernel, grid((int64_t)B * Lk), dim3(IDS_THREADS), 0, s, a);
        DGL_CHECK_LAUNCH("dgl_document_ids (insert)");
    }
    if (Lq + Lk > 0) {
        hipLaunchKernelGGL(ids_look_up_kernel, grid((int64_t)B * ((int64_t)Lq + Lk)), dim3(IDS_THREADS), 0, s, a);
        DGL_CHECK_LAUNCH("dgl_document_ids");
    }
    return DGL_OK;
}
