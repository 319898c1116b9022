// The 4-bit paged KV cache: addressing and argument checks shared by the
// append, gather and attention kernels. The format is described at
// AmcuKv4Cache in aethermind_b200.h.
#pragma once
#include "../amcu_internal.h"
#include "common.cuh"

namespace amcu {

constexpr int kKv4Group = 64;            // elements that share a scale and a minimum
constexpr float kKv4StepMax = 4366.f;    // largest scale: 15 steps of it stay inside fp16
constexpr float kHalfMax = 65504.f;

// What the kernels need of AmcuKv4Cache / AmcuKv4Batch, by value.
struct Kv4View {
    uint8_t* kc;
    uint8_t* kp;
    uint8_t* vc;
    uint8_t* vp;
    int64_t cps, pps;          // bytes between pages
    const int32_t* table;
    int64_t table_stride;
    const int32_t* row_start;
    const int32_t* ctx_len;
    int32_t* status;
    int32_t num_pages, max_pages;
    int32_t n_seq, rows;
    int32_t page_shift;        // log2 of the page size
    int32_t nkv;
};

// First (row0) and count of sequence b's rows, kept inside [0, rows).
__device__ __forceinline__ void kv4_rows(const Kv4View& v, int b, int& row0, int& n) {
    int r0 = v.row_start[b], r1 = v.row_start[b + 1];
    r0 = min(max(r0, 0), v.rows);
    r1 = min(max(r1, r0), v.rows);
    row0 = r0;
    n = r1 - r0;
}

// Sequence of a row: the last b with row_start[b] <= row, found by the whole
// warp, 32 probes at a time (one load latency for up to 32 sequences, two for
// up to 1024). -1 where row_start does not cover the row.
__device__ __forceinline__ int kv4_find_seq(const Kv4View& v, int row) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = v.n_seq;   // the answer is in [lo, lo + n) or there is none
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int i = lane * step;
        const bool le = i < n && v.row_start[lo + i] <= row;
        const unsigned m = __ballot_sync(0xffffffffu, le);
        if (m == 0) return -1;
        const int at = (31 - __clz(m)) * step;
        lo += at;
        n = min(step, n - at);
    }
    return v.row_start[lo] <= row && row < v.row_start[lo + 1] ? lo : -1;
}

// Page of position pos of sequence b, or -1 (and the status word) where there is none.
__device__ __forceinline__ int kv4_page(const Kv4View& v, int b, int pos) {
    const int i = pos >> v.page_shift;
    int page = -1;
    if (pos >= 0 && i < v.max_pages) page = v.table[b * v.table_stride + i];
    if (page < 0 || page >= v.num_pages) {
        if (v.status) *v.status = (int32_t)AM_STATUS_OUT_OF_RANGE;
        return -1;
    }
    return page;
}

// Byte offsets of a head's row in the code and parameter planes.
template <int D>
__device__ __forceinline__ int64_t kv4_code_off(const Kv4View& v, int page, int head, int slot) {
    return (int64_t)page * v.cps + (((int64_t)head << v.page_shift) + slot) * (D / 2);
}
template <int D>
__device__ __forceinline__ int64_t kv4_param_off(const Kv4View& v, int page, int head, int slot) {
    return (int64_t)page * v.pps + (((int64_t)head << v.page_shift) + slot) * (D / 16);
}

// Positions in a call's flat list of work: sequence b has cost(b) items (the
// same in every thread), and the CTA wants item pick(all items). Every thread of the block
// (THREADS of them) calls this; it returns true in the one thread that found
// the sequence, with off = the item's place in sequence b. `total` is
// the same in all threads. Each thread adds up a run of sequences.
template <int THREADS, typename P, typename F>
__device__ __forceinline__ bool kv4_share(int n_seq, P pick, F cost, int64_t& total, int& b, int64_t& off) {
    __shared__ int64_t part[THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunk = (n_seq + THREADS - 1) / THREADS;
    const int lo = threadIdx.x * chunk, hi = min(lo + chunk, n_seq);
    int64_t mine = 0;
    for (int i = lo; i < hi; ++i) mine += cost(i);
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) part[warp] = incl;
    __syncthreads();
    int64_t base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) base += part[w];
        total += part[w];
    }
    off = pick(total) - (base + incl - mine);
    b = lo;
    if (off < 0 || off >= mine) return false;
    for (;; ++b) {
        const int64_t c = cost(b);
        if (off < c) return true;
        off -= c;
    }
}

// Rows of the call that no sequence has (row_start does not begin at 0 or does not
// end at `rows`) are zero in the attention's output. first, end: row_start's ends.
template <typename T, int THREADS>
__device__ __forceinline__ void kv4_zero_uncovered(const Kv4View& v, int first, int end, void* out, int64_t stride, int width) {
    first = min(max(first, 0), v.rows);
    end = min(max(end, first), v.rows);
    const int n = first + v.rows - end;
    if (n == 0) return;
    if (v.status && threadIdx.x == 0) *v.status = (int32_t)AM_STATUS_OUT_OF_RANGE;
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        T* o = static_cast<T*>(out) + (int64_t)(i < first ? i : end + (i - first)) * stride;
        for (int e = threadIdx.x; e < width; e += THREADS) o[e] = Act<T>::store(0.f);
    }
}

struct Kv4AttnParams {
    Kv4View v;
    const void* q;
    void* out;
    int64_t qs, os;
    int nq, grp;
    float scale;
    int vec;   // q and out rows start on 16-byte boundaries
};

// Prompts (bf16): whether their kernel is the faster one for this call, and its launch.
bool kv4_prefill_wanted(const Kv4View& v, int64_t grp);
am_status_code kv4_prefill_launch(const Kv4AttnParams& p, int64_t d, cudaStream_t s);

// Checks the cache and batch of a call and fills the view.
am_status_code kv4_check(const char* what, const AmcuKv4Cache& c, const AmcuKv4Batch& b, Kv4View* out);

}  // namespace amcu
