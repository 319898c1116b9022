// Token sampling: temperature, min-p, top-k, top-p and an inverse-CDF draw
// from a given uniform number (the definition is at amcu_sample).
//
// The weights are whole numbers of 2^-40, w = floor(expf(z) * 2^40): sums of
// them are exact in 64 bits (vocabularies up to 2^22), so the chosen token
// does not depend on how a row is split or in which order it is added up.
// Tokens are ordered by (|z| bits, index): z <= 0, so the bits of |z| grow as
// the logits fall.
#include "../amcu_internal.h"
#include "common.cuh"

namespace amcu {

struct SampleParams {
    const void* logits;
    int64_t stride, vocab;
    const float* uniform;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int64_t* out;
    float* prob;
};

constexpr int kSampleThreads = 1024;
constexpr float kSampleOne = 1099511627776.f;  // 2^40

// |z| of a logit, as orderable bits. NaN and -inf give +inf.
__device__ __forceinline__ uint32_t sample_key(float x, float mx, float t) {
    if (x == mx) return 0u;
    const float z = __fdiv_rn(__fsub_rn(x, mx), t);
    return z <= 0.f ? __float_as_uint(-z) & 0x7fffffffu : 0x7f800000u;  // NaN: comparison is false
}
__device__ __forceinline__ unsigned long long sample_weight(uint32_t key) {
    return (unsigned long long)__fmul_rn(expf(-__uint_as_float(key)), kSampleOne);
}

__device__ unsigned long long block_sum_u64(unsigned long long v) {
    __shared__ unsigned long long part[32];
    __shared__ unsigned long long all;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) part[w] = v;
    __syncthreads();
    if (w == 0) {
        v = part[lane];
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) all = v;
    }
    __syncthreads();
    return all;
}

// One CTA per row. A cut (key, index) keeps the tokens up to it in the order;
// it is found by bisection over the 64-bit composite (key, index).
template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_simple_kernel(SampleParams p) {
    typedef unsigned long long u64;
    __shared__ float red[32];
    __shared__ long long found;
    pdl_wait();
    pdl_trigger();
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.stride;
    float mx = -INFINITY;
    for (int64_t i = threadIdx.x; i < p.vocab; i += kSampleThreads) mx = fmaxf(mx, Act<T>::load(x[i]));
    mx = warp_max(mx);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
    __syncthreads();
    mx = warp_max(red[threadIdx.x & 31]);
    if (mx == -INFINITY) {
        if (threadIdx.x == 0) {
            p.out[row] = -1;
            if (p.prob) p.prob[row] = 0.f;
        }
        return;
    }
    float t = p.temperature ? p.temperature[row] : 1.f;
    long long k = p.top_k ? p.top_k[row] : 0;
    const float tp = p.top_p ? p.top_p[row] : 1.f, mp = p.min_p ? p.min_p[row] : 0.f;
    if (!(t > 0.f)) {
        t = 1.f;
        k = 1;
    }
    const u64 least = mp > 0.f ? (u64)ceil((double)mp * (double)kSampleOne) : 0;
    // count (what = 0) or mass (1) of the tokens up to the cut
    auto upto = [&](u64 cut, int what, u64 cap) {
        u64 s = 0;
        for (int64_t i = threadIdx.x; i < p.vocab; i += kSampleThreads) {
            const uint32_t key = sample_key(Act<T>::load(x[i]), mx, t);
            const u64 c = ((u64)key << 32) | (u64)i;
            const u64 w = sample_weight(key);
            if (c <= cut && c <= cap && w >= least) s += what ? w : 1;
        }
        return block_sum_u64(s);
    };
    const u64 kAll = ~0ull;
    u64 cut = kAll;
    for (int what = 0; what < 2; ++what) {  // top-k, then top-p of what that keeps
        u64 need;
        if (what == 0) {
            if (k <= 0 || (u64)k >= upto(kAll, 0, kAll)) continue;
            need = (u64)k;
        } else {
            if (!(tp < 1.f)) continue;
            const double want = ceil((double)tp * (double)upto(kAll, 1, cut));
            need = want < 1.0 ? 1 : (u64)want;
        }
        u64 lo = 0, hi = (0x7f800000ull << 32) | 0xffffffffull;  // least cut with upto(cut) >= need
        while (lo < hi) {
            const u64 mid = lo + (hi - lo) / 2;
            if (upto(mid, what, cut) >= need) hi = mid;
            else lo = mid + 1;
        }
        cut = min(cut, lo);
    }
    const u64 total = upto(kAll, 1, cut);
    const double ud = floor((double)p.uniform[row] * (double)total);
    u64 r = ud > 0.0 ? (u64)ud : 0;
    if (r >= total) r = total - 1;
    // first index whose running mass is above r
    u64 before = 0;
    if (threadIdx.x == 0) found = -1;
    for (int64_t i0 = 0; i0 < p.vocab; i0 += kSampleThreads) {
        const int64_t i = i0 + threadIdx.x;
        u64 w = 0;
        if (i < p.vocab) {
            const uint32_t key = sample_key(Act<T>::load(x[i]), mx, t);
            if ((((u64)key << 32) | (u64)i) <= cut) w = sample_weight(key);
            if (w < least) w = 0;
        }
        const u64 chunk = block_sum_u64(w);
        if (before + chunk > r) {  // the same in every thread: scan this chunk
            __shared__ u64 ws[kSampleThreads];
            ws[threadIdx.x] = w;
            __syncthreads();
            if (threadIdx.x == 0) {
                for (int j = 0; j < kSampleThreads; ++j) {
                    before += ws[j];
                    if (before > r) {
                        p.out[row] = i0 + j;
                        if (p.prob) p.prob[row] = (float)ws[j] / (float)total;
                        break;
                    }
                }
            }
            return;
        }
        before += chunk;
    }
}

}  // namespace amcu

using namespace amcu;

extern "C" am_status_code amcu_sample(const AmcuSampleArgs* a, void* stream) {
    clear_error();
    AMCU_REQUIRE(a != nullptr, "amcu_sample: null args");
    AMCU_REQUIRE(a->rows >= 0 && a->rows <= INT32_MAX, "amcu_sample: bad rows");
    AMCU_REQUIRE(a->vocab > 0 && a->vocab <= (1 << 22), "amcu_sample: vocab must be in [1, 2^22]");
    AMCU_REQUIRE(a->row_stride == 0 || a->row_stride >= a->vocab || a->rows <= 1, "amcu_sample: row_stride below vocab");
    AMCU_REQUIRE(a->dtype == AMCU_F32 || a->dtype == AMCU_BF16, "amcu_sample: dtype must be f32 or bf16");
    if (a->rows == 0) return AM_STATUS_OK;
    AMCU_REQUIRE(a->logits && a->uniform && a->out_index, "amcu_sample: null pointer");
    SampleParams p;
    p.logits = a->logits;
    p.stride = a->row_stride ? a->row_stride : a->vocab;
    p.vocab = a->vocab;
    p.uniform = a->uniform;
    p.temperature = a->temperature;
    p.top_k = a->top_k;
    p.top_p = a->top_p;
    p.min_p = a->min_p;
    p.out = a->out_index;
    p.prob = a->out_prob;
    const dim3 grid((unsigned)a->rows), block(kSampleThreads);
    a->dtype == AMCU_F32 ? launch_pdl(sample_simple_kernel<float>, grid, block, 0, as_stream(stream), p)
                         : launch_pdl(sample_simple_kernel<__nv_bfloat16>, grid, block, 0, as_stream(stream), p);
    return check_launch("amcu_sample");
}
