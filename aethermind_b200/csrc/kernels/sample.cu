// Token sampling: temperature, min-p, top-k, top-p and an inverse-CDF draw
// from a given uniform number (the definition is at amcu_sample).
//
// The weights are whole numbers of 2^-40, w = floor(expf(z) * 2^40): sums of
// them are exact in 64 bits (vocabularies up to 2^22), so the chosen token
// does not depend on how a row is split or in which order it is added up.
// Tokens are ordered by (|z| bits, index): z <= 0, so the bits of |z| grow as
// the logits fall.
#include <cooperative_groups.h>

#include "../amcu_internal.h"
#include "common.cuh"

namespace amcu {

struct SampleParams {
    const void* logits;
    int64_t stride, vocab, rows;
    int64_t ahead;  // rows between one that runs and the one that takes its place
    const float* uniform;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int64_t* out;
    float* prob;
};

typedef unsigned long long u64;
namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 256;
constexpr int kSampleList = kSampleThreads;       // most candidates that are sorted
constexpr int kSampleWarpList = 64;               // of one warp's tokens
constexpr int kSampleQueue = 128;                 // tokens of a cut's bin that a warp keeps the indices of
constexpr int kSamplePlace = 9;                   // bits of a place among them
constexpr int kSampleTop = 256;                   // largest top-k whose tokens are gathered
constexpr int kSampleSlice = 16384;               // most logits that a CTA keeps in shared memory
constexpr float kSampleOne = 1099511627776.f;     // 2^40
constexpr float kSampleBinScale = kSampleBins / 28.f;  // weights end at z = -27.7
constexpr uint32_t kSampleNever = 0x7f800000u;    // key of a masked token

// |z| of a logit, as orderable bits. NaN and -inf give +inf.
__device__ __forceinline__ uint32_t sample_key(float x, float mx, float t) {
    if (x == mx) return 0u;
    const float z = __fdiv_rn(__fsub_rn(x, mx), t);
    return z <= 0.f ? __float_as_uint(-z) & 0x7fffffffu : kSampleNever;  // NaN: comparison is false
}
// The same for rows in whose whole range no step leaves the normal numbers
// (sample_plain): two corrections of the quotient by its exact remainder with a
// correctly rounded reciprocal give the correctly rounded quotient (Markstein,
// IBM J. Res. Dev. 34, 1990), without a branch.
__device__ __forceinline__ uint32_t sample_key_plain(float x, float mx, float t, float inv) {
    const float a = __fsub_rn(x, mx);
    float z = __fmul_rn(a, inv);
    z = __fmaf_rn(__fmaf_rn(-z, t, a), inv, z);
    z = __fmaf_rn(__fmaf_rn(-z, t, a), inv, z);
    return __float_as_uint(z) & 0x7fffffffu;  // masked tokens: NaN, whose weight is 0 and whose bin is the last
}
// The largest logit is not tiny (differences from it are then 0 or above 2^-85)
// nor infinite, and the temperature is within 2^+-40.
__device__ __forceinline__ bool sample_plain(float mx, float t) {
    return fabsf(mx) >= 0x1p-60f && fabsf(mx) <= 0x1p120f && t >= 0x1p-40f && t <= 0x1p40f;
}
// floor(e * 2^40) of an e in [0, 1], its upper 21 and lower 20 bits, each added to
// a sum together with kSampleHi, kSampleLo (an addition that truncates at 2^-20,
// one of the exact rest at 2^-40; 64-bit conversions and shifts are slow).
constexpr uint32_t kSampleHi = 0x41000000u, kSampleLo = 0x37000000u;  // 8 and 2^-17
__device__ __forceinline__ void sample_split(float e, uint32_t& hi, uint32_t& lo) {
    const float a = __fadd_rz(e, 8.f);
    hi += __float_as_uint(a);
    lo += __float_as_uint(__fadd_rz(__fsub_rn(e, __fsub_rn(a, 8.f)), 0x1p-17f));
}
__device__ __forceinline__ u64 sample_whole(float e) {
    uint32_t hi = 0u - kSampleHi, lo = 0u - kSampleLo;
    sample_split(e, hi, lo);
    return ((u64)hi << 20) + lo;
}
__device__ __forceinline__ float sample_exp(uint32_t key) { return expf(-__uint_as_float(key)); }
__device__ __forceinline__ u64 sample_weight(uint32_t key) { return sample_whole(sample_exp(key)); }
// Position of a key on a scale of 256 bins (a weight above 0 is below 254); bin
// and sub-bin are monotone in the key.
__device__ __forceinline__ float sample_place(uint32_t key) { return __fmul_rn(__uint_as_float(key), kSampleBinScale); }
__device__ __forceinline__ int sample_bin(float place) {  // truncated by an addition; NaN is in the last bin
    return (int)(__float_as_uint(__fadd_rz(fminf(place, (float)(kSampleBins - 1)), 0x1p23f)) - 0x4b000000u);
}
__device__ __forceinline__ int sample_sub(float place, int bin) {
    return min((int)__fmul_rn(__fsub_rn(place, (float)bin), 256.f), kSampleBins - 1);
}

// A weight's bits for 32-bit sums (64-bit shared atomics are far slower): two
// fields of 20 bits and 21 for slices of up to 2^14 tokens, three of 14 for slices
// up to 2^18. Lanes with the same low bits share a copy of the histogram, which
// so gets 2^11 tokens (2^16) at most.
template <bool kRes> struct SampleSplit {
    static constexpr int kFields = kRes ? 2 : 3, kBits = kRes ? 20 : 14, kCopies = kRes ? 8 : 4;
    static __device__ __forceinline__ int at(int field, int bin, int copy) {
        return (field * kSampleBins + bin) * kCopies + copy;
    }
};
constexpr int kSampleHist = 2 * kSampleBins * 8;

struct SampleShared {
    u64 mass[2][kSampleBins];  // of the tokens in a bin: weights, or their number
    uint32_t count[2][kSampleBins];
    float group[kSampleThreads];       // maxima of the threads, or of 2, 4 or 8 neighbours
    u64 list[kSampleWarps][kSampleWarpList];  // each warp's candidates
    uint32_t n_list[kSampleWarps];
    uint32_t n_queue[kSampleWarps];
    union {
        alignas(16) uint32_t hist[kSampleHist];
        struct {
            u64 all[kSampleList];        // every CTA's
            u64 weight[kSampleList];     // by place: weights of the kept
            u64 tmp[kSampleList];
        };
    };
    uint32_t queue[kSampleWarps][kSampleQueue];
    u64 part[kSampleWarps];
    u64 scan[kSampleBins / 32];
    u64 xchg[2];
    uint32_t kmin, kmax;
    u64 top, cut, before;
    uint32_t members;
    int bin;
};

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_max_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ u64 warp_scan_u64(u64 v) {  // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 z = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += z;
    }
    return v;
}

// What the row's CTAs do together: rank r of C holds tokens [r * slice, ...).
struct SampleTeam {
    SampleShared* s;
    cg::cluster_group cl;
    int rank, C, turn;

    template <typename V>
    __device__ __forceinline__ V at(int r, const V* p) { return *cl.map_shared_rank(const_cast<V*>(p), r); }

    // Sum over the cluster; `before`: of the ranks below this one. One cluster barrier.
    __device__ u64 sum(u64 v, u64* before = nullptr) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        v = warp_sum_u64(v);
        if (lane == 0) s->part[w] = v;
        __syncthreads();
        if (w == 0) {
            v = warp_sum_u64(lane < kSampleWarps ? s->part[lane] : 0);
            if (lane == 0) s->xchg[turn & 1] = v;
        }
        return gather(before);
    }
    // The same once xchg[turn & 1] holds this CTA's value.
    __device__ u64 gather(u64* before) {
        const int lane = threadIdx.x & 31;
        cl.sync();
        const u64 x = lane < C ? at(lane, &s->xchg[turn & 1]) : 0;
        ++turn;
        if (before) *before = warp_sum_u64(lane < rank ? x : 0);
        return warp_sum_u64(x);
    }

    // Every warp's list (in index order, as the warps and CTAs are) into all[],
    // members as (key, index, place in all[]); returns their number, or -1 where
    // they are too many.
    __device__ int collect() {
        cl.sync();
        int n = 0;
        for (int first = 0; first < C * kSampleWarps; first += kSampleThreads) {  // one list per thread (C <= 16: once)
            const int q = first + threadIdx.x, r = q / kSampleWarps;
            const int m = q < C * kSampleWarps ? (int)at(r, &s->n_list[q % kSampleWarps]) : 0;
            u64 all;
            const bool bad = __syncthreads_or(m > kSampleWarpList);
            int o = n + (int)scan((u64)m, all) - m;
            n += (int)all;
            if (bad || n > kSampleList) return -1;
            for (int i = 0; i < m; ++i, ++o) {
                const u64 c = at(r, &s->list[q % kSampleWarps][i]);
                s->all[o] = (c & 0xffffffff00000000ull) | ((c & 0x3fffffu) << kSamplePlace) | (u64)o;
            }
        }
        __syncthreads();
        return n;
    }

    // all[0 .. m) in ascending order, one per thread (~0 past the end): up to 128
    // by counting the smaller ones; more are put into the 256 bins of z first and
    // counted within their bin (33 rows of 509 tokens: 9.9 us a call, by a bitonic
    // sort 12.4).
    __device__ u64 sorted(int m) {
        const int tid = threadIdx.x;
        const u64 me = tid < m ? s->all[tid] : ~0ull;
        if (m <= 128) {
            if (tid < m) {
                int less = 0;
#pragma unroll 8
                for (int j = 0; j < m; ++j) less += s->all[j] < me;
                s->tmp[less] = me;
            }
            __syncthreads();
            return tid < m ? s->tmp[tid] : ~0ull;
        }
        uint32_t* const cnt = s->count[0];
        uint32_t* const first = s->count[1];
        if (tid < kSampleBins) cnt[tid] = 0;
        __syncthreads();
        const int bin = sample_bin(sample_place((uint32_t)(me >> 32)));
        const uint32_t at_ = tid < m ? atomicAdd(&cnt[bin], 1u) : 0u;
        __syncthreads();
        const uint32_t c = tid < kSampleBins ? cnt[tid] : 0u;
        u64 all;
        const u64 inc = scan(c, all);
        if (tid < kSampleBins) first[tid] = (uint32_t)inc - c;
        __syncthreads();
        if (tid < m) s->tmp[first[bin] + at_] = me;
        __syncthreads();
        if (tid < m) {
            const uint32_t lo = first[bin], n = cnt[bin];
            uint32_t less = 0;
#pragma unroll 4
            for (uint32_t j = 0; j < n; ++j) less += s->tmp[lo + j] < me;
            s->weight[lo + less] = me;
        }
        __syncthreads();
        return tid < m ? s->weight[tid] : ~0ull;
    }

    // Running total of v over the block's threads, and the block's.
    __device__ u64 scan(u64 v, u64& all) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const u64 inc = warp_scan_u64(v);
        if (lane == 31) s->part[warp] = inc;
        __syncthreads();
        u64 b = 0;
        all = 0;
#pragma unroll
        for (int w = 0; w < kSampleWarps; ++w) {
            const u64 y = s->part[w];
            if (w < warp) b += y;
            all += y;
        }
        __syncthreads();
        return b + inc;
    }
};

// One cluster per row, its CTAs each holding a contiguous slice of the row in
// shared memory as fp32 (kRes; larger vocabularies read the logits again).
//
// * Greedy rows, top-k 1: the (logit, index) maximum is the answer.
// * top-k up to kSampleTop: the k-th largest of the maxima of 512 to 1024 groups
//   of tokens bounds the k-th largest token from below, so their histogram gives
//   a threshold that little more than k tokens pass; the first CTA sorts those and
//   does the rest alone. Rows of at most 512 tokens go there at once.
// * Otherwise a cut is found by a histogram of 256 bins of z, one of 256 parts
//   of the bin that it falls in, and sorting what is in that part; equal keys by
//   the thousand (bf16 logits) are told apart by their index alone.
//
// Bound by latency (exchanges of the cluster, barriers) and, without top-k, by
// the instructions per token (22 for the mass, 30 and two shared atomics for the
// histogram). The next row of these SMs is fetched into L2 meanwhile. 192 fp32
// rows of 128256: 38 us if all are greedy, 80 with top-k 40, 85 with the
// temperature alone, 173 with top-p 0.95, 162 with top-k 1000. Before the
// division without a branch, split sums, copies of the histogram and the
// drawn run walked by a warp: 50, 91, 139, 265, 227.
template <typename T, bool kRes>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleParams p, int slice) {
    using Split = SampleSplit<kRes>;
    extern __shared__ __align__(16) float xs[];
    __shared__ SampleShared s;
    SampleTeam team{&s, cg::this_cluster(), 0, 0, 0};
    team.rank = (int)team.cl.block_rank();
    team.C = (int)team.cl.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / team.C;
    pdl_wait();
    pdl_trigger();

    const int64_t i0 = (int64_t)team.rank * slice;
    const int n = (int)max((int64_t)0, min((int64_t)slice, p.vocab - i0));
    const T* x = static_cast<const T*>(p.logits) + row * p.stride + i0;
    float t = p.temperature ? p.temperature[row] : 1.f;
    int64_t k = p.top_k ? p.top_k[row] : 0;
    const float tp = p.top_p ? p.top_p[row] : 1.f, mp = p.min_p ? p.min_p[row] : 0.f;
    const float un = p.uniform[row];
    // the least e whose weight floor(e * 2^40) is above 0 and reaches min_p
    const float least = mp > 0.f ? __double2float_ru(fmax(ceil((double)fminf(mp, 1.f) * (double)kSampleOne), 1.0) / (double)kSampleOne)
                                 : 1.f / kSampleOne;

    // Place of the draw in a mass of `total` > 0.
    auto draw = [&](u64 total) -> u64 {
        const double ud = floor((double)un * (double)total);
        const u64 r = ud > 0.0 ? (u64)ud : 0;
        return r >= total ? total - 1 : r;
    };
    // list_if: what f(i) gives of the CTA's tokens, without the kNone, into the
    // warps' lists in index order; n_list counts them, also past the end. A warp
    // has a run of tokens, a lane four neighbours at a time; quick(i) may rule out
    // tokens i .. i + 3 (i a multiple of 4) together.
    constexpr u64 kNone = ~0ull;
    const int seg = ((n + 4 * kSampleWarps - 1) / (4 * kSampleWarps)) * 4, seg_lo = min(warp * seg, n), seg_hi = min(seg_lo + seg, n);
    auto list_if = [&](auto quick, auto f) {
        uint32_t c = 0;
#pragma unroll 2
        for (int at = seg_lo; at < seg_hi; at += 128) {
            const int i = at + 4 * lane;
            const bool maybe = i < seg_hi && quick(i);
            if (__ballot_sync(0xffffffffu, maybe) == 0) continue;
            u64 y[4];
            uint32_t mine = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = maybe && i + e < seg_hi ? f(i + e) : kNone;
                mine += y[e] != kNone;
            }
            if (__ballot_sync(0xffffffffu, mine) == 0) continue;
            uint32_t o = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t z = __shfl_up_sync(0xffffffffu, o, d);
                if (lane >= d) o += z;
            }
            const uint32_t all = __shfl_sync(0xffffffffu, o, 31);
            o += c - mine;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (y[e] != kNone) {
                    if (o < kSampleWarpList) s.list[warp][o] = y[e];
                    ++o;
                }
            c += all;
        }
        if (lane == 0) s.n_list[warp] = c;
    };
    // A thread has a run of an odd number of tokens (odd: neighbours in different banks).
    const int run = ((n + kSampleThreads - 1) / kSampleThreads) | 1, run_lo = min(tid * run, n), run_hi = min(run_lo + run, n);

    // ---- the row's largest logit and its first index: (order key, ~index)
    float mx = -INFINITY;
    int at = 0;
    {
        constexpr int V = 16 / sizeof(T);
        const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
        const int nv = vec ? n / V : 0;
#pragma unroll 4
        for (int j = tid; j < nv; j += kSampleThreads) {  // a thread's indices ascend
            const uint4 y = ld_stream_u4(x + (int64_t)j * V);
            const uint32_t w[4] = {y.x, y.y, y.z, y.w};
            float f[V];
#pragma unroll
            for (int e = 0; e < V; ++e)
                f[e] = sizeof(T) == 4 ? __uint_as_float(w[e * 4 / V]) : __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
            float top = f[0];
#pragma unroll
            for (int e = 1; e < V; ++e) top = fmaxf(top, f[e]);
            if (kRes) {
#pragma unroll
                for (int e = 0; e < V; e += 4)
                    *reinterpret_cast<float4*>(xs + j * V + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
            }
            if (top > mx) {  // a few times per thread
                mx = top;
#pragma unroll
                for (int e = V - 1; e >= 0; --e)
                    if (f[e] == top) at = j * V + e;
            }
        }
#pragma unroll 4
        for (int i = nv * V + tid; i < n; i += kSampleThreads) {
            const float f = Act<T>::load(x[i]);
            if (kRes) xs[i] = f;
            if (f > mx) {
                mx = f;
                at = i;
            }
        }
        if (kRes && tid < ((-n) & 3)) xs[n + tid] = -INFINITY;
        if (tid == 0 && vec && n * (int)sizeof(T) >= 16 && row + p.ahead < p.rows) {
            const T* next = x + p.ahead * p.stride;
            if ((reinterpret_cast<uintptr_t>(next) & 15) == 0)
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(next), "r"(n * (int)sizeof(T) & ~15) : "memory");
        }
        u64 best = mx > -INFINITY ? ((u64)float_order_key(mx + 0.f) << 32) | (0xffffffffu - (uint32_t)(i0 + at)) : 0;
        best = warp_max_u64(best);
        if (lane == 0) s.part[warp] = best;
        float gm = mx;  // 512 to 1024 group maxima in the cluster
        const int gs = min(team.C, 8);
        for (int o = 1; o < gs; o *= 2) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
        if ((tid & (gs - 1)) == 0) s.group[tid / gs] = gm;
        if (tid < kSampleBins) s.count[0][tid] = 0;
        __syncthreads();
        if (warp == 0) {
            best = warp_max_u64(lane < kSampleWarps ? s.part[lane] : 0);
            if (lane == 0) s.top = best;
        }
        team.cl.sync();
        best = warp_max_u64(lane < team.C ? team.at(lane, &s.top) : 0);
        if (best == 0 || !(t > 0.f) || k == 1) {  // nothing to draw from, or nothing to choose
            if (team.rank == 0 && tid == 0) {
                p.out[row] = best ? (int64_t)(0xffffffffu - (uint32_t)best) : -1;
                if (p.prob) p.prob[row] = best ? 1.f : 0.f;
            }
            team.cl.sync();  // nobody leaves while its maximum is read
            return;
        }
        const uint32_t o = (uint32_t)(best >> 32);
        const float all = __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
        // ---- few tokens to keep (those above the k-th largest group maximum), or few tokens at all
        const bool few = p.vocab <= kSampleList;
        if (few || (k > 0 && k <= kSampleTop)) {
            float edge = -INFINITY;
            int bin = kSampleBins - 1;
            if (!few) {
                const int per = kSampleThreads / gs, groups = per * team.C;
                for (int q = tid; q < groups; q += kSampleThreads) {
                    const uint32_t key = sample_key(team.at(q / per, &s.group[q % per]), all, t);
                    if (key < kSampleNever) atomicAdd(&s.count[0][sample_bin(sample_place(key))], 1u);
                }
                if (tid == 0) s.bin = kSampleBins - 1;
                __syncthreads();
                const u64 c = tid < kSampleBins ? s.count[0][tid] : 0;
                u64 any;
                const u64 inc = team.scan(c, any);
                if (inc - c < (u64)k && inc >= (u64)k) s.bin = tid;
                __syncthreads();
                bin = s.bin;
                // the bin's far edge as a logit, with room for the roundings: a quick test before the exact one
                if (bin < kSampleBins - 1 && fabsf(all) < INFINITY)
                    edge = all - ((float)(bin + 1) / kSampleBinScale * t * 1.0001f + 1e-6f * fabsf(all));
            }
            list_if([&](int i) -> bool {  // four neighbours: does any of them reach the edge?
                if (!kRes || i + 4 > n) return true;
                const float4 y = *reinterpret_cast<const float4*>(xs + i);
                return fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)) >= edge;
            }, [&](int i) -> u64 {
                const float f = kRes ? xs[i] : Act<T>::load(x[i]);
                if (!(f >= edge)) return kNone;
                const uint32_t key = sample_key(f, all, t);
                if (key >= kSampleNever || sample_bin(sample_place(key)) > bin || !(sample_exp(key) >= least)) return kNone;
                return ((u64)key << 32) | (u64)(i0 + i);
            });
            const int m = team.collect();
            if (m >= 0) {
                team.cl.sync();  // the lists are read: the others may leave
                if (team.rank) return;
                const u64 me = team.sorted(m);
                const u64 w = tid < m && (k <= 0 || tid < k) ? sample_weight((uint32_t)(me >> 32)) : 0;
                u64 total;
                const u64 before = team.scan(w, total) - w;
                bool keep = w > 0;
                if (tp < 1.f) {
                    const double want = ceil((double)tp * (double)total);
                    keep = keep && before < (want < 1.0 ? 1 : (u64)want);
                }
                if (tid < m) s.weight[(uint32_t)me & (kSampleList - 1)] = keep ? w : 0;
                __syncthreads();
                const u64 mine = tid < m ? s.weight[tid] : 0;
                const u64 inc = team.scan(mine, total);
                const u64 r = draw(total);
                if (inc - mine <= r && r < inc) {
                    p.out[row] = (int64_t)((uint32_t)s.all[tid] >> kSamplePlace);
                    if (p.prob) p.prob[row] = (float)mine / (float)total;
                }
                return;
            }
        }
        mx = all;
    }

    // ---- the general case
    team.cl.sync();  // lists of an attempt above are read
    bool keyed = false;  // xs holds keys: the first histogram makes them
    const bool plain = sample_plain(mx, t);
    const float inv = __frcp_rn(t);
    if (kRes && !plain) {
        for (int i = tid; i < ((n + 3) & ~3); i += kSampleThreads) xs[i] = __uint_as_float(sample_key(xs[i], mx, t));
        keyed = true;
        __syncthreads();
    }
    auto key_of = [&](int i) -> uint32_t {
        if (kRes) return keyed ? __float_as_uint(xs[i]) : sample_key_plain(xs[i], mx, t, inv);
        const float f = Act<T>::load(x[i]);
        return plain ? sample_key_plain(f, mx, t, inv) : sample_key(f, mx, t);
    };
    bool any_cut = false;
    u64 cut = ~0ull;  // tokens up to it in the order of (key, index) are kept
    auto comp_of = [&](uint32_t key, int i) -> u64 { return ((u64)key << 32) | (u64)(i0 + i); };
    auto exp_of = [&](uint32_t key, int i) -> float {  // 0 where the token is not kept
        if (any_cut && comp_of(key, i) > cut) return 0.f;
        const float e = sample_exp(key);
        return e >= least ? e : 0.f;
    };
    auto weight_of = [&](uint32_t key, int i) -> u64 { return sample_whole(exp_of(key, i)); };
    // The kept mass of the thread's run.
    auto run_mass = [&]() -> u64 {
        const uint32_t c = (uint32_t)(run_hi - run_lo);
        uint32_t hi = 0u - c * kSampleHi, lo = 0u - c * kSampleLo;
        if (kRes && !keyed) {
#pragma unroll 4
            for (int i = run_lo; i < run_hi; ++i) sample_split(exp_of(sample_key_plain(xs[i], mx, t, inv), i), hi, lo);
        } else {
#pragma unroll 4
            for (int i = run_lo; i < run_hi; ++i) sample_split(exp_of(key_of(i), i), hi, lo);
        }
        return ((u64)hi << 20) + lo;  // runs are 512 tokens at most
    };
    // scan_runs: the sum over the thread's run, those of the threads before it, and
    // the CTA's total in xchg; walk: the first token of the CTA with a running f
    // above `target`, given to `hit` by the lane that finds it (`before` and `mine`
    // as scan_runs left them, plus what other CTAs have): the warp whose thread's
    // run it is in goes through that run together.
    auto scan_runs = [&](auto f, u64& mine, u64& before) {
        mine = f();
        u64 all;
        before = team.scan(mine, all) - mine;
        if (tid == 0) s.xchg[team.turn & 1] = all;
    };
    auto walk = [&](auto f, u64 before, u64 mine, u64 target, auto hit) {
        const uint32_t owner = __ballot_sync(0xffffffffu, before <= target && target - before < mine);
        if (!owner) return;
        const int src = __ffs(owner) - 1;
        const int lo = __shfl_sync(0xffffffffu, run_lo, src), hi = __shfl_sync(0xffffffffu, run_hi, src);
        before = __shfl_sync(0xffffffffu, before, src);
        for (int at = lo; at < hi; at += 32) {
            const u64 v = at + lane < hi ? f(at + lane) : 0, inc = before + warp_scan_u64(v);
            if (inc - v <= target && target < inc) hit(at + lane);
            before = __shfl_sync(0xffffffffu, inc, 31);
            if (target < before) return;
        }
    };

    bool known = false;  // whether `local`, summed over the CTA, is its kept mass
    u64 local = 0;
    // The least cut at which the kept tokens' count (by_mass false) or mass
    // reaches what is asked for: k tokens, or top_p of the mass.
    auto find_cut = [&](bool by_mass) {
        u64 before = 0, need = 0;   // before: of the tokens in earlier bins
        int bins[2] = {0, 0};
        uint32_t members = 0;
        int queued = -1;  // this warp's tokens of the first level's bin, in s.queue; -1: too many
        for (int level = 0; level < 2; ++level) {
            for (int j = tid; j < kSampleHist / 4; j += kSampleThreads) reinterpret_cast<uint4*>(s.hist)[j] = make_uint4(0, 0, 0, 0);
            if (tid < kSampleBins) s.count[level][tid] = 0;
            if (lane == 0) s.n_queue[warp] = 0;
            __syncthreads();
            const float bin_lo = (float)bins[0], bin_hi = bin_lo + 1.f;
            const int copy = lane & (Split::kCopies - 1);
            auto add = [&](int i, uint32_t key) {
                const float place = sample_place(key);
                if (level == 1 && !(place >= bin_lo && place < bin_hi)) return;
                const int bin = level == 1 ? sample_sub(place, bins[0]) : sample_bin(place);
                const float e = exp_of(key, i);
                if (!(e > 0.f)) return;
                if (by_mass && kRes) {
                    uint32_t hi = 0u - kSampleHi, lo = 0u - kSampleLo;
                    sample_split(e, hi, lo);
                    atomicAdd(&s.hist[Split::at(0, bin, copy)], lo);
                    if (hi) atomicAdd(&s.hist[Split::at(1, bin, copy)], hi);
                    if (level == 1) atomicAdd(&s.count[1][bin], 1u);
                } else if (by_mass) {
                    const u64 w = sample_whole(e);
                    constexpr uint32_t low = (1u << Split::kBits) - 1;
                    atomicAdd(&s.hist[Split::at(0, bin, copy)], (uint32_t)w & low);
#pragma unroll
                    for (int f = 1; f < Split::kFields; ++f) {
                        const uint32_t v = (uint32_t)(w >> (f * Split::kBits)) & (f < Split::kFields - 1 ? low : ~0u);
                        if (v) atomicAdd(&s.hist[Split::at(f, bin, copy)], v);
                    }
                    if (level == 1) atomicAdd(&s.count[1][bin], 1u);
                } else {
                    atomicAdd(&s.hist[Split::at(0, bin, copy)], 1u);
                }
            };
            if (level == 0) {
                if (kRes) {
                    for (int i = 4 * tid; i < n; i += 4 * kSampleThreads) {
                        uint4 y = *reinterpret_cast<const uint4*>(xs + i);
                        if (!keyed) {
                            y.x = sample_key_plain(__uint_as_float(y.x), mx, t, inv);
                            y.y = sample_key_plain(__uint_as_float(y.y), mx, t, inv);
                            y.z = sample_key_plain(__uint_as_float(y.z), mx, t, inv);
                            y.w = sample_key_plain(__uint_as_float(y.w), mx, t, inv);
                            *reinterpret_cast<uint4*>(xs + i) = y;
                        }
                        add(i, y.x);
                        add(i + 1, y.y);
                        add(i + 2, y.z);
                        add(i + 3, y.w);
                    }
                    keyed = true;
                } else {
#pragma unroll 2
                    for (int i = tid; i < n; i += kSampleThreads) add(i, key_of(i));
                }
            } else {
                // the bin's tokens first, so that they are looked at by full warps
                auto put = [&](int i, uint32_t key) {
                    const float place = sample_place(key);
                    if (!(place >= bin_lo && place < bin_hi)) return;
                    const uint32_t o = atomicAdd(&s.n_queue[warp], 1u);
                    if (o < kSampleQueue) s.queue[warp][o] = (uint32_t)i;
                };
                if (kRes) {
                    const uint32_t lo = __float_as_uint(bin_lo / kSampleBinScale * 0.999999f);  // a little wider than the bin
                    const uint32_t span = __float_as_uint(bin_hi / kSampleBinScale * 1.000001f) - lo;
#pragma unroll 4
                    for (int i = seg_lo + 4 * lane; i < seg_hi; i += 128) {
                        const uint4 y = *reinterpret_cast<const uint4*>(xs + i);
                        if (min(min(y.x - lo, y.y - lo), min(y.z - lo, y.w - lo)) > span) continue;
                        put(i, y.x);
                        put(i + 1, y.y);
                        put(i + 2, y.z);
                        put(i + 3, y.w);
                    }
                } else {
                    for (int i = seg_lo + lane; i < seg_hi; i += 32) put(i, key_of(i));
                }
                __syncwarp();
                const int c = (int)s.n_queue[warp];
                queued = c <= kSampleQueue ? c : -1;
                if (queued >= 0)
                    for (int j = lane; j < queued; j += 32) add((int)s.queue[warp][j], key_of((int)s.queue[warp][j]));
                else
                    for (int i = seg_lo + lane; i < seg_hi; i += 32) add(i, key_of(i));
            }
            __syncthreads();
            if (tid < kSampleBins) {
                u64 sum = 0;
#pragma unroll
                for (int f = 0; f < Split::kFields; ++f) {
                    u64 part = 0;
#pragma unroll
                    for (int c = 0; c < Split::kCopies; c += 4) {
                        const uint4 y = *reinterpret_cast<const uint4*>(&s.hist[Split::at(f, tid, c)]);
                        part += (u64)y.x + y.y + y.z + y.w;
                    }
                    sum += part << (f * Split::kBits);
                }
                s.mass[level][tid] = sum;
            }
            team.cl.sync();
            u64 v = 0, cnt = 0;
            if (tid < kSampleBins) {
#pragma unroll 4
                for (int r = 0; r < team.C; ++r) {
                    v += team.at(r, &s.mass[level][tid]);
                    if (by_mass && level == 1) cnt += team.at(r, &s.count[1][tid]);
                }
                if (!by_mass) cnt = v;
            }
            const u64 inc = warp_scan_u64(v);
            if (lane == 31 && warp < kSampleBins / 32) s.scan[warp] = inc;
            __syncthreads();
            if (level == 0) {
                u64 all = 0;
                for (int w = 0; w < kSampleBins / 32; ++w) all += s.scan[w];
                if (by_mass) {
                    const double want = ceil((double)tp * (double)all);
                    need = want < 1.0 ? 1 : (u64)want;
                } else {
                    need = (u64)k;
                    if (need >= all) {  // nothing to cut
                        team.cl.sync();  // the masses are read
                        return;
                    }
                }
            }
            if (tid < kSampleBins) {
                u64 b = before;
                for (int w = 0; w < warp; ++w) b += s.scan[w];
                if (b + inc - v < need && need <= b + inc) {
                    s.bin = tid;
                    s.before = b + inc - v;
                    s.members = (uint32_t)cnt;
                }
            }
            __syncthreads();
            bins[level] = s.bin;
            before = s.before;
            members = s.members;
        }
        const float bin_lo = (float)bins[0], bin_hi = bin_lo + 1.f;
        auto in_bin = [&](int i) -> u64 {  // weight of a candidate
            const uint32_t key = key_of(i);
            const float place = sample_place(key);
            return place >= bin_lo && place < bin_hi && sample_sub(place, bins[0]) == bins[1] ? weight_of(key, i) : 0;
        };
        if (members <= kSampleList) {
            if (queued >= 0) {
                uint32_t c = 0;
                for (int j0 = 0; j0 < queued; j0 += 32) {
                    const int i = j0 + lane < queued ? (int)s.queue[warp][j0 + lane] : -1;
                    const bool hit = i >= 0 && in_bin(i);
                    const uint32_t m = __ballot_sync(0xffffffffu, hit), o = c + __popc(m & ((1u << lane) - 1));
                    if (hit && o < kSampleWarpList) s.list[warp][o] = comp_of(key_of(i), i);
                    c += __popc(m);
                }
                if (lane == 0) s.n_list[warp] = c;
            } else {
                list_if([](int) { return true; }, [&](int i) -> u64 { return in_bin(i) ? comp_of(key_of(i), i) : kNone; });
            }
            const int m = team.collect();
            if (m >= 0) {
                const u64 me = team.sorted(m), w = tid < m ? (by_mass ? sample_weight((uint32_t)(me >> 32)) : 1) : 0;
                u64 all;
                const u64 inc = before + team.scan(w, all);
                if (w && inc - w < need && need <= inc)
                    s.cut = (me & 0xffffffff00000000ull) | ((uint32_t)me >> kSamplePlace);
                __syncthreads();
                cut = s.cut;
                any_cut = true;
                // this CTA's kept mass: earlier bins, earlier parts of the bin, its own listed tokens
                u64 part = 0;
                if (by_mass) {
#pragma unroll
                    for (int level = 0; level < 2; ++level)
                        if (tid < bins[level]) part += s.mass[level][tid];
                    for (int j = lane; j < (int)s.n_list[warp]; j += 32)
                        if (s.list[warp][j] <= cut) part += sample_weight((uint32_t)(s.list[warp][j] >> 32));
                }
                known = by_mass;
                local = part;
                return;
            }
        }
        known = false;
        any_cut = true;
        // too many: equal keys as a rule
        uint32_t lo = ~0u, hi = 0;
        if (tid == 0) {
            s.kmin = ~0u;
            s.kmax = 0;
        }
        u64 mine, ahead, earlier;
        scan_runs([&]() -> u64 {
            u64 c = 0;
            for (int i = run_lo; i < run_hi; ++i)
                if (in_bin(i)) {
                    lo = min(lo, key_of(i));
                    hi = max(hi, key_of(i));
                    ++c;
                }
            return c;
        }, mine, ahead);  // its barrier comes after kmin and kmax are set
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0) {
            atomicMin(&s.kmin, lo);
            atomicMax(&s.kmax, hi);
        }
        team.gather(&earlier);
        lo = __reduce_min_sync(0xffffffffu, lane < team.C ? team.at(lane, &s.kmin) : ~0u);
        hi = __reduce_max_sync(0xffffffffu, lane < team.C ? team.at(lane, &s.kmax) : 0u);
        if (lo == hi) {  // the m-th of equal ones, in index order
            const u64 w = by_mass ? sample_weight(lo) : 1, m = (need - before + w - 1) / w;
            if (tid == 0) s.cut = 0;
            __syncthreads();
            walk([&](int j) -> u64 { return in_bin(j) ? 1 : 0; }, ahead + earlier, mine, m - 1,
                 [&](int i) { s.cut = comp_of(lo, i); });
            team.cl.sync();
            const u64 c = lane < team.C ? team.at(lane, &s.cut) : 0;  // one of them is not 0 (or the cut is)
            cut = warp_sum_u64(c);
            team.cl.sync();
            return;
        }
        // distinct keys closer than the bins tell apart: bisection over (key, index)
        u64 a = (u64)lo << 32, z = ((u64)hi << 32) | 0xffffffffull;
        while (a < z) {
            const u64 mid = a + (z - a) / 2;
            u64 v = 0;
            for (int i = tid; i < n; i += kSampleThreads) {
                const u64 w = in_bin(i);
                if (w && comp_of(key_of(i), i) <= mid) v += by_mass ? w : 1;
            }
            if (before + team.sum(v) >= need) z = mid;
            else a = mid + 1;
        }
        cut = a;
    };

    if (k > 0) find_cut(false);
    if (tp < 1.f) find_cut(true);
    auto kept = [&](int i) -> u64 { return weight_of(key_of(i), i); };
    u64 mine = 0, ahead = 0, earlier, total;
    if (known) {  // only the CTA that the draw falls into looks at its tokens again
        total = team.sum(local, &earlier);
    } else {
        scan_runs(run_mass, mine, ahead);
        total = team.gather(&earlier);
    }
    const u64 here = s.xchg[(team.turn - 1) & 1], r = draw(total);
    team.cl.sync();  // shared memory of others is read: the CTAs without the drawn token leave
    if (r < earlier || r - earlier >= here) return;
    if (known) {
        mine = run_mass();
        u64 all;
        ahead = team.scan(mine, all) - mine;
    }
    walk(kept, ahead + earlier, mine, r, [&](int i) {
        p.out[row] = i0 + i;
        if (p.prob) p.prob[row] = (float)kept(i) / (float)total;
    });
}

}  // namespace amcu

using namespace amcu;

namespace {

template <typename T, bool kRes>
void launch_sample(const SampleParams& p, int64_t rows, int c, int slice, size_t smem, cudaStream_t s) {
    const void* f = reinterpret_cast<const void*>(&sample_kernel<T, kRes>);
    set_func_attr_once(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleSlice * 4);
    set_func_attr_once(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * c));
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)c;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, sample_kernel<T, kRes>, p, slice);
}

}  // namespace

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
    p.rows = a->rows;
    p.uniform = a->uniform;
    p.temperature = a->temperature;
    p.top_k = a->top_k;
    p.top_p = a->top_p;
    p.min_p = a->min_p;
    p.out = a->out_index;
    p.prob = a->out_prob;
    // CTAs per row: as few as hold the row's keys in shared memory, and more
    // (down to 2048 tokens each) while the rows alone leave SMs idle.
    int c = 1;
    while (c < 16 && ceil_div(a->vocab, c) > kSampleSlice) c *= 2;
    while (c < 16 && a->rows * c * 2 <= num_sms() && ceil_div(a->vocab, 2 * c) >= 2048) c *= 2;
    p.ahead = 2 * num_sms() / c;
    const int slice = (int)(ceil_div(a->vocab, 8 * c) * 8);  // the slices of an aligned row are aligned
    const bool res = slice <= kSampleSlice, f32 = a->dtype == AMCU_F32;
    AMCU_REQUIRE(a->rows * c <= INT32_MAX, "amcu_sample: too many rows");
    const size_t smem = res ? (size_t)slice * 4 : 0;
    cudaStream_t st = as_stream(stream);
    if (f32) res ? launch_sample<float, true>(p, a->rows, c, slice, smem, st)
                 : launch_sample<float, false>(p, a->rows, c, slice, smem, st);
    else res ? launch_sample<__nv_bfloat16, true>(p, a->rows, c, slice, smem, st)
             : launch_sample<__nv_bfloat16, false>(p, a->rows, c, slice, smem, st);
    return check_launch("amcu_sample");
}
