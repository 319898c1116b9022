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
    int64_t stride, vocab;
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
// floor(expf(-|z|) * 2^40), from the float's fields (a 64-bit conversion is slow).
__device__ __forceinline__ u64 sample_weight(uint32_t key) {
    const uint32_t f = __float_as_uint(expf(-__uint_as_float(key)));
    const uint32_t m = (f & 0x007fffffu) | 0x00800000u;
    const int sh = (int)(f >> 23) - 110;
    return sh >= 0 ? (u64)m << sh : (u64)(sh > -24 ? m >> -sh : 0u);
}
// Position of a key on a scale of 256 bins (a weight above 0 is below 254); bin
// and sub-bin are monotone in the key.
__device__ __forceinline__ float sample_place(uint32_t key) { return __fmul_rn(__uint_as_float(key), kSampleBinScale); }
__device__ __forceinline__ int sample_bin(float place) { return (int)fminf(place, (float)(kSampleBins - 1)); }
__device__ __forceinline__ int sample_sub(float place, int bin) {
    return min((int)__fmul_rn(__fsub_rn(place, (float)bin), 256.f), kSampleBins - 1);
}

struct SampleShared {
    uint32_t mass[2][3][kSampleBins];  // a weight's bits 0-13, 14-27 and 28-40 (64-bit shared atomics are far slower)
    uint32_t count[2][kSampleBins];
    float group[kSampleThreads];       // maxima of the threads, or of 2, 4 or 8 neighbours
    u64 list[kSampleWarps][kSampleWarpList];  // each warp's candidates
    uint32_t n_list[kSampleWarps];
    uint32_t queue[kSampleWarps][kSampleQueue];
    u64 all[kSampleList];        // every CTA's
    u64 weight[kSampleList];     // by place: weights of the kept
    u64 tmp[kSampleList];
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
    // counted within their bin (512 tokens of a row: 1 us, a bitonic sort 4).
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
template <typename T, bool kRes>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleParams p, int slice) {
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
    const u64 least = mp > 0.f ? max((u64)ceil((double)fminf(mp, 1.f) * (double)kSampleOne), (u64)1) : 1;

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
                if (key >= kSampleNever || sample_bin(sample_place(key)) > bin || sample_weight(key) < least) return kNone;
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
    bool keyed = false;  // xs holds keys: the first pass over the tokens makes them
    auto key_of = [&](int i) -> uint32_t {
        if (kRes && keyed) return __float_as_uint(xs[i]);
        return sample_key(kRes ? xs[i] : Act<T>::load(x[i]), mx, t);
    };
    bool any_cut = false;
    u64 cut = ~0ull;  // tokens up to it in the order of (key, index) are kept
    auto comp_of = [&](uint32_t key, int i) -> u64 { return ((u64)key << 32) | (u64)(i0 + i); };
    auto weight_of = [&](uint32_t key, int i) -> u64 {  // 0 where the token is not kept
        if (any_cut && comp_of(key, i) > cut) return 0;
        const u64 w = sample_weight(key);
        return w >= least ? w : 0;
    };
    // scan_runs: f's sum over the thread's run, the sums of the threads before it,
    // and the CTA's total in xchg; walk: the first i of the run whose running f is
    // above `target`.
    auto scan_runs = [&](auto f, u64& mine, u64& before) {
        mine = 0;
#pragma unroll 4
        for (int i = run_lo; i < run_hi; ++i) mine += f(i);
        u64 all;
        before = team.scan(mine, all) - mine;
        if (tid == 0) s.xchg[team.turn & 1] = all;
    };
    auto walk = [&](auto f, u64 before, u64 target) -> int {
        for (int i = run_lo;; ++i) {
            before += f(i);
            if (before > target) return i;
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
            if (tid < kSampleBins) {
                s.mass[level][0][tid] = s.mass[level][1][tid] = s.mass[level][2][tid] = 0;
                s.count[level][tid] = 0;
            }
            __syncthreads();
            const float bin_lo = (float)bins[0], bin_hi = bin_lo + 1.f;
            auto add = [&](int i, uint32_t key) {
                const float place = sample_place(key);
                if (level == 1 && !(place >= bin_lo && place < bin_hi)) return;
                const int bin = level == 1 ? sample_sub(place, bins[0]) : sample_bin(place);
                const u64 w = weight_of(key, i);
                if (!w) return;
                if (by_mass) {
                    const uint32_t lo = (uint32_t)w & 0x3fffu, mid = (uint32_t)(w >> 14) & 0x3fffu, hi = (uint32_t)(w >> 28);
                    atomicAdd(&s.mass[level][0][bin], lo);
                    if (mid) atomicAdd(&s.mass[level][1][bin], mid);
                    if (hi) atomicAdd(&s.mass[level][2][bin], hi);
                }
                if (!by_mass || level == 1) atomicAdd(&s.count[level][bin], 1u);
            };
            if (level == 0) {
                if (kRes && !keyed) {
#pragma unroll 2
                    for (int i = tid; i < n; i += kSampleThreads) {
                        xs[i] = __uint_as_float(sample_key(xs[i], mx, t));
                        add(i, __float_as_uint(xs[i]));
                    }
                    keyed = true;
                    __syncthreads();
                } else {
#pragma unroll 2
                    for (int i = tid; i < n; i += kSampleThreads) add(i, key_of(i));
                }
            } else {
                // the bin's tokens first, so that they are looked at by full warps
                uint32_t c = 0;
#pragma unroll 2
                for (int at = seg_lo; at < seg_hi; at += 32) {
                    const float place = at + lane < seg_hi ? sample_place(key_of(at + lane)) : -1.f;
                    const uint32_t m = __ballot_sync(0xffffffffu, place >= bin_lo && place < bin_hi);
                    const uint32_t o = c + __popc(m & ((1u << lane) - 1));
                    if (((m >> lane) & 1u) && o < kSampleQueue) s.queue[warp][o] = (uint32_t)(at + lane);
                    c += __popc(m);
                }
                __syncwarp();
                queued = c <= kSampleQueue ? (int)c : -1;
                if (queued >= 0)
                    for (int j = lane; j < queued; j += 32) add((int)s.queue[warp][j], key_of((int)s.queue[warp][j]));
                else
                    for (int i = seg_lo + lane; i < seg_hi; i += 32) add(i, key_of(i));
            }
            team.cl.sync();
            u64 v = 0, cnt = 0;
            if (tid < kSampleBins) {
#pragma unroll 4
                for (int r = 0; r < team.C; ++r) {
                    if (by_mass)
                        v += (u64)team.at(r, &s.mass[level][0][tid]) + ((u64)team.at(r, &s.mass[level][1][tid]) << 14) +
                             ((u64)team.at(r, &s.mass[level][2][tid]) << 28);
                    if (!by_mass || level == 1) cnt += team.at(r, &s.count[level][tid]);
                }
                if (!by_mass) v = cnt;
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
                    if (need >= all) return;  // nothing to cut
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
                        if (tid < bins[level])
                            part += (u64)s.mass[level][0][tid] + ((u64)s.mass[level][1][tid] << 14) + ((u64)s.mass[level][2][tid] << 28);
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
        scan_runs([&](int i) -> u64 {
            if (!in_bin(i)) return 0;
            lo = min(lo, key_of(i));
            hi = max(hi, key_of(i));
            return 1;
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
            ahead += earlier;
            if (ahead < m && m <= ahead + mine)
                s.cut = comp_of(lo, walk([&](int j) -> u64 { return in_bin(j) ? 1 : 0; }, ahead, m - 1));
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
        scan_runs(kept, mine, ahead);
        total = team.gather(&earlier);
    }
    const u64 here = s.xchg[(team.turn - 1) & 1], r = draw(total);
    if (r >= earlier && r < earlier + here) {  // the whole CTA
        if (known) {
            mine = 0;
#pragma unroll 4
            for (int i = run_lo; i < run_hi; ++i) mine += kept(i);
            u64 all;
            ahead = team.scan(mine, all) - mine;
        }
        ahead += earlier;
        if (r >= ahead && r < ahead + mine) {
            const int i = walk(kept, ahead, r);
            p.out[row] = i0 + i;
            if (p.prob) p.prob[row] = (float)kept(i) / (float)total;
        }
    }
    team.cl.sync();  // nobody leaves while its shared memory is read
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
