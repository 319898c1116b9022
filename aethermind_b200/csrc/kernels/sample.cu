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
constexpr int kSampleList = kSampleThreads;       // candidates of a cut that are ranked against one another
constexpr int kSampleSlice = 16384;               // most keys that a CTA keeps in shared memory
constexpr float kSampleOne = 1099511627776.f;     // 2^40
constexpr float kSampleBinScale = kSampleBins / 28.f;  // weights end at z = -27.7
constexpr uint32_t kSampleNever = 0x7f800000u;    // key of a masked token

// |z| of a logit, as orderable bits. NaN and -inf give +inf.
__device__ __forceinline__ uint32_t sample_key(float x, float mx, float t) {
    if (x == mx) return 0u;
    const float z = __fdiv_rn(__fsub_rn(x, mx), t);
    return z <= 0.f ? __float_as_uint(-z) & 0x7fffffffu : kSampleNever;  // NaN: comparison is false
}
__device__ __forceinline__ u64 sample_weight(uint32_t key) {
    return (u64)__fmul_rn(expf(-__uint_as_float(key)), kSampleOne);
}
// Position of a key on a scale of 256 bins; bin and sub-bin are monotone in the key.
__device__ __forceinline__ float sample_place(uint32_t key) { return __fmul_rn(__uint_as_float(key), kSampleBinScale); }
__device__ __forceinline__ int sample_bin(float place) { return min((int)place, kSampleBins - 1); }
__device__ __forceinline__ int sample_sub(float place, int bin) {
    return min((int)__fmul_rn(__fsub_rn(place, (float)bin), 256.f), kSampleBins - 1);
}

struct SampleShared {
    u64 mass[2][kSampleBins];
    uint32_t count[2][kSampleBins];
    u64 list[kSampleList];       // this CTA's candidates
    u64 all[kSampleList];        // every CTA's
    u64 part[kSampleWarps];
    u64 scan[kSampleBins / 32];
    u64 xchg[2];
    float mx;
    float red[kSampleWarps];
    uint32_t n_list, kmin, kmax;
    u64 cut, before;
    uint32_t members;
    int bin, where;
};

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// What the row's CTAs do together: rank r of C holds tokens [r * slice, ...).
struct SampleTeam {
    SampleShared* s;
    cg::cluster_group cl;
    int rank, C, turn;

    __device__ __forceinline__ u64 at(int r, const u64* p) { return *cl.map_shared_rank(const_cast<u64*>(p), r); }

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
        cl.sync();
        const u64 x = lane < C ? at(lane, &s->xchg[turn & 1]) : 0;
        ++turn;
        if (before) *before = warp_sum_u64(lane < rank ? x : 0);
        return warp_sum_u64(x);
    }
};

// One cluster per row, its CTAs each holding a contiguous slice of the keys in
// shared memory (kRes; larger vocabularies compute them again from the logits).
template <typename T, bool kRes>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleParams p, int slice) {
    extern __shared__ __align__(16) uint32_t keys[];
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
    const bool greedy = !(t > 0.f);
    if (greedy) t = 1.f;
    const u64 least = mp > 0.f ? max((u64)ceil((double)mp * (double)kSampleOne), (u64)1) : 1;

    // ---- the row's largest logit
    float mx = -INFINITY;
    for (int i = tid; i < n; i += kSampleThreads) {
        const float f = Act<T>::load(x[i]);
        if (kRes) keys[i] = __float_as_uint(f);
        mx = fmaxf(mx, f);
    }
    mx = warp_max(mx);
    if (lane == 0) s.red[warp] = mx;
    __syncthreads();
    if (warp == 0) {
        mx = warp_max(lane < kSampleWarps ? s.red[lane] : -INFINITY);
        if (lane == 0) s.mx = mx;
    }
    team.cl.sync();
    mx = warp_max(lane < team.C ? *team.cl.map_shared_rank(&s.mx, lane) : -INFINITY);
    if (mx == -INFINITY) {  // nothing to draw from
        if (team.rank == 0 && tid == 0) {
            p.out[row] = -1;
            if (p.prob) p.prob[row] = 0.f;
        }
        team.cl.sync();  // nobody leaves while its maximum is read
        return;
    }
    if (kRes) {
        for (int i = tid; i < n; i += kSampleThreads) keys[i] = sample_key(__uint_as_float(keys[i]), mx, t);
    }
    __syncthreads();
    auto key_of = [&](int i) -> uint32_t { return kRes ? keys[i] : sample_key(Act<T>::load(x[i]), mx, t); };
    u64 cut = ~0ull;  // tokens up to it in the order of (key, index) are kept
    auto comp_of = [&](uint32_t key, int i) -> u64 { return ((u64)key << 32) | (u64)(i0 + i); };
    // weight of token i among the kept, 0 if it is not
    auto kept = [&](int i) -> u64 {
        const uint32_t key = key_of(i);
        if (comp_of(key, i) > cut) return 0;
        const u64 w = sample_weight(key);
        return w >= least ? w : 0;
    };
    // First local index whose running f() is above `target`; the caller knows there is one.
    auto locate = [&](auto f, u64 target) -> int {
        const int seg = (n + kSampleWarps - 1) / kSampleWarps;
        const int lo = min(warp * seg, n), hi = min(lo + seg, n);
        u64 v = 0;
        for (int i = lo + lane; i < hi; i += 32) v += f(i);
        v = warp_sum_u64(v);
        if (lane == 0) s.part[warp] = v;
        __syncthreads();
        u64 b = 0;
        for (int w = 0; w < warp; ++w) b += s.part[w];
        if (target >= b && target < b + v) {
            for (int c = lo; c < hi; c += 32) {
                const int i = c + lane;
                u64 y = i < hi ? f(i) : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 z = __shfl_up_sync(0xffffffffu, y, o);
                    if (lane >= o) y += z;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, b + y > target);
                if (hit) {
                    if (lane == 0) s.where = c + __ffs(hit) - 1;
                    break;
                }
                b += __shfl_sync(0xffffffffu, y, 31);
            }
        }
        __syncthreads();
        return s.where;
    };

    // The least cut at which the kept tokens' count (by_mass false) or mass reaches `need`.
    auto find_cut = [&](bool by_mass, u64 need) {
        u64 before = 0;   // of the tokens in earlier bins
        int bins[2] = {0, 0};
        uint32_t members = 0;
        for (int level = 0; level < 2; ++level) {
            if (tid < kSampleBins) {
                s.mass[level][tid] = 0;
                s.count[level][tid] = 0;
            }
            __syncthreads();
            for (int i = tid; i < n; i += kSampleThreads) {
                const u64 w = kept(i);
                if (!w) continue;
                const float place = sample_place(key_of(i));
                int bin = sample_bin(place);
                if (level == 1) {
                    if (bin != bins[0]) continue;
                    bin = sample_sub(place, bin);
                }
                if (by_mass) atomicAdd(&s.mass[level][bin], w);
                if (!by_mass || level == 1) atomicAdd(&s.count[level][bin], 1u);
            }
            team.cl.sync();
            u64 v = 0, cnt = 0;
            if (tid < kSampleBins) {
                for (int r = 0; r < team.C; ++r) {
                    if (by_mass) v += team.at(r, &s.mass[level][tid]);
                    if (!by_mass || level == 1) cnt += *team.cl.map_shared_rank(&s.count[level][tid], r);
                }
                if (!by_mass) v = cnt;
            }
            u64 inc = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 z = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += z;
            }
            if (lane == 31 && warp < kSampleBins / 32) s.scan[warp] = inc;
            __syncthreads();
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
        auto in_bin = [&](int i) -> u64 {  // weight of a candidate
            const float place = sample_place(key_of(i));
            return sample_bin(place) == bins[0] && sample_sub(place, bins[0]) == bins[1] ? kept(i) : 0;
        };
        if (members <= kSampleList) {  // rank them against one another
            if (tid == 0) s.n_list = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kSampleThreads)
                if (in_bin(i)) s.list[atomicAdd(&s.n_list, 1u)] = comp_of(key_of(i), i);
            team.cl.sync();
            int at = 0;
            for (int r = 0; r < team.C; ++r) {
                const int m = (int)*team.cl.map_shared_rank(&s.n_list, r);
                if (tid < m) s.all[at + tid] = team.at(r, &s.list[tid]);
                at += m;
            }
            __syncthreads();
            if (tid < at) {
                const u64 me = s.all[tid];
                u64 sum = before, own = 1;
                for (int j = 0; j < at; ++j) {
                    const u64 c = s.all[j];
                    const u64 w = by_mass ? sample_weight((uint32_t)(c >> 32)) : 1;
                    if (c <= me) sum += w;
                    if (c == me) own = w;
                }
                if (sum >= need && sum - own < need) s.cut = me;
            }
            __syncthreads();
            cut = s.cut;
            return;
        }
        // too many: equal keys as a rule
        uint32_t lo = ~0u, hi = 0;
        u64 mine = 0;
        for (int i = tid; i < n; i += kSampleThreads)
            if (in_bin(i)) {
                lo = min(lo, key_of(i));
                hi = max(hi, key_of(i));
                ++mine;
            }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (tid == 0) {
            s.kmin = ~0u;
            s.kmax = 0;
        }
        __syncthreads();
        if (lane == 0) {
            atomicMin(&s.kmin, lo);
            atomicMax(&s.kmax, hi);
        }
        u64 earlier = 0;
        team.sum(mine, &earlier);  // its barrier also publishes kmin and kmax
        lo = __reduce_min_sync(0xffffffffu, lane < team.C ? *team.cl.map_shared_rank(&s.kmin, lane) : ~0u);
        hi = __reduce_max_sync(0xffffffffu, lane < team.C ? *team.cl.map_shared_rank(&s.kmax, lane) : 0u);
        const u64 here = team.s->xchg[(team.turn - 1) & 1];  // this CTA's candidates
        if (lo == hi) {  // the m-th of equal ones, in index order
            const u64 w = by_mass ? sample_weight(lo) : 1, m = (need - before + w - 1) / w;
            const bool own = earlier < m && m <= earlier + here;
            if (own) {
                const int i = locate([&](int j) -> u64 { return in_bin(j) ? 1 : 0; }, m - earlier - 1);
                if (tid == 0) s.cut = comp_of(lo, i);
            } else if (tid == 0) {
                s.cut = 0;
            }
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

    if (greedy) k = 1;
    auto total_kept = [&](bool count, u64* earlier) {
        u64 v = 0;
        for (int i = tid; i < n; i += kSampleThreads) {
            const u64 w = kept(i);
            v += count ? (w ? 1 : 0) : w;
        }
        return team.sum(v, earlier);
    };
    if (k > 0 && (u64)k < total_kept(true, nullptr)) find_cut(false, (u64)k);
    if (tp < 1.f) {
        const double want = ceil((double)tp * (double)total_kept(false, nullptr));
        find_cut(true, want < 1.0 ? 1 : (u64)want);
    }
    u64 earlier = 0;
    const u64 total = total_kept(false, &earlier);
    const u64 here = s.xchg[(team.turn - 1) & 1];
    const double ud = floor((double)un * (double)total);
    u64 r = ud > 0.0 ? (u64)ud : 0;
    if (r >= total) r = total - 1;
    if (r >= earlier && r < earlier + here) {
        const int i = locate(kept, r - earlier);
        if (tid == 0) {
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
    const int slice = (int)ceil_div(a->vocab, c);
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
