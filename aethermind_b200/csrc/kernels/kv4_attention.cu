// Causal GQA attention over the 4-bit paged KV cache.
//
// out[row, h] = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q . k_j - max), over
// the positions j <= pos of the row's sequence; k_j = m + s * code.
#include <algorithm>

#include "kv4.cuh"
#include "mma_int4.cuh"

namespace amcu {

// ---------------------------------------------------------------------------
// Single tokens and short runs of rows.
//
// The columns of a product are (row, q head) pairs of one kv head, 8 to a tile
// (fp32: 4, each as a high and a low fp16 half in neighbouring columns), the
// rows are keys: S^T = K Q^T and O^T = V^T P^T with mma.sync m16n8k16, so the
// big operand needs no padding whatever the group size. The work is cut in
// units of 16 keys of one (sequence, kv head, column tile); the units of the
// whole call lie in one row, and every CTA takes an equal, contiguous share
// of them (found from row_start and ctx_len on the device), so ragged batches
// and single long sequences fill the GPU alike. A CTA's 8 warps take its units
// in turn, each through a cp.async ring of its own. An item cut between CTAs
// leaves partial sums that kv4_combine_kernel adds in the order of the CTAs.
//
// Codes enter both products without any conversion: a nibble in bits 0-3 of a
// half is the fp16 subnormal c * 2^-24, one in bits 4-7 is c * 2^-20. q is scaled
// by a power of two to [1, 2) and its elements at the low nibbles by 16 more,
// which makes the integer dot product exact up to fp32 sums; scale and minimum
// of a key's group are applied to the 64-element sums (m through sum(q)). In the
// second product the rows that come from low nibbles are 2^-4 of the others until
// the end, the scales of V go into p (p s, rounded to 11 bits), and the minima and
// the softmax denominator are three more rows of the product. p and p s are fp16: a
// tail of many keys under one that has most of the mass keeps its bits because p is
// counted in 2^-10 of the largest (p of 2^-20 lost 2 to 80% of such a tail where it was
// counted in the largest itself), and scales below 2^-4 or above 4 are lifted by a power
// of two, so that precision is relative to the largest that the warp meets. The MMA
// aligns its products by their operands' exponents, subnormals' by that of 2^-14: sums
// with such codes are good to 2^-17 of their largest term, which bf16 does not see.
//
// fp32 calls work with normal halves around zero, c - 8 = (1024 + c) - 1032, and 8 s
// more in the minimum. An average over many keys is small beside its terms, so
// there V's elements are formed whole, m + s c in fp32, and go into the product as
// a high and a low half; p, counted in 2^-12 of the largest, does too, its low half
// times 2^11 so that it keeps its bits where p is small. The MMA truncates what it adds
// to an accumulator, so a unit's sums start at 0 and are added to the others' by
// rounding additions (600 keys, one with nearly all the mass, in one warp: relative
// error 2.1e-5 without either, 3.7e-6 with both; 64 sequences of 65536 keys: 9.7e-6 and
// 1.1e-7. Thousands of equal keys under one that has half the mass still lose up to
// 1e-4, as in any running sum of 32 bits).
constexpr int kDecWarps = 8;
constexpr int kDecThreads = kDecWarps * 32;
constexpr int kDecStages = 4;  // 64 ragged rows: 103.4 us, 103.8 with 3, 104.8 with 5
constexpr int kDecUnit = 16;       // keys per unit
// Units of a CTA at least: one for each warp, or what an item has on average where
// that is less (an item costs a CTA 2 to 5 us whatever its length: one row over 7
// keys, 8 kv heads of 64, 21.5 us with all items in one CTA, 6.0 with one in each).
constexpr int kDecMinUnits = 8;
// A warp takes whole items by itself, without the CTA's merge, where a CTA would
// have kDecMany or more of them and none is longer than kDecLong units for each of
// those (a single long one would keep the others waiting). Sequences of one row,
// 32 / 8 heads of 128, us so / by CTAs: 64 of 20 keys 12 / 17, 128 of 100 20 / 34, 128
// of 250 23 / 34, 256 of 100 21 / 47, 256 of 300 34 / 65, 256 of 600 55 / 84.
constexpr int kDecMany = 2, kDecLong = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kDecLift = 3.f;    // scores pass their largest so far by that much (log2) before the reference moves
// The reference lies that far below the largest score: p is up to 2^13 (fp32: 2^15) and
// an fp16 normal, rounded to 11 bits, down to 2^-24 (2^-26) of the largest one.
constexpr float kLowUp = 2048.f;   // fp32: the low half of p is held times 2^11, as large as the high one
template <typename T> constexpr float dec_head() { return sizeof(T) == 2 ? 10.f : 12.f; }

template <typename T> constexpr int dec_cols() { return sizeof(T) == 2 ? 8 : 4; }  // (row, head) pairs per tile
template <int D> constexpr int dec_stage_bytes() { return 2 * kDecUnit * (D / 2 + D / 16) + 16; }
template <int D> constexpr int dec_merge_stride() { return D + 4; }
template <int D> constexpr int dec_merge_bytes() { return kDecWarps * 8 * (dec_merge_stride<D>() + 4) * 4; }
template <int D> constexpr int dec_smem_bytes() {
    const int ring = kDecWarps * kDecStages * dec_stage_bytes<D>();
    return ring > dec_merge_bytes<D>() ? ring : dec_merge_bytes<D>();
}

struct DecMeta {   // for the CTA that holds an item's last unit but not its first
    int32_t first;   // CTA of the first unit; -1: nothing to combine
    int32_t row0, head0, col0, cols;  // the sequence's first row, the kv head's first q head, the tile's columns
    int32_t pad[3];
};
struct DecWork {
    float2* ml;    // [CTA][2][8] (reference, denominator)
    float* o;      // [CTA][2][8][D]
    DecMeta* meta; // [CTA]
    int64_t items; // (sequence, kv head, column tile) triples of the call, at most
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t movm_trans(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// 16-byte chunk of a stage that holds chunk c of token tk: the rows of a
// 128-byte line are XOR-swizzled so that a K read (8 bytes or 16 of 4 or 2
// neighbouring tokens) and a V read (every second token) both touch every
// bank once.
template <int D>
__device__ __forceinline__ int dec_chunk(int tk, int c) {
    return D == 128 ? (tk >> 1) * 8 + ((((tk & 1) << 2) + c) ^ (((tk >> 1) & 3) << 1))
                    : (tk >> 2) * 8 + ((((tk & 3) << 1) + c) ^ (((tk >> 2) & 1) << 1));
}

// Codes in bits 0-3 (high: 4-7) of both halves as an MMA operand; kNormal: code - 8.
template <bool kNormal>
__device__ __forceinline__ uint32_t dec_code(uint32_t w, bool high) {
    if (!kNormal) return high ? w & 0x00F000F0u : w & 0x000F000Fu;
    return h2u(high ? __hadd2(u2h((w & 0x00F000F0u) | 0x54005400u), __float2half2_rn(-72.f))
                    : __hadd2(u2h((w & 0x000F000Fu) | 0x64006400u), __float2half2_rn(-1032.f)));
}

// Cost of sequence b in units, and what a segment needs of it.
struct DecSeq {
    int row0, n, ctx, units, tiles;
};
template <typename T>
__device__ __forceinline__ DecSeq dec_seq(const Kv4View& v, int grp, int b) {
    DecSeq s;
    kv4_rows(v, b, s.row0, s.n);
    s.ctx = v.ctx_len[b];
    const int64_t cap = (int64_t)v.max_pages << v.page_shift;
    const int vis = (int)min((int64_t)max(s.ctx, 0), cap);
    s.units = max((vis + kDecUnit - 1) / kDecUnit, 1);
    s.tiles = (int)(((int64_t)s.n * grp + dec_cols<T>() - 1) / dec_cols<T>());
    return s;
}

template <typename T, int D>
__global__ void __launch_bounds__(kDecThreads, 2) kv4_decode_kernel(Kv4AttnParams p, DecWork ws) {
    constexpr int G = D / kKv4Group, CT = dec_cols<T>();
    constexpr bool kWide = sizeof(T) == 4;  // fp32: two halves per value
    constexpr int kCodes = kDecUnit * D / 2, kParams = kDecUnit * D / 16;
    constexpr int kStage = dec_stage_bytes<D>(), S = kDecStages;
    constexpr int kMS = dec_merge_stride<D>();
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t s_off;
    __shared__ int s_b;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_trigger();

    // ---- this CTA's share [x, x_end) of all units
    const Kv4View& v = p.v;
    const int row_first = v.row_start[0], row_end = v.row_start[v.n_seq];
    int most = 0;  // units of an item
    auto cost_of = [&](int i) {
        const DecSeq q = dec_seq<T>(v, p.grp, i);
        if (q.tiles) most = max(most, q.units);
        return (int64_t)q.units * q.tiles * v.nkv;
    };
    int64_t total, share, x;
    bool alone = false;  // a warp to an item
    {
        int b;
        int64_t off;
        const bool have = kv4_share<kDecThreads>(
                v.n_seq,
                [&](int64_t all) {
                    const int64_t many = ws.items / gridDim.x;
                    alone = many >= kDecMany && !__syncthreads_or(most > kDecLong * many);
                    share = alone ? (all + gridDim.x * kDecWarps - 1) / (gridDim.x * kDecWarps) * kDecWarps
                                  : max((all + gridDim.x - 1) / gridDim.x, min((all + ws.items - 1) / ws.items, (int64_t)kDecMinUnits));
                    return x = blockIdx.x * share;
                },
                cost_of, total, b, off);
        if (have) {
            s_b = b;
            s_off = off;
        }
    }
    kv4_zero_uncovered<T, kDecThreads>(v, row_first, row_end, p.out, p.os, p.nq * D);
    int64_t x_end = min(x + share, total);
    if (threadIdx.x == 0) ws.meta[blockIdx.x].first = -1;
    if (x >= x_end) return;
    __syncthreads();
    int b = s_b;
    int64_t off = s_off;
    // unit k of this warp's part of a segment is its first + w0 + (k << w_shift)
    const int w0 = alone ? 0 : warp, w_shift = alone ? 0 : 3;
    if (alone) {  // the items that begin in this warp's part of the share
        x += warp * (share / kDecWarps);
        off += warp * (share / kDecWarps);
        x_end = min(x + share / kDecWarps, total);
    }
    const uint32_t ring = smem_u32(smem) + warp * (S * kStage);
    const uint8_t* ring_p = smem + warp * (S * kStage);
    const int page_units_shift = v.page_shift - 4;

    while (x < x_end) {
        const DecSeq sq = dec_seq<T>(v, p.grp, b);
        const int64_t cost = (int64_t)sq.units * sq.tiles * v.nkv;
        if (off >= cost) {
            off -= cost;
            ++b;
            continue;
        }
        const int item = (int)(off / sq.units), u0 = (int)(off - (int64_t)item * sq.units);
        if (alone && u0 > 0) {
            x += sq.units - u0;
            off += sq.units - u0;
            continue;
        }
        const int kvh = item / sq.tiles, ct = item - kvh * sq.tiles;
        const int u1 = alone ? sq.units : (int)min((int64_t)sq.units, u0 + (x_end - x));
        const int cap = (int)min((int64_t)max(sq.ctx, 0), (int64_t)v.max_pages << v.page_shift);  // keys that can exist
        const int cols = min(CT, sq.n * p.grp - ct * CT);
        // keys past the page table, or rows before position 0 (alone: no other warp meets the item)
        if ((sq.ctx > cap || sq.ctx < sq.n) && v.status && lane == 0) *v.status = (int32_t)AM_STATUS_OUT_OF_RANGE;

        // ---- the tile's columns: this lane's is r (MMA operand), its results are of columns 2t, 2t + 1
        const int c_op = kWide ? r >> 1 : r;
        const bool c_live = c_op < cols;
        const int fc = ct * CT + (c_live ? c_op : 0);
        const int c_row = fc / p.grp, c_head = kvh * p.grp + fc - c_row * p.grp;
        const T* qp = static_cast<const T*>(p.q) + (int64_t)(sq.row0 + c_row) * p.qs + (int64_t)c_head * D + 16 * t;
        float qv[G][16];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 16; ++i) qv[g][i] = c_live ? Act<T>::load(qp[g * kKv4Group + i]) : 0.f;
        const int lim_op = c_live ? min(sq.ctx - sq.n + c_row, cap - 1) : -1;  // last visible position
        // keys past the last column's limit need no unit; before the first one's, no mask
        const int lim_last = __shfl_sync(0xffffffffu, lim_op, kWide ? 8 * (cols - 1) : 4 * (cols - 1));
        const int lim_first = __shfl_sync(0xffffffffu, lim_op, 0);
        const int u_end = min(u1, (lim_last + kDecUnit) / kDecUnit);  // lim_last = -1: none
        const int full = (lim_first + 1) / kDecUnit;  // units before it need no mask

        // ---- ring
        const int u_first = u0 + w0, nk = u_end > u_first ? (u_end - u_first - 1 >> w_shift) + 1 : 0;
        int pages = -1;
        bool holes = false;   // a page that is none was met
        const int64_t head_c = ((int64_t)kvh << v.page_shift) * (D / 2), head_p = ((int64_t)kvh << v.page_shift) * (D / 16);
        constexpr int PC = kParams / 16;
        const uint8_t* const k_src = v.kc + head_c + lane * 16;
        const uint8_t* const v_src = v.vc + head_c + lane * 16;
        const uint8_t* const p_src = lane < PC ? v.kp + head_p + lane * 16 : v.vp + head_p + (lane - PC) * 16;
        const uint32_t c_dst = ring + (uint32_t)dec_chunk<D>(lane / (D / 32), lane % (D / 32)) * 16;
        const uint32_t p_dst = ring + 2 * kCodes + lane * 16;
        const uint32_t slot_mask = (1u << page_units_shift) - 1;
        auto fetch = [&](int k) {
            if (k < nk) {
                if ((k & 31) == 0) {  // page ids of the next 32 units, one per lane
                    const int u = u_first + ((k + lane) << w_shift);
                    pages = u < u_end ? kv4_page(v, b, u * kDecUnit) : 0;
                    holes |= __any_sync(0xffffffffu, pages < 0);
                }
                const int page = __shfl_sync(0xffffffffu, pages, k & 31);
                const uint32_t st = (uint32_t)(k % S) * kStage, ok = page >= 0 ? 16u : 0u, pg = page >= 0 ? page : 0;
                const uint32_t slot = (uint32_t)(u_first + (k << w_shift)) & slot_mask;
                const uint64_t co = pg * (uint64_t)(uint32_t)v.cps + slot * kCodes;  // pages are below 4 GB
#pragma unroll
                for (int i = 0; i < kCodes / 512; ++i) {  // 512 bytes are whole swizzled lines
                    cp16(c_dst + st + i * 512, k_src + co + i * 512, ok);
                    cp16(c_dst + st + kCodes + i * 512, v_src + co + i * 512, ok);
                }
                if (lane < 2 * PC) cp16(p_dst + st, p_src + pg * (uint64_t)(uint32_t)v.pps + slot * kParams, ok);
                if (lane == 0) *reinterpret_cast<int*>(const_cast<uint8_t*>(ring_p) + st + 2 * (kCodes + kParams)) = page;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };

        // on their way while q is prepared
#pragma unroll
        for (int k = 0; k < S - 1; ++k) fetch(k);

        uint32_t amax = 0;  // bits of the largest |q|: NaN above infinity above the rest
        float qsum[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
            for (int i = 0; i < 16; ++i) amax = max(amax, __float_as_uint(qv[g][i]) & 0x7fffffffu);
            float half_sum[8];  // by halves: 6 roundings for 64 elements
#pragma unroll
            for (int i = 0; i < 8; ++i) half_sum[i] = qv[g][i] + qv[g][i + 8];
#pragma unroll
            for (int w = 4; w > 0; w /= 2)
#pragma unroll
                for (int i = 0; i < w; ++i) half_sum[i] += half_sum[i + w];
            qsum[g] = half_sum[0];
            qsum[g] += __shfl_xor_sync(0xffffffffu, qsum[g], 1);
            qsum[g] += __shfl_xor_sync(0xffffffffu, qsum[g], 2);
        }
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const uint32_t eb = min(max(amax >> 23, 1u), 253u);
        // a row with an element that is no number or infinite has no softmax: all its scores are NaN
        const float inv = __uint_as_float(amax < 0x7f800000u ? (254u - eb) << 23 : 0x7fc00000u);
        uint32_t qf[2 * G][2][2];  // [word][half of the word][b0, b1]
#pragma unroll
        for (int j = 0; j < 2 * G; ++j)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int e = 0; e < 2; ++e) {  // nibbles 2 hh + e and 2 hh + e + 4
                    const int i = 8 * (j / G) + 2 * hh + e;
                    float a = qv[j % G][i] * inv, c = qv[j % G][i + 4] * inv;
                    if (kWide) {
                        const float ah = __half2float(__float2half_rn(a)), ch = __half2float(__float2half_rn(c));
                        a = (r & 1) ? a - ah : ah;
                        c = (r & 1) ? c - ch : ch;
                    }
                    const float lift = !kWide && e == 0 ? 16.f : 1.f;
                    qf[j][hh][e] = h2u(__floats2half2_rn(a * lift, c * lift));
                }
        // results: factor of the integer sums, sum(q) per group, last visible position
        const float sl = p.scale * kLog2e;
        const float f_op = __uint_as_float(eb << 23) * sl * (kWide ? 1.f : 1048576.f);
        float f[2], qg[G][2];
        int lim[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int src = kWide ? 8 * t : 8 * t + 4 * j;
            f[j] = __shfl_sync(0xffffffffu, f_op, src);
            lim[j] = __shfl_sync(0xffffffffu, lim_op, src);
#pragma unroll
            for (int g = 0; g < G; ++g) qg[g][j] = __shfl_sync(0xffffffffu, qsum[g] * sl, src);
        }
        float ref[2] = {-1e30f, -1e30f};
        float lift = 0.f;     // fp32: V's elements are multiplied by it (0: not chosen yet)
        uint32_t s_most = 0;  // bf16: 4 / lift in both halves, a power of two; a scale above it asks for another lift
        auto lift_of = [](uint32_t most) {  // 0: not chosen yet, every scale so far is 0
            return __uint_as_float((256u << 23) - __float_as_uint(__low2float(u2h(most))));
        };
        float o[G][4][4], xa[4] = {};
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[g][i][c] = 0.f;
        for (int k = 0; k < nk; ++k) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
            __syncwarp();
            fetch(k + S - 1);
            const uint8_t* st = ring_p + (k % S) * kStage;
            const int u = u_first + (k << w_shift);
            const uint8_t* kpar = st + 2 * kCodes;
            const uint8_t* vpar = kpar + kParams;

            // ---- S^T: keys r and r + 8
            float a[G][4];
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int c = 0; c < 4; ++c) a[g][c] = 0.f;
            uint32_t k0[2 * G], k1[2 * G];
            if (D == 128) {
                const uint4 w0 = lds_u4(st + dec_chunk<D>(r, t) * 16), w1 = lds_u4(st + dec_chunk<D>(r + 8, t) * 16);
                k0[0] = w0.x; k0[1] = w0.y; k0[2 * G - 2] = w0.z; k0[2 * G - 1] = w0.w;
                k1[0] = w1.x; k1[1] = w1.y; k1[2 * G - 2] = w1.z; k1[2 * G - 1] = w1.w;
            } else {
                const uint2 w0 = *reinterpret_cast<const uint2*>(st + dec_chunk<D>(r, t >> 1) * 16 + (t & 1) * 8);
                const uint2 w1 = *reinterpret_cast<const uint2*>(st + dec_chunk<D>(r + 8, t >> 1) * 16 + (t & 1) * 8);
                k0[0] = w0.x; k0[1] = w0.y;
                k1[0] = w1.x; k1[1] = w1.y;
            }
#pragma unroll
            for (int j = 0; j < 2 * G; ++j) {
                const uint32_t lo[4] = {dec_code<kWide>(k0[j], false), dec_code<kWide>(k1[j], false), dec_code<kWide>(k0[j], true),
                                        dec_code<kWide>(k1[j], true)};
                mma_f16_16816(a[j % G], lo, qf[j][0][0], qf[j][0][1]);
                const uint32_t s0 = k0[j] >> 8, s1 = k1[j] >> 8;
                const uint32_t hi[4] = {dec_code<kWide>(s0, false), dec_code<kWide>(s1, false), dec_code<kWide>(s0, true),
                                        dec_code<kWide>(s1, true)};
                mma_f16_16816(a[j % G], hi, qf[j][1][0], qf[j][1][1]);
            }
            float sc[4];  // (key r: columns 2t, 2t + 1), (key r + 8: ...); fp32: one head, in [0] and [2]
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                float2 sm[G];
                const uint8_t* kr = kpar + (r + 8 * hh) * (4 * G);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    sm[g] = __half22float2(*reinterpret_cast<const __half2*>(kr + 4 * g));
                    if (kWide) sm[g].y = fmaf(8.f, sm[g].x, sm[g].y);  // codes are 8 less
                }
#pragma unroll
                for (int j = 0; j < (kWide ? 1 : 2); ++j) {
                    float dot = 0.f, add = 0.f;
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float ag = kWide ? a[g][2 * hh] + a[g][2 * hh + 1] : a[g][2 * hh + j];
                        dot = fmaf(sm[g].x, ag, dot);
                        add = fmaf(sm[g].y, qg[g][j], add);
                    }
                    sc[2 * hh + j] = fmaf(dot, f[j], add);
                }
                if (kWide) sc[2 * hh + 1] = sc[2 * hh];
            }
            // V's parameters of tokens 2t, 2t + 1 and 2t + 8, 2t + 9
            uint32_t vs[2][G], vm[2][G];  // (token, token + 1) pairs: scales, minima
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                uint32_t w[2 * G];
                const uint8_t* vr = vpar + (2 * t + 8 * hh) * (4 * G);
                if (G == 2) {
                    const uint4 y = lds_u4(vr);
                    w[0] = y.x; w[1] = y.y; w[2 * G - 2] = y.z; w[2 * G - 1] = y.w;
                } else {
                    const uint2 y = *reinterpret_cast<const uint2*>(vr);
                    w[0] = y.x; w[1] = y.y;
                }
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    vs[hh][g] = __byte_perm(w[g], w[G + g], 0x5410);
                    vm[hh][g] = __byte_perm(w[g], w[G + g], 0x7632);
                }
            }
            if (u >= full || holes) {  // masks; nothing of an unseen key may reach a product
                const bool none = *reinterpret_cast<const int*>(st + 2 * (kCodes + kParams)) < 0;
                const int key = u * kDecUnit + r;
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (none || key + 8 * hh > lim[j]) sc[2 * hh + j] = -INFINITY;
                    const int vk = u * kDecUnit + 2 * t + 8 * hh;
                    const uint32_t keep = (vk <= lim_last ? 0x0000FFFFu : 0u) | (vk + 1 <= lim_last ? 0xFFFF0000u : 0u);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        vs[hh][g] &= keep;
                        vm[hh][g] &= keep;
                    }
                }
                // A group of V that is NaN (its minimum or scale is) may be of a key that only some
                // columns see: 0 times it would reach the others. It goes into the sums of those that do.
                uint32_t odd = 0;
#pragma unroll
                for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                    for (int g = 0; g < G; ++g) odd |= __hneu2_mask(u2h(vm[hh][g]), u2h(vm[hh][g])) | __hneu2_mask(u2h(vs[hh][g]), u2h(vs[hh][g]));
                if (__any_sync(0xffffffffu, odd != 0)) {
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            const uint32_t nan = __hneu2_mask(u2h(vm[hh][g]), u2h(vm[hh][g])) | __hneu2_mask(u2h(vs[hh][g]), u2h(vs[hh][g]));
                            vm[hh][g] &= ~nan;
                            vs[hh][g] &= ~nan;
                            // the first such key of the eight (lanes of equal t hold the same two)
                            int at = 0x7fffffff;
                            if (nan) at = u * kDecUnit + 2 * t + 8 * hh + (nan & 0xffffu ? 0 : 1);
                            at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (at <= lim[c & 1]) {
#pragma unroll
                                    for (int i = 0; i < 4; ++i) o[g][i][c] = __uint_as_float(0x7fc00000u);
                                }
                        }
                }
            }
            // fp32: elements of V to where their two halves keep their bits, at the warp's first unit and
            // again for much larger ones
            if (kWide) {
                float top = 0.f;  // the largest element of the unit's 16 keys
#pragma unroll
                for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float2 sv = __half22float2(u2h(vs[hh][g])), mv = __half22float2(u2h(vm[hh][g]));
                        top = fmaxf(top, fmaxf(fmaxf(fabsf(mv.x), fabsf(fmaf(15.f, sv.x, mv.x))),
                                               fmaxf(fabsf(mv.y), fabsf(fmaf(15.f, sv.y, mv.y)))));
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float fits = __uint_as_float((264u - (__float_as_uint(fmaxf(top, 6e-8f)) >> 23)) << 23);  // to [1024, 2048)
                if (lift == 0.f) {
                    lift = fits;
                } else if (top * lift >= 32768.f) {
                    const float corr = fits / lift;
                    lift = fits;
#pragma unroll
                    for (int g = 0; g < G; ++g)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int c = 0; c < 4; ++c) o[g][i][c] *= corr;
                }
            }
            // ---- softmax: the reference moves only when a score passes the largest so far by kDecLift;
            // bf16: and V's lift when a scale passes s_most
            constexpr float kHead = dec_head<T>();
            float pr[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) pr[c] = sc[c] - ref[c & 1];
            __half2 s_top = u2h(vs[0][0]);
#pragma unroll
            for (int e = 1; e < 2 * G; ++e) s_top = __hmax2(s_top, u2h(vs[e & 1][e >> 1]));
            const bool odd_scale = !kWide && __hgt2_mask(s_top, u2h(s_most)) != 0;
            if (__any_sync(0xffffffffu, odd_scale || fmaxf(fmaxf(pr[0], pr[1]), fmaxf(pr[2], pr[3])) > kHead + kDecLift)) {
                float s_corr = 1.f;
                if (!kWide && __any_sync(0xffffffffu, odd_scale)) {
                    float top = fmaxf(__low2float(s_top), __high2float(s_top));  // over the unit's 16 keys
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    // usual scales stay as they are, others go to [1/4, 1/2): p s is up to 2^15, and normal
                    // down to p of 2^-20 of the largest
                    const float fits = __uint_as_float((252u - min(__float_as_uint(top) >> 23, 138u)) << 23);
                    const float next = s_most == 0 && top >= 0.0625f && top <= 4.f ? 1.f : fits;
                    if (s_most != 0) s_corr = next * __uint_as_float((254u << 23) - __float_as_uint(lift_of(s_most)));
                    s_most = h2u(__float2half2_rn(__uint_as_float((256u << 23) - __float_as_uint(next))));
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float m = fmaxf(sc[j], sc[2 + j]);
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    m = fmaxf(m - kHead, ref[j]);
                    const float corr = ex2(ref[j] - m), o_corr = corr * s_corr;
                    ref[j] = m;
                    pr[j] = sc[j] - m;
                    pr[2 + j] = sc[2 + j] - m;
                    xa[j] *= corr;
                    xa[2 + j] *= corr;
#pragma unroll
                    for (int g = 0; g < G; ++g)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            o[g][i][j] *= o_corr;
                            o[g][i][2 + j] *= o_corr;
                        }
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) pr[c] = ex2(pr[c]);
            uint32_t pb[2], ps[2][G];  // p, and p times the groups' scales (bf16)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                if (kWide) {
                    auto two = [](float x) {
                        const __half h = __float2half_rn(x);
                        return movm_trans(h2u(__halves2half2(h, __float2half_rn((x - __half2float(h)) * kLowUp))));
                    };
                    pb[hh] = two(pr[2 * hh]);
                } else {
                    pb[hh] = movm_trans(h2u(__floats2half2_rn(pr[2 * hh], pr[2 * hh + 1])));
                    if (s_most != 0x44004400u) {
                        const float lift = lift_of(s_most);
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            const float2 y = __half22float2(u2h(vs[hh][g]));
                            vs[hh][g] = h2u(__floats2half2_rn(y.x * lift, y.y * lift));
                        }
                    }
#pragma unroll
                    for (int g = 0; g < G; ++g) ps[hh][g] = h2u(__hmul2(u2h(pb[hh]), u2h(vs[hh][g])));
                }
            }
            // ---- rows: minima of the groups (fp32: none), ones
            {
                uint32_t e[4] = {0, 0, 0, 0};
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    uint32_t w = r == G ? 0x3C003C00u : 0u;
#pragma unroll
                    for (int g = 0; g < G; ++g) w = !kWide && r == g ? vm[hh][g] : w;
                    e[2 * hh] = w;
                }
                if (kWide) {
                    float sum[4] = {};
                    mma_f16_16816(sum, e, pb[0], pb[1]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) xa[c] += sum[c];
                } else {
                    mma_f16_16816(xa, e, pb[0], pb[1]);
                }
            }
            // ---- O^T: this lane's rows are elements 8 r .. 8 r + 7 of each group
            uint32_t vw[2][2][G];  // [half][token of the pair][group]
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int tk = 2 * t + 8 * hh + y;
                    if (G == 2) {
                        const uint2 w = *reinterpret_cast<const uint2*>(st + kCodes + dec_chunk<D>(tk, r >> 1) * 16 + (r & 1) * 8);
                        vw[hh][y][0] = w.x;
                        vw[hh][y][G - 1] = w.y;
                    } else {
                        vw[hh][y][0] = *reinterpret_cast<const uint32_t*>(st + kCodes + dec_chunk<D>(tk, r >> 2) * 16 + (r & 3) * 4);
                    }
                }
#pragma unroll
            for (int g = 0; g < G; ++g) {
#pragma unroll
                for (int part = 0; part < 2; ++part) {  // elements 4 part .. 4 part + 3
                    uint32_t w[2];
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh)
                        w[hh] = __byte_perm(vw[hh][0][g], vw[hh][1][g], part ? 0x7632 : 0x5410);
#pragma unroll
                    for (int q2 = 0; q2 < 2; ++q2) {
                        const uint32_t wa = q2 ? w[0] >> 8 : w[0], wb = q2 ? w[1] >> 8 : w[1];
                        const uint32_t e[4] = {dec_code<kWide>(wa, false), dec_code<kWide>(wa, true), dec_code<kWide>(wb, false),
                                               dec_code<kWide>(wb, true)};
                        if (kWide) {
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {  // tokens 2t, 2t + 1 (i < 2) or 2t + 8, 2t + 9
                                const float2 c = __half22float2(u2h(e[i])), sv = __half22float2(u2h(vs[i >> 1][g])),
                                             mv = __half22float2(u2h(vm[i >> 1][g]));
                                const float v0 = fmaf(c.x, sv.x, fmaf(8.f, sv.x, mv.x)) * lift;
                                const float v1 = fmaf(c.y, sv.y, fmaf(8.f, sv.y, mv.y)) * lift;
                                const __half2 h = __floats2half2_rn(v0, v1);
                                const float2 hf = __half22float2(h);
                                hi[i] = h2u(h);
                                lo[i] = h2u(__floats2half2_rn(v0 - hf.x, v1 - hf.y));
                            }
                            float sum[4] = {};
                            mma_f16_16816(sum, hi, pb[0], pb[1]);
                            mma_f16_16816(sum, lo, pb[0], pb[1]);
#pragma unroll
                            for (int c = 0; c < 4; ++c) o[g][2 * part + q2][c] += sum[c];
                        } else {
                            mma_f16_16816(o[g][2 * part + q2], e, ps[0][g], ps[1][g]);
                        }
                    }
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // ---- the warps' sums together: [warp][column][D] and (reference, denominator, minima)
        if (alone) __syncwarp();
        else __syncthreads();  // the rings are read out
        float* mo = reinterpret_cast<float*>(alone ? smem + warp * (S * kStage) : smem);
        float* mx = mo + (alone ? 1 : kDecWarps) * 8 * kMS;  // [warp][column][4]
        // low nibbles are in units of 2^-24, high ones of 2^-20 (fp32: of 1), both times lift
        const float unlift = kWide ? (lift > 0.f ? 1.f / lift : 0.f) : 0.25f * __low2float(u2h(s_most));
        const float lo_unit = (kWide ? 1.f : 16777216.f) * unlift, hi_unit = (kWide ? 1.f : 1048576.f) * unlift;
        if (kWide) {  // high and low columns of one head
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
                xa[c] = fmaf(xa[c + 1], 1.f / kLowUp, xa[c]);
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[g][i][c] = fmaf(o[g][i][c + 1], 1.f / kLowUp, o[g][i][c]);
            }
        }
#pragma unroll
        for (int j = 0; j < (kWide ? 1 : 2); ++j) {
            const int col = kWide ? t : 2 * t + j;
            float* dst = mo + (w0 * 8 + col) * kMS;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<float2*>(dst + g * kKv4Group + 8 * r + 2 * i) = make_float2(o[g][i][j] * lo_unit, o[g][i][2 + j] * hi_unit);
            if (r <= G) mx[(w0 * 8 + col) * 4 + (r == G ? 1 : 2 + r)] = xa[j];
            if (r == 0) mx[(w0 * 8 + col) * 4] = ref[j];
        }
        auto put = [&](int col, int d, float val, float l) {
            const int fcol = ct * CT + col, rw = fcol / p.grp, hd = kvh * p.grp + fcol - rw * p.grp;
            static_cast<T*>(p.out)[(int64_t)(sq.row0 + rw) * p.os + (int64_t)hd * D + d] = Act<T>::store(l == 0.f ? 0.f : val / l);  // 0: no key; NaN stays
        };
        if (alone) {
            __syncwarp();
            for (int e = lane; e < cols * D; e += 32) {
                const int col = e / D, d = e % D;
                const float4 y = *reinterpret_cast<const float4*>(mx + col * 4);
                put(col, d, mo[col * kMS + d] + (d < kKv4Group ? y.z : y.w), y.y);
            }
            __syncwarp();
            x += sq.units;
            off += sq.units;
            continue;
        }
        __syncthreads();
        const bool whole = u0 == 0 && u1 == sq.units;
        const int slot = blockIdx.x * 2 + (u0 == 0 ? 1 : 0);
        if (!whole && threadIdx.x == 0 && u0 > 0 && u1 == sq.units)
            ws.meta[blockIdx.x] = {(int)((x - u0) / share), sq.row0, kvh * p.grp, ct * CT, cols, {}};
        for (int e = threadIdx.x; e < cols * D; e += kDecThreads) {
            const int col = e / D, d = e % D;
            float m = -1e30f;
#pragma unroll
            for (int w = 0; w < kDecWarps; ++w) m = fmaxf(m, mx[(w * 8 + col) * 4]);
            float l = 0.f, val = 0.f;
#pragma unroll
            for (int w = 0; w < kDecWarps; ++w) {
                const float4 y = *reinterpret_cast<const float4*>(mx + (w * 8 + col) * 4);
                const float fw = ex2(y.x - m);
                l = fmaf(fw, y.y, l);
                val = fmaf(fw, mo[(w * 8 + col) * kMS + d] + (d < kKv4Group ? y.z : y.w), val);
            }
            if (whole) {
                put(col, d, val, l);
            } else {
                ws.o[((int64_t)slot * 8 + col) * D + d] = val;
                if (d == 0) ws.ml[slot * 8 + col] = make_float2(m, l);
            }
        }
        __syncthreads();  // before the next segment's copies overwrite the sums
        x += u1 - u0;
        off += u1 - u0;
    }
}

// Partial sums of an item that was cut between CTAs, one column per CTA row.
// Bound by latency: a warp's partials are loaded together, four at a time (one
// row over 65531 keys, 37 partials of each item: 33.9 us a call, one after another
// 35.5).
constexpr int kCombineWarps = 8;
template <typename T, int D>
__global__ void __launch_bounds__(kCombineWarps * 32) kv4_combine_kernel(Kv4AttnParams p, DecWork ws) {
    constexpr int E = D / 32, B = 4;
    __shared__ float so[kCombineWarps][D];
    __shared__ float2 sm[kCombineWarps];
    pdl_wait();
    pdl_trigger();
    const DecMeta me = ws.meta[blockIdx.x];
    const int col = blockIdx.y, last = blockIdx.x;
    if (me.first < 0 || col >= me.cols) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = -1e30f, l = 0.f, acc[E] = {};
    for (int c0 = me.first + warp; c0 <= last; c0 += B * kCombineWarps) {
        float2 y[B];
        float val[B][E];
#pragma unroll
        for (int q = 0; q < B; ++q) {
            const int c = c0 + q * kCombineWarps, slot = 2 * c + (c == me.first ? 1 : 0);
            y[q] = make_float2(-1e30f, 0.f);
#pragma unroll
            for (int i = 0; i < E; ++i) val[q][i] = 0.f;
            if (c <= last) {
                y[q] = ws.ml[slot * 8 + col];
                const float* o = ws.o + ((int64_t)slot * 8 + col) * D + lane * E;
                if (E == 4) {
                    const float4 z = *reinterpret_cast<const float4*>(o);
                    val[q][0] = z.x; val[q][1] = z.y; val[q][E - 2] = z.z; val[q][E - 1] = z.w;
                } else {
                    const float2 z = *reinterpret_cast<const float2*>(o);
                    val[q][0] = z.x; val[q][1] = z.y;
                }
            }
        }
#pragma unroll
        for (int q = 0; q < B; ++q) {
            const float nm = fmaxf(m, y[q].x), fa = ex2(m - nm), fb = ex2(y[q].x - nm);
            l = l * fa + y[q].y * fb;
#pragma unroll
            for (int i = 0; i < E; ++i) acc[i] = acc[i] * fa + val[q][i] * fb;
            m = nm;
        }
    }
    if (lane == 0) sm[warp] = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < E; ++i) so[warp][lane * E + i] = acc[i];
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= D) return;
    float mm = -1e30f, ls = 0.f, vs = 0.f;
#pragma unroll
    for (int w = 0; w < kCombineWarps; ++w) mm = fmaxf(mm, sm[w].x);
#pragma unroll
    for (int w = 0; w < kCombineWarps; ++w) {
        const float fw = ex2(sm[w].x - mm);
        ls = fmaf(fw, sm[w].y, ls);
        vs = fmaf(fw, so[w][d], vs);
    }
    const int fcol = me.col0 + col, rw = fcol / p.grp, hd = me.head0 + fcol - rw * p.grp;
    static_cast<T*>(p.out)[(int64_t)(me.row0 + rw) * p.os + (int64_t)hd * D + d] = Act<T>::store(ls == 0.f ? 0.f : vs / ls);
}

}  // namespace amcu

using namespace amcu;

namespace {

int64_t dec_items(const AmcuKv4AttentionArgs* a) {
    const int64_t cols = a->dtype == AMCU_F32 ? dec_cols<float>() : dec_cols<__nv_bfloat16>();
    const int64_t tiles = ceil_div(a->batch.rows * (a->n_q_heads / a->cache.n_kv_heads), cols) + a->batch.n_seq;
    return tiles * a->cache.n_kv_heads;
}

// CTAs of a call: two to an SM, fewer where the page table cannot hold that many units.
int64_t dec_ctas(const AmcuKv4AttentionArgs* a) {
    const int64_t units = ceil_div(a->batch.max_pages * a->cache.page_size, kDecUnit);
    const double bound = (double)dec_items(a) * std::max(1.0, (double)units / kDecMinUnits);
    const int64_t most = 2 * num_sms();
    return bound >= (double)most ? most : (int64_t)bound + 1;
}

// The decode workspace: partial sums and their bookkeeping, 16-byte aligned parts.
size_t dec_layout(int64_t ctas, int64_t d, uint8_t* base, DecWork* w) {
    const size_t o = (size_t)ctas * 16 * d * sizeof(float), ml = (size_t)ctas * 16 * sizeof(float2);
    if (w) {
        w->o = reinterpret_cast<float*>(base);
        w->ml = reinterpret_cast<float2*>(base + o);
        w->meta = reinterpret_cast<DecMeta*>(base + o + ml);
    }
    return o + ml + (size_t)ctas * sizeof(DecMeta);
}

template <typename T, int D>
void launch_decode(const Kv4AttnParams& p, const DecWork& w, unsigned ctas, cudaStream_t s) {
    constexpr int smem = dec_smem_bytes<D>();
    set_func_attr_once(reinterpret_cast<const void*>(&kv4_decode_kernel<T, D>),
                       cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    launch_pdl(kv4_decode_kernel<T, D>, dim3(ctas), dim3(kDecThreads), smem, s, p, w);
    launch_pdl(kv4_combine_kernel<T, D>, dim3(ctas, dec_cols<T>()), dim3(kCombineWarps * 32), 0, s, p, w);
}

}  // namespace

extern "C" size_t amcu_attn_kv4_workspace_bytes(const AmcuKv4AttentionArgs* a) {
    if (!a || a->batch.rows <= 0 || a->batch.n_seq <= 0 || a->n_q_heads <= 0 || a->cache.n_kv_heads <= 0 ||
        a->batch.max_pages < 0 || a->cache.page_size <= 0)
        return 0;
    return dec_layout(dec_ctas(a), a->cache.head_dim, nullptr, nullptr);
}

extern "C" am_status_code amcu_attn_kv4(const AmcuKv4AttentionArgs* a, void* stream) {
    clear_error();
    AMCU_REQUIRE(a != nullptr, "amcu_attn_kv4: null args");
    Kv4AttnParams p;
    am_status_code st = kv4_check("amcu_attn_kv4", a->cache, a->batch, &p.v);
    if (st != AM_STATUS_OK) return st;
    AMCU_REQUIRE(a->dtype == AMCU_F32 || a->dtype == AMCU_BF16, "amcu_attn_kv4: dtype must be f32 or bf16");
    AMCU_REQUIRE(a->n_q_heads > 0 && a->n_q_heads <= 65536 && a->n_q_heads % a->cache.n_kv_heads == 0,
                 "amcu_attn_kv4: n_q_heads must be a positive multiple of n_kv_heads");
    AMCU_REQUIRE(a->scale >= 0.f && a->scale < INFINITY, "amcu_attn_kv4: scale must be finite and not negative");
    AMCU_REQUIRE(a->batch.rows * a->n_q_heads <= (1 << 28), "amcu_attn_kv4: rows * n_q_heads must be at most 2^28");
    if (a->batch.rows == 0 || a->batch.n_seq == 0) return AM_STATUS_OK;
    AMCU_REQUIRE(a->q && a->out, "amcu_attn_kv4: null pointer");
    p.q = a->q;
    p.out = a->out;
    p.qs = a->q_stride;
    p.os = a->out_stride;
    p.nq = (int)a->n_q_heads;
    p.grp = (int)(a->n_q_heads / a->cache.n_kv_heads);
    p.scale = a->scale > 0.f ? a->scale : 1.f / sqrtf((float)a->cache.head_dim);
    p.vec = aligned(a->q, 16) && aligned(a->out, 16) && a->q_stride % 8 == 0 && a->out_stride % 8 == 0;
    const bool prompts = a->dtype == AMCU_BF16 && kv4_prefill_wanted(p.v, p.grp);
    const size_t need = amcu_attn_kv4_workspace_bytes(a);
    AMCU_REQUIRE(a->workspace && a->workspace_size >= need && aligned(a->workspace, 16),
                 "amcu_attn_kv4: needs a 16-byte aligned workspace of %zu bytes", need);
    DecWork w;
    const unsigned ctas = (unsigned)dec_ctas(a);
    dec_layout(ctas, a->cache.head_dim, static_cast<uint8_t*>(a->workspace), &w);
    w.items = dec_items(a);
    const bool f32 = a->dtype == AMCU_F32;
    cudaStream_t s = as_stream(stream);
    if (prompts) return kv4_prefill_launch(p, a->cache.head_dim, s);
    if (a->cache.head_dim == 64)
        f32 ? launch_decode<float, 64>(p, w, ctas, s) : launch_decode<__nv_bfloat16, 64>(p, w, ctas, s);
    else
        f32 ? launch_decode<float, 128>(p, w, ctas, s) : launch_decode<__nv_bfloat16, 128>(p, w, ctas, s);
    return check_launch("amcu_attn_kv4");
}
