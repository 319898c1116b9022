// Causal attention of prompts over the 4-bit paged KV cache on the
// 5th-generation tensor cores (tcgen05 + TMEM), bf16.
//
// The rows of a product are (token, q head) pairs of one kv head, 256 to a CTA
// (two tiles of 128), so a key tile is dequantised once for all of the group's
// heads. Per key tile of 128:
//   S = Q K^T   A = Q (shared memory, fp16, scaled by a power of two per row),
//               B = K, S in tensor memory (one lane per row)
//   P = 2^(S f - ref) by one thread per row, in fp16 over S's own columns
//   O += P V    A = P (tensor memory), B = V^T, O in tensor memory
// Warps 0-3 and 4-7 are the softmax of the two row tiles, warps 8-11 turn K's
// codes into fp16 tiles and warps 12-15 V's, warp 16 issues the MMAs and owns the
// tensor memory. While one row tile's softmax runs, the other's products do, and
// O's first 64 keys are added while the other 64 are weighed (353 against 363 us,
// d = 64 280 against 288, 3 x 100 rows over 5000 keys of 28 / 4 heads 101 against
// 106). (An
// issuing warp for each row tile measured 469 against 432 us, the issuer as the
// block's first warp 442, polling waits with a sleep 472: 2 x 2048 rows over 8192
// keys, 32 / 8 heads of 128.)
//
// K tile and V^T tile have the 128-byte-swizzled K-major layout. A word of 8
// codes is one 16-byte chunk of a K row; its nibbles come out in the order
// 0 4 1 5 2 6 3 7, and Q's elements are stored in that order too. V is read
// across 8 tokens, so a chunk of V^T is 8 keys of one element. Values are
// m + s c in fp16: (1024 + c) - 1024 exactly, then one fused multiply-add
// rounded once to 11 bits (an element beyond fp16 becomes 65504).
//
// The softmax reference of a row lies 2^6 to 2^7 below the largest score when it is
// set, and moves only when a score passes it by 2^15 (p is in fp16), and to a whole
// power of two: the sum, O and what the tile has of P already are then rescaled
// without a rounding (P where it stays normal). So the scores are read once, without
// knowing their tile's maximum first. (With the reference at the largest score itself
// p of 2^-20 kept 4 bits: 3% of a row of many such keys under one that has most of the
// mass.)
//
// Waits are bounded: one that runs out records an error code, and the CTA goes
// through its control flow without waiting again.
#include "kv4.cuh"
#include "tcgen05.cuh"

namespace amcu {

constexpr int kPfRows = 256, kPfKeys = 128;
constexpr int kPfThreads = 17 * 32;
constexpr int kPfMmaWarp = 16;
constexpr int kPfDqThreads = 128;
constexpr int32_t kErrKv4Wait = 0x501;
constexpr float kPfLog2e = 1.4426950408889634f;
// A score may pass the largest so far by kPfLift before the reference moves, to
// kPfHead below the new largest: p is up to 2^15, and an fp16 normal, rounded to 11 bits,
// down to 2^-20 of the largest one (2^-31 is still counted).
constexpr float kPfLift = 8.f, kPfHead = 7.f;

template <int D>
struct PfLayout {  // shared memory, bytes
    static constexpr int kQ = 128 * D * 2;            // one row tile of Q
    static constexpr int kK = kPfKeys * D * 2;        // a K or V^T stage
    static constexpr int kVPitch = 8 * D / 2 + 16;    // 8 tokens of V codes
    static constexpr int kRawV = kPfKeys / 8 * kVPitch;
    static constexpr int kVParPitch = 8 * D / 16 + 16;
    static constexpr int kParV = kPfKeys / 8 * kVParPitch;
    static constexpr int oQ = 0, oK = oQ + 2 * kQ, oV = oK + 2 * kK, oRawV = oV + 2 * kK, oParV = oRawV + 2 * kRawV,
                         oBar = oParV + 2 * kParV;
    // Registers from the dequantising warps to the softmax: 8 x kDqRegs + 8 x (192 -
    // kDqRegs) + 96 = 17 x 96 a lane. As many as neither spills with (2 x 2048 rows
    // over 8192 keys, 32 / 8 heads: 329 us of d = 128 with 80, 345 with 72; 271 us of
    // d = 64 with 72, 273 with 80).
    static constexpr int kDqRegs = D == 128 ? 80 : 72;
    static constexpr int kTotal = oBar + 256 + 1024;  // + alignment slack
};

// Offset of 16-byte chunk c of row r in a K-major tile of ROWS rows: halves of
// 64 elements (128 bytes a row), 16-byte chunks XOR-swizzled by row % 8.
template <int ROWS>
__device__ __forceinline__ uint32_t pf_sw(int r, int c) {
    return (uint32_t)((c >> 3) * (ROWS * 128) + (r >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void tc_ld32_issue(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
            "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
              "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
              "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
              "=r"(r[30]), "=r"(r[31])
            : "r"(taddr));
}
// Waits for this thread's tcgen05.ld; the registers are tied so that nothing reads them earlier.
__device__ __forceinline__ void tc_ld32_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
// 32 lanes x 16 columns, complete on return.
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr)
            : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    tc_st_32x32b_x32(taddr, r);
}
// The products and commits are issued by one elected lane of a warp that runs
// its loop as a whole.
__device__ __forceinline__ void pf_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
            "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
            " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc)
            : "memory");
}
__device__ __forceinline__ void pf_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
            "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
            " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
            "r"(a), "l"(b), "r"(idesc), "r"(acc)
            : "memory");
}
__device__ __forceinline__ void pf_commit(uint64_t* bar) {
    asm volatile(
            "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
            " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar))
            : "memory");
}
__device__ __forceinline__ float pf_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pf_h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 pf_u2h(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void pf_cp16(void* dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

// m + s c of a register's two codes: low nibbles in bits 0-3 of the halves, or in bits 4-7.
__device__ __forceinline__ __half2 pf_value(uint32_t w, bool high, __half2 s, __half2 m) {
    const __half2 c = high ? __hadd2(pf_u2h((w & 0x00F000F0u) | 0x54005400u), __float2half2_rn(-64.f))
                           : __hadd2(pf_u2h((w & 0x000F000Fu) | 0x64006400u), __float2half2_rn(-1024.f));
    return __hfma2(c, s, m);
}

template <int D>
__global__ void __launch_bounds__(kPfThreads, 1) kv4_prefill_kernel(Kv4AttnParams p, int32_t* err) {
    using L = PfLayout<D>;
    constexpr int G = D / kKv4Group, WPR = D / 8;  // groups, words per row
    extern __shared__ uint8_t pf_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pf_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bar = reinterpret_cast<uint64_t*>(sm + L::oBar);
    uint64_t *k_full = bar, *k_empty = bar + 2, *v_full = bar + 4, *v_empty = bar + 6, *s_full = bar + 8,
             *p_full = bar + 10, *o_full = bar + 12, *q_full = bar + 14, *p_half = bar + 16, *o_half = bar + 18;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 20);
    int* s_item = reinterpret_cast<int*>(bar + 21);  // b, item of b
    int* s_nan = reinterpret_cast<int*>(bar + 22);   // first key whose group of V is NaN

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();

    // ---- this CTA's item: sequence, kv head and row tile
    const Kv4View& v = p.v;
    {
        const int row_first = v.row_start[0], row_end = v.row_start[v.n_seq];
        auto cost = [&](int b) {
            int r0, n;
            kv4_rows(v, b, r0, n);
            return ((int64_t)n * p.grp + kPfRows - 1) / kPfRows * v.nkv;
        };
        int64_t total, off;
        int b;
        const bool have = kv4_share<kPfThreads>(v.n_seq, [&](int64_t) { return (int64_t)blockIdx.x; }, cost, total, b, off);
        kv4_zero_uncovered<__nv_bfloat16, kPfThreads>(v, row_first, row_end, p.out, p.os, p.nq * D);
        if ((int64_t)blockIdx.x >= total) return;
        if (have) {
            s_item[0] = b;
            s_item[1] = (int)off;
        }
    }
    if (warp == kPfMmaWarp) {
        if (lane == 0) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&k_full[i], 4);
                mbar_init(&k_empty[i], 1);
                mbar_init(&v_full[i], 4);
                mbar_init(&v_empty[i], 1);
                mbar_init(&s_full[i], 1);
                mbar_init(&p_full[i], 4);
                mbar_init(&o_full[i], 1);
                mbar_init(&q_full[i], 4);
                mbar_init(&p_half[i], 4);
                mbar_init(&o_half[i], 1);
            }
            fence_mbar_init();
            s_nan[0] = s_nan[1] = 0x7fffffff;
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const int b = s_item[0];
    int row0, n;
    kv4_rows(v, b, row0, n);
    const int nt_rows = (int)(((int64_t)n * p.grp + kPfRows - 1) / kPfRows);
    const int tile = nt_rows - 1 - s_item[1] / v.nkv, kvh = s_item[1] % v.nkv;  // the longest rows first
    const int ctx = v.ctx_len[b];
    const int cap = (int)min((int64_t)max(ctx, 0), (int64_t)v.max_pages << v.page_shift);
    const int m0 = tile * kPfRows, m_end = min(m0 + kPfRows, n * p.grp);  // flat rows: token * grp + head
    const int lim_last = min(ctx - n + (m_end - 1) / p.grp, cap - 1);     // last key that any row sees
    const int nt = lim_last >= 0 ? lim_last / kPfKeys + 1 : 0;            // key tiles
    const int ni = m_end - m0 > 128 ? 2 : 1;                              // row tiles
    if ((ctx > cap || ctx < n) && v.status && threadIdx.x == 0) *v.status = (int32_t)AM_STATUS_OUT_OF_RANGE;

    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    bool ok = true;
    auto wait = [&](uint64_t* w, uint32_t parity) {
        if (ok && !mbar_wait(w, parity)) {
            ok = false;
            record_device_error(err, kErrKv4Wait);
        }
    };

    if (warp == kPfMmaWarp) {
        // ---- MMA issuer
        // nt and ni the same in every lane also to the compiler: branches and descriptors stay uniform
        const int nt_ = __shfl_sync(0xffffffffu, nt, 0), ni_ = __shfl_sync(0xffffffffu, ni, 0);
        if (nt_ > 0) {
            constexpr uint32_t id_s = tc_idesc_f16(128, kPfKeys), id_o = tc_idesc_f16(128, D);
            // descriptors of the tiles' starts; a K step adds to the address field (16-byte
            // units). Built anew for every MMA they cost this one thread more time than
            // the MMA takes (152 cycles against 64).
            const uint64_t q_desc = tc_desc_sw128(smem_u32(sm + L::oQ)), k_desc = tc_desc_sw128(smem_u32(sm + L::oK)),
                           v_desc = tc_desc_sw128(smem_u32(sm + L::oV));
            auto qk = [&](int i, int j) {
                const uint64_t a = q_desc + (uint64_t)(i * (L::kQ >> 4)), bb = k_desc + (uint64_t)((j & 1) * (L::kK >> 4));
                const uint32_t d = tmem + (uint32_t)(128 * i);
#pragma unroll
                for (int s = 0; s < D / 16; ++s) {
                    constexpr int kHalf = 16384 >> 4;
                    const uint64_t o = (uint64_t)((s >> 2) * kHalf + (s & 3) * 2);
                    pf_mma_ss(d, a + o, bb + o, id_s, s != 0);
                }
            };
            wait(&k_full[0], 0);
            for (int i = 0; i < ni_; ++i) {
                wait(&q_full[i], 0);
                tc_fence_after();
                qk(i, 0);
                pf_commit(&s_full[i]);
            }
            pf_commit(&k_empty[0]);
            for (int j = 0; j < nt_; ++j) {
                const bool more = j + 1 < nt_;
                wait(&v_full[j & 1], (j >> 1) & 1);
                if (more) wait(&k_full[(j + 1) & 1], ((j + 1) >> 1) & 1);
                for (int i = 0; i < ni_; ++i) {
                    const uint64_t bb = v_desc + (uint64_t)((j & 1) * (L::kK >> 4));
                    const uint32_t d = tmem + 256u + (uint32_t)(128 * i), a = tmem + (uint32_t)(128 * i);
                    constexpr int kHalf = (D * 128) >> 4;  // of V^T: 64 keys
                    // the first 64 keys' products run beside the weights of the others
                    wait(&p_half[i], j & 1);
                    tc_fence_after();
#pragma unroll
                    for (int s = 0; s < kPfKeys / 32; ++s)
                        pf_mma_ts(d, a + (uint32_t)(8 * s), bb + (uint64_t)(s * 2), id_o, s != 0 || j != 0);
                    pf_commit(&o_half[i]);
                    wait(&p_full[i], j & 1);
                    tc_fence_after();
#pragma unroll
                    for (int s = kPfKeys / 32; s < kPfKeys / 16; ++s)
                        pf_mma_ts(d, a + (uint32_t)(8 * s), bb + (uint64_t)(kHalf + (s & 3) * 2), id_o, 1);
                    if (more) qk(i, j + 1);
                    pf_commit(more ? &s_full[i] : &o_full[i]);
                }
                pf_commit(&v_empty[j & 1]);
                if (more) pf_commit(&k_empty[(j + 1) & 1]);
            }
        }
        __syncwarp();
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kDqRegs));
        const int t = threadIdx.x & 127;
        const int kmax = lim_last + 1;    // keys past it are zeros
        // pages of a tile's eight 16-key blocks, in lanes 0-7; fetched two tiles ahead
        // (positions below kmax are inside the page table) and checked when used
        auto pages_of = [&](int j) {
            const int key = j * kPfKeys + lane * 16;
            return lane < 8 && key < kmax ? v.table[b * v.table_stride + (key >> v.page_shift)] : 0;
        };
        auto checked = [&](int pg) {
            if (pg >= 0 && pg < v.num_pages) return pg;
            if (v.status) *v.status = (int32_t)AM_STATUS_OUT_OF_RANGE;
            return -1;
        };
        if (warp < 12) {
            // ---- K codes to fp16: row t of the tile, read straight into registers a tile ahead
            uint32_t raw[WPR], par[G];
            auto load = [&](int j, int pg) {
                const int key = j * kPfKeys + t;
                int page = __shfl_sync(0xffffffffu, pg, t >> 4);
                if (key >= kmax) page = -1;
                const int slot = key & ((1 << v.page_shift) - 1);
#pragma unroll
                for (int i = 0; i < WPR; ++i) raw[i] = 0;
#pragma unroll
                for (int g = 0; g < G; ++g) par[g] = 0;
                if (page >= 0) {
                    const uint4* src = reinterpret_cast<const uint4*>(v.kc + kv4_code_off<D>(v, page, kvh, slot));
#pragma unroll
                    for (int c = 0; c < WPR / 4; ++c) {
                        const uint4 y = src[c];
                        raw[4 * c] = y.x; raw[4 * c + 1] = y.y; raw[4 * c + 2] = y.z; raw[4 * c + 3] = y.w;
                    }
                    const uint32_t* ps = reinterpret_cast<const uint32_t*>(v.kp + kv4_param_off<D>(v, page, kvh, slot));
#pragma unroll
                    for (int g = 0; g < G; ++g) par[g] = ps[g];
                }
            };
            int pages = pages_of(0), ahead = pages_of(1);
            if (nt > 0) load(0, checked(pages));
            pages = ahead;
            ahead = pages_of(2);
            for (int j = 0; j < nt; ++j) {
                const int s = j & 1;
                if (j >= 2) wait(&k_empty[s], ((j >> 1) & 1) ^ 1);
                __half2 sc[G], mn[G];
                bool big = false;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const __half2 y = pf_u2h(par[g]);
                    sc[g] = __low2half2(y);
                    mn[g] = __high2half2(y);
                    big |= __half2float(__high2half(y)) + 15.f * __half2float(__low2half(y)) >= 65504.f;
                }
                uint8_t* K = sm + L::oK + s * L::kK;
#pragma unroll
                for (int i = 0; i < WPR; ++i) {
                    const int g = i % G;
                    __half2 h[4] = {pf_value(raw[i], false, sc[g], mn[g]), pf_value(raw[i], true, sc[g], mn[g]),
                                    pf_value(raw[i] >> 8, false, sc[g], mn[g]), pf_value(raw[i] >> 8, true, sc[g], mn[g])};
                    if (big) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) h[q] = __hmin2(h[q], __float2half2_rn(65504.f));
                    }
                    *reinterpret_cast<uint4*>(K + pf_sw<kPfKeys>(t, 8 * g + i / G)) =
                            make_uint4(pf_h2u(h[0]), pf_h2u(h[1]), pf_h2u(h[2]), pf_h2u(h[3]));
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[s]);
                if (j + 1 < nt) load(j + 1, checked(pages));
                pages = ahead;
                ahead = pages_of(j + 3);
            }
        } else {
            // ---- V codes to fp16, transposed: tokens 8 tg .. + 7, words of 8 elements of one or both groups
            const int w = warp & 3;
            constexpr int CPT = D / 32;       // 16-byte chunks of codes per token
            auto load = [&](int j, int pg) {
                uint8_t* codes = sm + L::oRawV + (j & 1) * L::kRawV;
                uint8_t* params = sm + L::oParV + (j & 1) * L::kParV;
                if (j < nt) {
#pragma unroll
                    for (int i = 0; i < CPT; ++i) {
                        const int e = i * kPfDqThreads + t, tk = e / CPT, c = e % CPT, key = j * kPfKeys + tk;
                        int page = __shfl_sync(0xffffffffu, pg, tk >> 4);
                        if (key >= kmax) page = -1;
                        const int slot = key & ((1 << v.page_shift) - 1);
                        const uint8_t* src = v.vc + (page >= 0 ? kv4_code_off<D>(v, page, kvh, slot) + 16 * c : 0);
                        pf_cp16(codes + (tk >> 3) * L::kVPitch + (tk & 7) * (D / 2) + 16 * c, src, page >= 0 ? 16u : 0u);
                    }
                    if (t < kPfKeys * D / 256) {  // parameters: 16 bytes are 2 (D = 128) or 4 tokens; whole warps
                        constexpr int TPC = 256 / D;
                        const int tk = t * TPC, key = j * kPfKeys + tk;
                        const int page = __shfl_sync(0xffffffffu, pg, tk >> 4);
                        const int slot = key & ((1 << v.page_shift) - 1);
                        const uint8_t* src = v.vp + (page >= 0 ? kv4_param_off<D>(v, page, kvh, slot) : 0);
                        // tokens past the last key may hold anything: leave them out
                        const int live = min(max(kmax - key, 0), TPC);
                        pf_cp16(params + (tk >> 3) * L::kVParPitch + (tk & 7) * (D / 16), src,
                                page >= 0 ? (uint32_t)(live * (D / 16)) : 0u);
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            int pages = pages_of(0), ahead = pages_of(1);
            load(0, checked(pages));
            pages = ahead;
            ahead = pages_of(2);
            for (int j = 0; j < nt; ++j) {
                const int s = j & 1;
                load(j + 1, checked(pages));  // its buffer was read out before the barrier of tile j - 1's end
                pages = ahead;
                ahead = pages_of(j + 3);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                named_bar_sync(1, kPfDqThreads);
                if (j >= 2) wait(&v_empty[s], ((j >> 1) & 1) ^ 1);
                const int tg = (lane & 7) + 8 * (w & 1), q8 = (lane >> 3) + 4 * (w >> 1);  // token group, word (pair)
                const uint8_t* src = sm + L::oRawV + s * L::kRawV + tg * L::kVPitch + q8 * (4 * G);
                const uint8_t* ps = sm + L::oParV + s * L::kParV + tg * L::kVParPitch;
                uint8_t* V = sm + L::oV + s * L::kK;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    __half2 sc[4], mn[4];
                    __half2 top;  // largest element of the tokens' groups
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const uint32_t p0 = lds_u32(ps + (2 * y) * (4 * G) + 4 * g), p1 = lds_u32(ps + (2 * y + 1) * (4 * G) + 4 * g);
                        sc[y] = pf_u2h(__byte_perm(p0, p1, 0x5410));
                        mn[y] = pf_u2h(__byte_perm(p0, p1, 0x7632));
                        const __half2 most = __hfma2(__float2half2_rn(15.f), sc[y], mn[y]);
                        top = y == 0 ? most : __hmax2_nan(top, most);
                    }
                    const bool big = !__hblt2(top, pf_u2h(0x7c007c00u));  // beyond fp16, or NaN
                    // a NaN becomes 65504 below, as 0 times it would reach rows that do not see the
                    // key; those that do take their NaN at the end (each thread looks at one token)
                    if (big) {
                        const __half2 par = pf_u2h(lds_u32(ps + q8 * (4 * G) + 4 * g));
                        if (__hneu2_mask(par, par)) atomicMin(&s_nan[g], j * kPfKeys + 8 * tg + q8);
                    }
                    uint32_t cw[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) cw[i] = lds_u32(src + i * (D / 2) + 4 * g);
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        uint32_t ww[4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) ww[y] = __byte_perm(cw[2 * y], cw[2 * y + 1], part ? 0x7632 : 0x5410);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {  // element 4 part + e
                            __half2 h[4];
#pragma unroll
                            for (int y = 0; y < 4; ++y) h[y] = pf_value(e < 2 ? ww[y] : ww[y] >> 8, e & 1, sc[y], mn[y]);
                            if (big) {
#pragma unroll
                                for (int y = 0; y < 4; ++y) h[y] = __hmin2(h[y], __float2half2_rn(65504.f));
                            }
                            *reinterpret_cast<uint4*>(V + pf_sw<D>(64 * g + 8 * q8 + 4 * part + e, tg)) =
                                    make_uint4(pf_h2u(h[0]), pf_h2u(h[1]), pf_h2u(h[2]), pf_h2u(h[3]));
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[s]);
                named_bar_sync(1, kPfDqThreads);  // the codes of this tile are read out
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(192 - L::kDqRegs));
        if (warp / 4 < ni) {
        // ---- softmax of row tile i: thread = row
        const int i = warp >> 2;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lane_base + (uint32_t)(128 * i), to = tmem + lane_base + 256u + (uint32_t)(128 * i);
        const int m = m0 + threadIdx.x;
        const bool row_live = m < m_end;
        const int tok = row_live ? m / p.grp : 0, head = kvh * p.grp + (row_live ? m - tok * p.grp : 0);
        const int lim = row_live ? min(ctx - n + tok, cap - 1) : -1;  // the row's last key
        const int64_t q_off = (int64_t)(row0 + tok) * p.qs + (int64_t)head * D;
        // Q into shared memory, 16 bytes a lane, CPR lanes to a row
        float f;  // 2^e scale log2(e) of this thread's row
        {
            constexpr int CPR = D / 8, RPW = 32 / CPR;  // chunks of a row, rows at a time
            uint8_t* Q = sm + L::oQ + i * L::kQ;
            const int c = lane % CPR;
            uint32_t eb_mine = 1;
            constexpr int B = D == 128 ? 4 : 8;  // loads in flight
#pragma unroll 1
            for (int st0 = 0; st0 < 32 / RPW; st0 += B) {
                uint32_t w[B][4];
#pragma unroll
                for (int u = 0; u < B; ++u) {
                    const int src = (st0 + u) * RPW + lane / CPR;  // lane whose row this is
                    const int64_t off = __shfl_sync(0xffffffffu, q_off, src);
                    const bool live = __shfl_sync(0xffffffffu, (int)row_live, src);
                    const __nv_bfloat16* qp = static_cast<const __nv_bfloat16*>(p.q) + off + 8 * c;
                    w[u][0] = w[u][1] = w[u][2] = w[u][3] = 0;
                    if (live && p.vec) {
                        const uint4 y = *reinterpret_cast<const uint4*>(qp);
                        w[u][0] = y.x; w[u][1] = y.y; w[u][2] = y.z; w[u][3] = y.w;
                    } else if (live) {
                        const uint16_t* qe = reinterpret_cast<const uint16_t*>(qp);
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[u][k] = (uint32_t)qe[2 * k] | ((uint32_t)qe[2 * k + 1] << 16);
                    }
                }
#pragma unroll
                for (int u = 0; u < B; ++u) {
                    float e[8];
                    uint32_t amax = 0;  // bits of the largest |q|: NaN above infinity above the rest
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        e[2 * k] = __uint_as_float(w[u][k] << 16);
                        e[2 * k + 1] = __uint_as_float(w[u][k] & 0xffff0000u);
                        amax = max(amax, max(__float_as_uint(e[2 * k]) & 0x7fffffffu, __float_as_uint(e[2 * k + 1]) & 0x7fffffffu));
                    }
#pragma unroll
                    for (int o = CPR / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                    const uint32_t eb = min(max(amax >> 23, 1u), 253u);
                    // a row with an element that is no number or infinite has no softmax: all its scores are NaN
                    const float inv = __uint_as_float(amax < 0x7f800000u ? (254u - eb) << 23 : 0x7fc00000u);
#pragma unroll
                    for (int k = 0; k < 8; ++k) e[k] *= inv;
                    // in the order 0 4 1 5 2 6 3 7
                    *reinterpret_cast<uint4*>(Q + pf_sw<128>((warp & 3) * 32 + (st0 + u) * RPW + lane / CPR, c)) =
                            make_uint4(pf_h2u(__floats2half2_rn(e[0], e[4])), pf_h2u(__floats2half2_rn(e[1], e[5])),
                                       pf_h2u(__floats2half2_rn(e[2], e[6])), pf_h2u(__floats2half2_rn(e[3], e[7])));
                    const uint32_t got = __shfl_sync(0xffffffffu, eb, (lane % RPW) * CPR);
                    if (lane / RPW == st0 + u) eb_mine = got;
                }
            }
            f = __uint_as_float(eb_mine << 23) * p.scale * kPfLog2e;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[i]);
        }
        // tiles below `full` need no mask in this warp
        const int full = __reduce_min_sync(0xffffffffu, row_live ? lim + 1 : 0x7fffffff) / kPfKeys;
        float ref = -1e30f;  // log2 units; a whole number once a key was seen
        uint64_t l2 = f2_pack(0.f, 0.f), l3 = l2;
        // pages that are none mask their 16 keys: looked up a tile ahead, one block per
        // lane (positions up to lim_last are inside the page table)
        auto page_at = [&](int j) {  // past the last key: a valid one
            const int key = j * kPfKeys + lane * 16;
            return lane < 8 && key <= lim_last ? v.table[b * v.table_stride + (key >> v.page_shift)] : 0;
        };
        int page = page_at(0);
        const uint64_t f2 = f2_pack(f, f);
        for (int j = 0; j < nt; ++j) {
            const unsigned bad = __ballot_sync(0xffffffffu, page < 0 || page >= v.num_pages);
            page = page_at(j + 1);
            wait(&s_full[i], j & 1);
            tc_fence_after();
            if (j >= full || bad != 0) {  // masked scores become -inf in place
#pragma unroll 1
                for (int q = 0; q < 4; ++q) {
                    uint32_t x[32];
                    tc_ld32_issue(ts + 32 * q, x);
                    tc_ld32_wait(x);
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (j * kPfKeys + 32 * q + c > lim || ((bad >> (2 * q + (c >> 4))) & 1u)) x[c] = 0xff800000u;
                    tc_st32(ts + 32 * q, x);
                }
            }
            uint32_t x[2][32];
            tc_ld32_issue(ts, x[0]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t(&z)[32] = x[q & 1];
                tc_ld32_wait(z);
                // the reference moves only for a score that passes the largest so far by kPfLift
                float m4[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) m4[c] = fmaxf(__uint_as_float(z[c]), __uint_as_float(z[c + 4]));
#pragma unroll
                for (int c = 8; c < 32; c += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        m4[k] = fmaxf(fmaxf(m4[k], __uint_as_float(z[c + k])), __uint_as_float(z[c + k + 4]));
                const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * f;
                if (__any_sync(0xffffffffu, mx > ref + (kPfHead + kPfLift))) {
                    // to a whole number, so that every rescaling is by a power of two
                    const float nref = mx > ref + kPfHead ? ceilf(fminf(mx, 1e30f)) - kPfHead : ref, corr = pf_ex2(ref - nref);
                    ref = nref;
                    l2 = f2_fma(l2, f2_pack(corr, corr), f2_pack(0.f, 0.f));
                    l3 = f2_fma(l3, f2_pack(corr, corr), f2_pack(0.f, 0.f));
                    const __half2 corr2 = __float2half2_rn(corr);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    if (q & 1) {  // this half's P so far: no product has taken it
                        uint32_t y[16];
                        tc_ld16(ts + 16 * (q - 1), y);
#pragma unroll
                        for (int c = 0; c < 16; ++c) y[c] = pf_h2u(__hmul2(pf_u2h(y[c]), corr2));
                        tc_st_32x32b_x16(ts + 16 * (q - 1), y);
                    }
                    // products of earlier tiles are complete (this tile's scores were
                    // committed after them), those of its first half have to be waited for
                    if (q >= 2) {
                        wait(&o_half[i], j & 1);
                        tc_fence_after();
                    }
                    if (j > 0 || q >= 2) {
#pragma unroll 1
                        for (int k = 0; k < D / 16; ++k) {
                            uint32_t y[16];
                            tc_ld16(to + 16 * k, y);
#pragma unroll
                            for (int c = 0; c < 16; ++c) y[c] = __float_as_uint(__uint_as_float(y[c]) * corr);
                            tc_st_32x32b_x16(to + 16 * k, y);
                        }
                    }
                }
                if (q < 3) tc_ld32_issue(ts + 32 * (q + 1), x[(q + 1) & 1]);
                const uint64_t r2 = f2_pack(-ref, -ref);
                uint32_t pk16[16];
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const uint64_t y = f2_fma(f2_pack(__uint_as_float(z[2 * c]), __uint_as_float(z[2 * c + 1])), f2, r2);
                    float a, bb;
                    f2_unpack(y, a, bb);
                    a = pf_ex2(a);
                    bb = pf_ex2(bb);
                    if (c & 1) l3 = f2_add(l3, f2_pack(a, bb));
                    else l2 = f2_add(l2, f2_pack(a, bb));
                    pk16[c] = pf_h2u(__floats2half2_rn(a, bb));
                }
                // columns 16 q .. + 15 hold scores that are in registers by now
                tc_st_32x32b_x16_nowait(ts + 16 * q, pk16);
                if (q & 1) {
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(q == 1 ? &p_half[i] : &p_full[i]);
                }
            }
        }
        // ---- out = O / l
        float la, lb;
        f2_unpack(f2_add(l2, l3), la, lb);
        const float l = la + lb, inv = 1.f / l;
        const bool any = nt > 0 && l != 0.f;  // a key was seen; NaN stays
        if (nt > 0) {
            wait(&v_full[(nt - 1) & 1], ((nt - 1) >> 1) & 1);  // s_nan is complete
            wait(&o_full[i], 0);
            tc_fence_after();
        }
        __nv_bfloat16* op = static_cast<__nv_bfloat16*>(p.out) + (int64_t)(row0 + tok) * p.os + (int64_t)head * D;
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
            uint32_t x[32];
            if (nt > 0) {
                tc_ld32_issue(to + 32 * q, x);
                tc_ld32_wait(x);
            }
            uint32_t y[16];
            const float mul = s_nan[q / 2] <= lim ? __uint_as_float(0x7fc00000u) : inv;
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                const float a = any ? __uint_as_float(x[2 * c]) * mul : 0.f;
                const float bb = any ? __uint_as_float(x[2 * c + 1]) * mul : 0.f;
                __nv_bfloat162 h = __floats2bfloat162_rn(a, bb);
                y[c] = *reinterpret_cast<uint32_t*>(&h);
            }
            if (!row_live || !ok) continue;
            if (p.vec) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *reinterpret_cast<uint4*>(op + 32 * q + 8 * c) = make_uint4(y[4 * c], y[4 * c + 1], y[4 * c + 2], y[4 * c + 3]);
            } else {
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    reinterpret_cast<uint16_t*>(op)[32 * q + c] = (uint16_t)(y[c / 2] >> (16 * (c & 1)));
            }
        }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kPfMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int D>
static void launch_prefill(const Kv4AttnParams& p, unsigned ctas, cudaStream_t s) {
    set_func_attr_once(reinterpret_cast<const void*>(&kv4_prefill_kernel<D>), cudaFuncAttributeMaxDynamicSharedMemorySize,
                       PfLayout<D>::kTotal);
    launch_pdl(kv4_prefill_kernel<D>, dim3(ctas), dim3(kPfThreads), PfLayout<D>::kTotal, s, p, device_error_word());
}

bool kv4_prefill_wanted(const Kv4View& v, int64_t grp) {
    // A wave of row tiles (one to an SM) takes about as long as 2.5 eight-column
    // tiles of the other kernel on every SM: this kernel once there are more columns.
    // Measured (us, this / the other), 32 / 8 heads of 128, one sequence: 4096 keys, 64
    // rows 76 / 52, 96 rows 77 / 73, 128 rows 77 / 89, 256 rows 77 / 159; 1000 keys, 64
    // rows 28 / 30, 128 rows 28 / 44; four sequences of 16 rows over 4096 keys 69 / 53, of
    // 32 70 / 89. Groups of 1, 7 and 8 heads have the same border in columns: 192 rows of
    // 16 / 16 heads 76 / 73, 128 of 28 / 4 77 / 81, 64 of 64 / 8 78 / 89 (4096 keys).
    // The rule knows no context, though this kernel takes as long for one row tile as
    // for a wave of them: 96 rows of 32 / 8 heads over 32768 keys 532 / 378. With heads of
    // 64 the other kernel is the faster one for up to half as many columns again: 96 rows
    // over 4096 keys 64 / 49, over 32768 458 / 245, 192 rows 65 / 81 and 459 / 473.
    const int64_t cols = v.rows * grp, tiles = (cols / kPfRows + v.n_seq) * v.nkv, sms = num_sms();
    return ceil_div(cols, 8) * v.nkv * 2 > 5 * sms * ceil_div(tiles, sms);
}

am_status_code kv4_prefill_launch(const Kv4AttnParams& p, int64_t d, cudaStream_t s) {
    const int64_t ctas = ((int64_t)p.v.rows * p.grp / kPfRows + p.v.n_seq) * p.v.nkv;  // at least as many as there are row tiles
    AMCU_REQUIRE(ctas <= INT32_MAX, "amcu_attn_kv4: too many rows");
    d == 64 ? launch_prefill<64>(p, (unsigned)ctas, s) : launch_prefill<128>(p, (unsigned)ctas, s);
    return check_launch("amcu_attn_kv4");
}

}  // namespace amcu
