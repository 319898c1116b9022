// New rows into the 4-bit paged KV cache, and rows of it read back.
//
// Append, per row and head: q and k are scaled by w / sqrt(mean(x^2) + eps)
// where a weight is given, rotated (out[i] = a_i c - b_i s, out[i + d/2] =
// b_i c + a_i s; a, b the halves), q is rounded once to its type, k and v are
// quantised per 64 elements from fp32: m = fp16(min), s = fp16((max - min) *
// (1/15)), code = rint((x - m) / s). Products and sums of the rotation are rounded
// one by one (no fused multiply-add) and (x - m) / s is an IEEE division, so the
// codes are those of the written expressions.
#include "kv4.cuh"

namespace amcu {

am_status_code kv4_check(const char* what, const AmcuKv4Cache& c, const AmcuKv4Batch& b, Kv4View* out) {
    AMCU_REQUIRE(c.head_dim == 64 || c.head_dim == 128, "%s: head_dim must be 64 or 128", what);
    AMCU_REQUIRE(c.page_size >= 16 && c.page_size <= 256 && (c.page_size & (c.page_size - 1)) == 0,
                 "%s: page_size must be 16, 32, 64, 128 or 256", what);
    AMCU_REQUIRE(c.n_kv_heads > 0 && c.n_kv_heads <= 4096, "%s: n_kv_heads must be in [1, 4096]", what);
    AMCU_REQUIRE(c.num_pages > 0 && c.num_pages <= INT32_MAX, "%s: num_pages must be positive", what);
    AMCU_REQUIRE(b.rows >= 0 && b.rows <= (1 << 24) && b.n_seq >= 0 && b.n_seq <= (1 << 24),
                 "%s: rows and n_seq must be in [0, 2^24]", what);
    AMCU_REQUIRE(b.max_pages >= 0 && b.max_pages <= (1 << 30) / c.page_size,
                 "%s: max_pages must be in [0, 2^30 / page_size]", what);
    const int64_t codes = c.n_kv_heads * c.page_size * c.head_dim / 2, params = codes / 8;
    AMCU_REQUIRE(c.codes_page_stride == 0 || (c.codes_page_stride >= codes && c.codes_page_stride % 16 == 0),
                 "%s: codes_page_stride must be a multiple of 16 and hold a page", what);
    AMCU_REQUIRE(c.params_page_stride == 0 || (c.params_page_stride >= params && c.params_page_stride % 16 == 0),
                 "%s: params_page_stride must be a multiple of 16 and hold a page", what);
    AMCU_REQUIRE(codes <= UINT32_MAX && c.codes_page_stride <= UINT32_MAX && c.params_page_stride <= UINT32_MAX,
                 "%s: pages must be smaller than 4 GB", what);
    AMCU_REQUIRE(b.table_stride == 0 || b.table_stride >= b.max_pages || b.n_seq <= 1,
                 "%s: table_stride below max_pages", what);
    if (b.rows > 0 && b.n_seq > 0) {
        AMCU_REQUIRE(c.k_codes && c.k_params && c.v_codes && c.v_params && b.row_start && b.ctx_len &&
                             (b.page_table || b.max_pages == 0),
                     "%s: null pointer in cache or batch", what);
        AMCU_REQUIRE(aligned(c.k_codes, 16) && aligned(c.k_params, 16) && aligned(c.v_codes, 16) &&
                             aligned(c.v_params, 16),
                     "%s: cache planes must be 16-byte aligned", what);
    }
    out->kc = static_cast<uint8_t*>(c.k_codes);
    out->kp = static_cast<uint8_t*>(c.k_params);
    out->vc = static_cast<uint8_t*>(c.v_codes);
    out->vp = static_cast<uint8_t*>(c.v_params);
    out->cps = c.codes_page_stride ? c.codes_page_stride : codes;
    out->pps = c.params_page_stride ? c.params_page_stride : params;
    out->table = b.page_table;
    out->table_stride = b.table_stride ? b.table_stride : b.max_pages;
    out->row_start = b.row_start;
    out->ctx_len = b.ctx_len;
    out->status = b.status;
    out->num_pages = (int32_t)c.num_pages;
    out->max_pages = (int32_t)b.max_pages;
    out->n_seq = (int32_t)b.n_seq;
    out->rows = (int32_t)b.rows;
    out->page_shift = 0;
    while ((1 << out->page_shift) < c.page_size) ++out->page_shift;
    out->nkv = (int32_t)c.n_kv_heads;
    return AM_STATUS_OK;
}

struct Kv4AppendParams {
    Kv4View v;
    const void* q;
    const void* k;
    const void* val;
    void* q_out;
    int64_t qs, ks, vs, qos;
    const void* qw;
    const void* kw;
    float eps;
    const float2* cs;
    int64_t max_pos;
    int nq;
    bool vec;  // rows and weights start on four-element boundaries
};

// Four neighbouring elements, as loaded (Raw4) and as floats.
template <typename T> struct Four;
template <> struct Four<float> {
    float4 r;
    __device__ __forceinline__ void load(const float* p, bool vec) {
        if (vec) {
            r = *reinterpret_cast<const float4*>(p);
        } else {
            const float2 a = reinterpret_cast<const float2*>(p)[0], b = reinterpret_cast<const float2*>(p)[1];
            r = make_float4(a.x, a.y, b.x, b.y);
        }
    }
    __device__ __forceinline__ void get(float (&f)[4]) const { f[0] = r.x; f[1] = r.y; f[2] = r.z; f[3] = r.w; }
    static __device__ __forceinline__ void store(float* p, const float (&f)[4], bool vec) {
        if (vec) {
            *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
            reinterpret_cast<float2*>(p)[0] = make_float2(f[0], f[1]);
            reinterpret_cast<float2*>(p)[1] = make_float2(f[2], f[3]);
        }
    }
};
template <> struct Four<__nv_bfloat16> {
    uint2 r;
    __device__ __forceinline__ void load(const __nv_bfloat16* p, bool vec) {
        if (vec) {
            r = *reinterpret_cast<const uint2*>(p);
        } else {
            r.x = reinterpret_cast<const uint32_t*>(p)[0];
            r.y = reinterpret_cast<const uint32_t*>(p)[1];
        }
    }
    __device__ __forceinline__ void get(float (&f)[4]) const {
        f[0] = __uint_as_float(r.x << 16);
        f[1] = __uint_as_float(r.x & 0xffff0000u);
        f[2] = __uint_as_float(r.y << 16);
        f[3] = __uint_as_float(r.y & 0xffff0000u);
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[4], bool vec) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
        const uint2 w = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        if (vec) {
            *reinterpret_cast<uint2*>(p) = w;
        } else {
            reinterpret_cast<uint32_t*>(p)[0] = w.x;
            reinterpret_cast<uint32_t*>(p)[1] = w.y;
        }
    }
};

__device__ __forceinline__ uint32_t kv4_code(float x, float s, float m) {
    // NaN converts to 0
    return s > 0.f ? (uint32_t)min(max(__float2int_rn(fminf(fmaxf(__fdiv_rn(__fsub_rn(x, m), s), -1.f), 16.f)), 0), 15) : 0u;
}
// Four codes. (x - m) times 1 / s is within 15 * 2^-21 of the division, so its
// nearest whole number is the division's unless it lies that close to a half;
// only then the division is done (a third of the instructions otherwise).
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[4], float s, float m, float inv) {
    uint32_t r = 0;
    bool tie = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float y = fminf(fmaxf((x[i] - m) * inv, 0.f), 15.f);  // NaN becomes 0
        const float n = rintf(y);
        tie |= fabsf(y - n) > 0.49999f;
        r |= (uint32_t)(int)n << (4 * i);
    }
    if (tie) r = kv4_code(x[0], s, m) | (kv4_code(x[1], s, m) << 4) | (kv4_code(x[2], s, m) << 8) | (kv4_code(x[3], s, m) << 12);
    return r;
}

// Minimum and scale of a group. lo is NaN where every element is: such a group
// stays NaN (m = NaN, s = 0), so that it shows in every row that sees it.
__device__ __forceinline__ __half kv4_min(float lo) {
    return __float2half_rn(lo != lo ? lo : fminf(fmaxf(lo, -kHalfMax), kHalfMax));
}
__device__ __forceinline__ __half kv4_step(float lo, float hi) {
    return __float2half_rn(lo != lo ? 0.f : fminf(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f), kKv4StepMax));
}

// q_out of a row that has no position: zeros, a head after another (a call of its
// own: inlined it made the append of 9188 rows 1.3 us slower, so 0.3).
template <typename T, int D>
__device__ __noinline__ void kv4_append_nowhere(T* o, int heads, int step, bool vec, int32_t* status) {
    if (status) *status = (int32_t)AM_STATUS_OUT_OF_RANGE;
    const float none[4] = {};
    for (; heads > 0; heads -= step, o += step * D) {
        Four<T>::store(o, none, vec);
        Four<T>::store(o + D / 2, none, vec);
    }
}

// A warp takes U times 32 / LPH heads of one row (q heads, then k, then v). A
// lane holds elements 4l .. 4l + 3 of each half of its head: both members of
// four rotation pairs, and half a word of codes of each half.
//
// Bound by instruction issue for prompts (260 per warp and step of 8 elements a
// lane; DRAM at a third of its rate): the row's sequence, cos / sin and norm
// weights are fetched once for U steps, whose loads are all in flight together.
// 9188 rows of 32 + 16 heads of 64 with norms: 51 us with this layout, 37.6 with
// the division avoided and the sums of four elements shared out over the lanes (fp32:
// 49).
template <typename T, int D, int U>
__global__ void __launch_bounds__(128) kv4_append_kernel(Kv4AppendParams p) {
    constexpr int LPH = D / 8, HPW = 32 / LPH, half = D / 2;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, l = lane % LPH;
    const int heads = p.nq + 2 * p.v.nkv, wpr = (heads + HPW * U - 1) / (HPW * U);
    const uint32_t w = blockIdx.x * 4 + (threadIdx.x >> 5);  // below 2^31
    const int row = (int)(w / (uint32_t)wpr);
    if (row >= p.v.rows) return;
    const int head0 = (int)(w - (uint32_t)row * wpr) * (HPW * U) + lane / LPH;
    // the row's heads in their tensors, numbered through: q, then k, then v
    const T* q_row = static_cast<const T*>(p.q) + row * p.qs + 4 * l;
    const T* k_row = static_cast<const T*>(p.k) + row * p.ks + 4 * l - (int64_t)p.nq * D;
    const T* v_row = static_cast<const T*>(p.val) + row * p.vs + 4 * l - (int64_t)(p.nq + p.v.nkv) * D;
    Four<T> xr[U], yr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int head = head0 + u * HPW;
        if (head < heads) {
            const T* src = (head < p.nq ? q_row : head < p.nq + p.v.nkv ? k_row : v_row) + head * D;
            xr[u].load(src, p.vec);
            yr[u].load(src + half, p.vec);
        }
    }
    const int b = kv4_find_seq(p.v, row);
    const int pos = b >= 0 ? p.v.ctx_len[b] - p.v.row_start[b + 1] + row : -1;
    if (pos < 0 || pos >= p.max_pos) {  // no rotation, no place in the cache
        kv4_append_nowhere<T, D>(static_cast<T*>(p.q_out) + row * p.qos + (int64_t)head0 * D + 4 * l,
                                 min(p.nq - head0, U * HPW), HPW, p.vec, p.v.status);
        return;
    }
    const bool has_q = head0 - lane / LPH < p.nq, has_kv = head0 - lane / LPH + HPW * U > p.nq;
    const int page = has_kv ? kv4_page(p.v, b, pos) : -1;
    const int slot = pos & ((1 << p.v.page_shift) - 1);
    const float4 cs0 = reinterpret_cast<const float4*>(p.cs + (int64_t)pos * half + 4 * l)[0];  // c0 s0 c1 s1
    const float4 cs1 = reinterpret_cast<const float4*>(p.cs + (int64_t)pos * half + 4 * l)[1];
    const float c[4] = {cs0.x, cs0.z, cs1.x, cs1.z}, sn[4] = {cs0.y, cs0.w, cs1.y, cs1.w};
    Four<T> wq[2], wk[2];
    if (p.qw && has_q) {
        wq[0].load(static_cast<const T*>(p.qw) + 4 * l, p.vec);
        wq[1].load(static_cast<const T*>(p.qw) + half + 4 * l, p.vec);
    }
    if (p.kw && has_kv) {
        wk[0].load(static_cast<const T*>(p.kw) + 4 * l, p.vec);
        wk[1].load(static_cast<const T*>(p.kw) + half + 4 * l, p.vec);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int head = head0 + u * HPW;
        if (head - lane / LPH >= heads) break;  // the whole warp
        const bool live = head < heads, is_q = head < p.nq, is_k = !is_q && head < p.nq + p.v.nkv;
        const int kvh = head - p.nq - (is_k ? 0 : p.v.nkv);
        float x[4] = {}, y[4] = {};
        if (live) {
            xr[u].get(x);
            yr[u].get(y);
        }
        if (p.qw || p.kw) {
            // Sum of squares in a fixed order, each addition rounded by itself: halves
            // onto each other down to one element (d = 64), or to runs of four
            // neighbours that are added first (d = 128).
            float ss;
            if (D == 128) {
                float a = __fmul_rn(x[0], x[0]), e = __fmul_rn(y[0], y[0]);
#pragma unroll
                for (int i = 1; i < 4; ++i) {
                    a = __fadd_rn(a, __fmul_rn(x[i], x[i]));
                    e = __fadd_rn(e, __fmul_rn(y[i], y[i]));
                }
                ss = __fadd_rn(a, e);
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, o));
            } else {
                float q[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) q[i] = __fadd_rn(__fmul_rn(x[i], x[i]), __fmul_rn(y[i], y[i]));
                // lanes 4, 2 and 1 apart share out the four sums: upper lanes go on with 2, 3, then 1, 3
                const bool up4 = l & 4, up2 = l & 2;
                float a = up4 ? q[2] : q[0], e = up4 ? q[3] : q[1];
                a = __fadd_rn(a, __shfl_xor_sync(0xffffffffu, up4 ? q[0] : q[2], 4));
                e = __fadd_rn(e, __shfl_xor_sync(0xffffffffu, up4 ? q[1] : q[3], 4));
                const float other = __shfl_xor_sync(0xffffffffu, up2 ? a : e, 2);
                a = __fadd_rn(up2 ? e : a, other);
                a = __fadd_rn(a, __shfl_xor_sync(0xffffffffu, a, 1));
                a = __fadd_rn(a, __shfl_xor_sync(0xffffffffu, a, 4));  // 0 + 2, 1 + 3
                ss = __fadd_rn(a, __shfl_xor_sync(0xffffffffu, a, 2));
            }
            if ((is_q && p.qw) || (is_k && p.kw)) {
                const float r = rsqrtf(__fadd_rn(ss * (1.f / D), p.eps));
                Four<T> wr[2] = {is_q ? wq[0] : wk[0], is_q ? wq[1] : wk[1]};
                float wa[4], wb[4];
                wr[0].get(wa);
                wr[1].get(wb);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = x[i] * r * wa[i];
                    y[i] = y[i] * r * wb[i];
                }
            }
        }
        if (is_q || is_k) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = x[i], e = y[i];
                x[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(e, sn[i]));
                y[i] = __fadd_rn(__fmul_rn(e, c[i]), __fmul_rn(a, sn[i]));
            }
        }
        if (is_q) {
            T* o = static_cast<T*>(p.q_out) + row * p.qos + (int64_t)head * D;
            Four<T>::store(o + 4 * l, x, p.vec);
            Four<T>::store(o + half + 4 * l, y, p.vec);
        }
        if (head - lane / LPH + HPW <= p.nq) continue;  // q heads only: nothing to quantise
        // groups: D = 128: x is in group 0 and y in group 1; D = 64: both in the one group
        float lo0 = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), hi0 = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        float lo1 = fminf(fminf(y[0], y[1]), fminf(y[2], y[3])), hi1 = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
        if (D == 64) {
            lo0 = fminf(lo0, lo1);
            hi0 = fmaxf(hi0, hi1);
        }
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) {
            lo0 = fminf(lo0, __shfl_xor_sync(0xffffffffu, lo0, o));
            hi0 = fmaxf(hi0, __shfl_xor_sync(0xffffffffu, hi0, o));
            if (D == 128) {
                lo1 = fminf(lo1, __shfl_xor_sync(0xffffffffu, lo1, o));
                hi1 = fmaxf(hi1, __shfl_xor_sync(0xffffffffu, hi1, o));
            }
        }
        if (D == 64) {
            lo1 = lo0;
            hi1 = hi0;
        }
        const __half m0 = kv4_min(lo0), m1 = kv4_min(lo1), s0 = kv4_step(lo0, hi0), s1 = kv4_step(lo1, hi1);
        const float f0 = __half2float(s0), f1 = __half2float(s1);
        const float i0 = f0 > 0.f ? __fdividef(1.f, f0) : 0.f, i1 = D == 64 ? i0 : f1 > 0.f ? __fdividef(1.f, f1) : 0.f;
        const uint32_t h0 = kv4_codes(x, f0, __half2float(m0), i0), h1 = kv4_codes(y, f1, __half2float(m1), i1);
        // even lanes complete the first half's word, odd lanes the second's
        const uint32_t got = __shfl_xor_sync(0xffffffffu, l & 1 ? h0 : h1, 1);
        const uint32_t word = l & 1 ? got | (h1 << 16) : h0 | (got << 16);
        if (is_q || !live || page < 0) continue;
        uint8_t* codes = (is_k ? p.v.kc : p.v.vc) + kv4_code_off<D>(p.v, page, kvh, slot);
        uint8_t* params = (is_k ? p.v.kp : p.v.vp) + kv4_param_off<D>(p.v, page, kvh, slot);
        // D = 128: words alternate between the groups (halves); D = 64: the second half follows the first
        *reinterpret_cast<uint32_t*>(codes + 4 * (D == 128 ? l : (l >> 1) + (l & 1) * 4)) = word;
        if (l == 0) *reinterpret_cast<__half2*>(params) = __halves2half2(s0, m0);
        if (D == 128 && l == 1) *reinterpret_cast<__half2*>(params + 4) = __halves2half2(s1, m1);
    }
}

struct Kv4GatherParams {
    Kv4View v;
    void* ko;
    void* vo;
    int64_t kos, vos;
};

__device__ __forceinline__ void kv4_put8(float* o, const float (&f)[8]) {
    reinterpret_cast<float4*>(o)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(o)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void kv4_put8(__nv_bfloat16* o, const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
}

// One thread per 16 bytes of codes (32 elements) of a row's k and v heads.
// 9188 rows of 8 heads of 64: 9.2 us to bf16 (24.1 MB read and written, 2.6 TB/s), 16.0 to
// fp32 (42.9 MB).
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_gather_kernel(Kv4GatherParams p) {
    constexpr int CPR = D / 32, G = D / kKv4Group;  // 16-byte chunks per head row, groups
    pdl_wait();
    pdl_trigger();
    const int wpr = (2 * p.v.nkv * CPR + 31) / 32;  // warps per row
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (w >= (int64_t)p.v.rows * wpr) return;
    const int row = (int)(w / wpr);
    const int item = (int)(w % wpr) * 32 + (threadIdx.x & 31);
    const int b = kv4_find_seq(p.v, row);
    int page = -1, slot = 0;
    if (b >= 0) {
        const int pos = p.v.ctx_len[b] - p.v.row_start[b + 1] + row;
        page = kv4_page(p.v, b, pos);
        slot = pos & ((1 << p.v.page_shift) - 1);
    } else if (p.v.status) {
        *p.v.status = (int32_t)AM_STATUS_OUT_OF_RANGE;
    }
    if (item >= 2 * p.v.nkv * CPR) return;
    const int chunk = item % CPR, kvh = (item / CPR) % p.v.nkv, is_v = item / (CPR * p.v.nkv);
    uint4 c = make_uint4(0, 0, 0, 0);
    float2 sm[G];
#pragma unroll
    for (int g = 0; g < G; ++g) sm[g] = make_float2(0.f, 0.f);
    if (page >= 0) {
        c = *reinterpret_cast<const uint4*>((is_v ? p.v.vc : p.v.kc) + kv4_code_off<D>(p.v, page, kvh, slot) + 16 * chunk);
        const __half2* par = reinterpret_cast<const __half2*>((is_v ? p.v.vp : p.v.kp) + kv4_param_off<D>(p.v, page, kvh, slot));
#pragma unroll
        for (int g = 0; g < G; ++g) sm[g] = __half22float2(par[g]);
    }
    T* o = static_cast<T*>(is_v ? p.vo : p.ko) + row * (is_v ? p.vos : p.kos) + (int64_t)kvh * D;
    const uint32_t words[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int word = 4 * chunk + i, g = i % G;  // four words start on a group boundary
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __fadd_rn(__fmul_rn((float)((words[i] >> (4 * e)) & 15u), sm[g].x), sm[g].y);
        kv4_put8(o + g * kKv4Group + (word / G) * 8, f);
    }
}

}  // namespace amcu

using namespace amcu;

extern "C" am_status_code amcu_kv4_append(const AmcuKv4AppendArgs* a, void* stream) {
    clear_error();
    AMCU_REQUIRE(a != nullptr, "amcu_kv4_append: null args");
    Kv4AppendParams p;
    am_status_code st = kv4_check("amcu_kv4_append", a->cache, a->batch, &p.v);
    if (st != AM_STATUS_OK) return st;
    AMCU_REQUIRE(a->dtype == AMCU_F32 || a->dtype == AMCU_BF16, "amcu_kv4_append: dtype must be f32 or bf16");
    AMCU_REQUIRE(a->n_q_heads > 0 && a->n_q_heads <= 65536, "amcu_kv4_append: n_q_heads must be in [1, 65536]");
    AMCU_REQUIRE(a->max_pos > 0, "amcu_kv4_append: max_pos must be positive");
    AMCU_REQUIRE(a->eps >= 0.f, "amcu_kv4_append: eps must not be negative");
    if (a->batch.rows == 0 || a->batch.n_seq == 0) return AM_STATUS_OK;
    AMCU_REQUIRE(a->q && a->k && a->v && a->q_out && a->cos_sin, "amcu_kv4_append: null pointer");
    const int64_t es = a->dtype == AMCU_F32 ? 8 : 4;  // bytes of a two-element vector
    AMCU_REQUIRE(aligned(a->q, es) && aligned(a->k, es) && aligned(a->v, es) && aligned(a->q_out, es) &&
                         (!a->q_norm || aligned(a->q_norm, es)) && (!a->k_norm || aligned(a->k_norm, es)) &&
                         a->q_stride % 2 == 0 && a->k_stride % 2 == 0 && a->v_stride % 2 == 0 &&
                         a->q_out_stride % 2 == 0,
                 "amcu_kv4_append: rows must start on two-element boundaries");
    AMCU_REQUIRE(aligned(a->cos_sin, 16), "amcu_kv4_append: cos_sin must be 16-byte aligned");
    p.q = a->q;
    p.k = a->k;
    p.val = a->v;
    p.q_out = a->q_out;
    p.qs = a->q_stride;
    p.ks = a->k_stride;
    p.vs = a->v_stride;
    p.qos = a->q_out_stride;
    p.qw = a->q_norm;
    p.kw = a->k_norm;
    p.eps = a->eps;
    p.cs = reinterpret_cast<const float2*>(a->cos_sin);
    p.max_pos = a->max_pos;
    p.nq = (int)a->n_q_heads;
    p.vec = aligned(a->q, 2 * es) && aligned(a->k, 2 * es) && aligned(a->v, 2 * es) && aligned(a->q_out, 2 * es) &&
            (!a->q_norm || aligned(a->q_norm, 2 * es)) && (!a->k_norm || aligned(a->k_norm, 2 * es)) &&
            a->q_stride % 4 == 0 && a->k_stride % 4 == 0 && a->v_stride % 4 == 0 && a->q_out_stride % 4 == 0;
    const int64_t steps = ceil_div(a->n_q_heads + 2 * a->cache.n_kv_heads, 256 / a->cache.head_dim);  // a warp's heads
    // Four steps to a warp once single steps would fill every SM's 64 warps twice.
    const bool many = a->batch.rows * steps > 128 * (int64_t)num_sms();
    const int64_t blocks = ceil_div(a->batch.rows * ceil_div(steps, many ? 4 : 1), 4);
    AMCU_REQUIRE(blocks <= INT32_MAX / 4, "amcu_kv4_append: too many rows");
    const dim3 grid((unsigned)blocks), block(128);
    cudaStream_t s = as_stream(stream);
    auto go = [&](auto one, auto four) { launch_pdl(many ? four : one, grid, block, 0, s, p); };
    const bool f32 = a->dtype == AMCU_F32;
    if (a->cache.head_dim == 64)
        f32 ? go(kv4_append_kernel<float, 64, 1>, kv4_append_kernel<float, 64, 4>)
            : go(kv4_append_kernel<__nv_bfloat16, 64, 1>, kv4_append_kernel<__nv_bfloat16, 64, 4>);
    else
        f32 ? go(kv4_append_kernel<float, 128, 1>, kv4_append_kernel<float, 128, 4>)
            : go(kv4_append_kernel<__nv_bfloat16, 128, 1>, kv4_append_kernel<__nv_bfloat16, 128, 4>);
    return check_launch("amcu_kv4_append");
}

extern "C" am_status_code amcu_kv4_gather(const AmcuKv4GatherArgs* a, void* stream) {
    clear_error();
    AMCU_REQUIRE(a != nullptr, "amcu_kv4_gather: null args");
    Kv4GatherParams p;
    am_status_code st = kv4_check("amcu_kv4_gather", a->cache, a->batch, &p.v);
    if (st != AM_STATUS_OK) return st;
    AMCU_REQUIRE(a->dtype == AMCU_F32 || a->dtype == AMCU_BF16, "amcu_kv4_gather: dtype must be f32 or bf16");
    if (a->batch.rows == 0 || a->batch.n_seq == 0) return AM_STATUS_OK;
    AMCU_REQUIRE(a->k_out && a->v_out, "amcu_kv4_gather: null pointer");
    AMCU_REQUIRE(aligned(a->k_out, 16) && aligned(a->v_out, 16) && a->k_out_stride % 8 == 0 && a->v_out_stride % 8 == 0,
                 "amcu_kv4_gather: output rows must start on 16-byte boundaries");
    p.ko = a->k_out;
    p.vo = a->v_out;
    p.kos = a->k_out_stride;
    p.vos = a->v_out_stride;
    const int64_t wpr = ceil_div(2 * a->cache.n_kv_heads * a->cache.head_dim / 32, 32);
    const int64_t blocks = ceil_div(a->batch.rows * wpr, 4);
    AMCU_REQUIRE(blocks <= INT32_MAX, "amcu_kv4_gather: too many rows");
    const dim3 grid((unsigned)blocks), block(128);
    const bool f32 = a->dtype == AMCU_F32;
    if (a->cache.head_dim == 64)
        f32 ? launch_pdl(kv4_gather_kernel<float, 64>, grid, block, 0, as_stream(stream), p)
            : launch_pdl(kv4_gather_kernel<__nv_bfloat16, 64>, grid, block, 0, as_stream(stream), p);
    else
        f32 ? launch_pdl(kv4_gather_kernel<float, 128>, grid, block, 0, as_stream(stream), p)
            : launch_pdl(kv4_gather_kernel<__nv_bfloat16, 128>, grid, block, 0, as_stream(stream), p);
    return check_launch("amcu_kv4_gather");
}
