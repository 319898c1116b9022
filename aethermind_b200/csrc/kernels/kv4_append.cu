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
};

template <typename T> __device__ __forceinline__ float2 kv4_ld2(const T* p);
template <> __device__ __forceinline__ float2 kv4_ld2<float>(const float* p) { return *reinterpret_cast<const float2*>(p); }
template <> __device__ __forceinline__ float2 kv4_ld2<__nv_bfloat16>(const __nv_bfloat16* p) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
}
__device__ __forceinline__ void kv4_st2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void kv4_st2(__nv_bfloat16* p, float a, float b) {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
}

// Reduction over the LPH lanes that hold one head.
template <int LPH>
__device__ __forceinline__ float head_min(float v) {
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <int LPH>
__device__ __forceinline__ float head_max(float v) {
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ int kv4_code(float x, float s, float m) {
    // NaN converts to 0
    return s > 0.f ? min(max(__float2int_rn(fminf(fmaxf(__fdiv_rn(__fsub_rn(x, m), s), -1.f), 16.f)), 0), 15) : 0;
}

// One warp per row and 32 / LPH heads (q heads, then k, then v). A lane holds
// elements 2l, 2l + 1 of each half of its head: both members of two rotation
// pairs, and one code byte of each half.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_append_kernel(Kv4AppendParams p) {
    constexpr int LPH = D / 4, HPW = 32 / LPH, half = D / 2;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, l = lane % LPH;
    const int heads = p.nq + 2 * p.v.nkv, wpr = (heads + HPW - 1) / HPW;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (w >= (int64_t)p.v.rows * wpr) return;
    const int row = (int)(w / wpr);
    const int head = (int)(w % wpr) * HPW + lane / LPH;
    const int b = kv4_find_seq(p.v, row);
    if (b < 0) return;
    const int pos = p.v.ctx_len[b] - p.v.row_start[b + 1] + row;
    if (pos < 0 || pos >= p.max_pos) {
        if (p.v.status) *p.v.status = (int32_t)AM_STATUS_OUT_OF_RANGE;
        return;
    }
    const bool is_q = head < p.nq, is_k = !is_q && head < p.nq + p.v.nkv, live = head < heads;
    const int kvh = is_q ? 0 : (head - p.nq) % p.v.nkv;
    const T* src = is_q ? static_cast<const T*>(p.q) + row * p.qs + (int64_t)head * D
                 : is_k ? static_cast<const T*>(p.k) + row * p.ks + (int64_t)kvh * D
                        : static_cast<const T*>(p.val) + row * p.vs + (int64_t)kvh * D;
    float2 x = make_float2(0.f, 0.f), y = x;
    if (live) {
        x = kv4_ld2<T>(src + 2 * l);
        y = kv4_ld2<T>(src + half + 2 * l);
    }
    const T* nw = static_cast<const T*>(is_q ? p.qw : is_k ? p.kw : nullptr);
    // Sum of squares in a fixed order, each addition rounded by itself: halves
    // onto each other down to one element (d = 64), or to runs of four
    // neighbours that are added first (d = 128).
    float2 q0 = make_float2(__fmul_rn(x.x, x.x), __fmul_rn(x.y, x.y)), q1 = make_float2(__fmul_rn(y.x, y.x), __fmul_rn(y.y, y.y));
    float ss;
    if (D == 128) {
        const float2 o0 = make_float2(__shfl_xor_sync(0xffffffffu, q0.x, 1), __shfl_xor_sync(0xffffffffu, q0.y, 1));
        const float2 o1 = make_float2(__shfl_xor_sync(0xffffffffu, q1.x, 1), __shfl_xor_sync(0xffffffffu, q1.y, 1));
        const bool odd = l & 1;
        const float a = __fadd_rn(__fadd_rn(odd ? __fadd_rn(o0.x, o0.y) : __fadd_rn(q0.x, q0.y), odd ? q0.x : o0.x), odd ? q0.y : o0.y);
        const float c = __fadd_rn(__fadd_rn(odd ? __fadd_rn(o1.x, o1.y) : __fadd_rn(q1.x, q1.y), odd ? q1.x : o1.x), odd ? q1.y : o1.y);
        ss = __fadd_rn(a, c);
#pragma unroll
        for (int o = 16; o > 1; o >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, o));
    } else {
        q0 = make_float2(__fadd_rn(q0.x, q1.x), __fadd_rn(q0.y, q1.y));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
            q0 = make_float2(__fadd_rn(q0.x, __shfl_xor_sync(0xffffffffu, q0.x, o)),
                             __fadd_rn(q0.y, __shfl_xor_sync(0xffffffffu, q0.y, o)));
        ss = __fadd_rn(q0.x, q0.y);
    }
    if (nw) {
        const float r = rsqrtf(__fadd_rn(ss / (float)D, p.eps));
        const float2 wa = kv4_ld2<T>(nw + 2 * l), wb = kv4_ld2<T>(nw + half + 2 * l);
        x = make_float2(x.x * r * wa.x, x.y * r * wa.y);
        y = make_float2(y.x * r * wb.x, y.y * r * wb.y);
    }
    if (is_q || is_k) {
        const float4 cs = *reinterpret_cast<const float4*>(p.cs + (int64_t)pos * half + 2 * l);  // c0 s0 c1 s1
        const float2 a = x, c = y;
        x.x = __fsub_rn(__fmul_rn(a.x, cs.x), __fmul_rn(c.x, cs.y));
        y.x = __fadd_rn(__fmul_rn(c.x, cs.x), __fmul_rn(a.x, cs.y));
        x.y = __fsub_rn(__fmul_rn(a.y, cs.z), __fmul_rn(c.y, cs.w));
        y.y = __fadd_rn(__fmul_rn(c.y, cs.z), __fmul_rn(a.y, cs.w));
    }
    if (is_q) {
        T* o = static_cast<T*>(p.q_out) + row * p.qos + (int64_t)head * D;
        kv4_st2(o + 2 * l, x.x, x.y);
        kv4_st2(o + half + 2 * l, y.x, y.y);
    }
    // groups: D = 128: x is in group 0 and y in group 1; D = 64: both in the one group
    float lo0 = fminf(x.x, x.y), hi0 = fmaxf(x.x, x.y), lo1 = fminf(y.x, y.y), hi1 = fmaxf(y.x, y.y);
    if (D == 64) {
        lo0 = lo1 = fminf(lo0, lo1);
        hi0 = hi1 = fmaxf(hi0, hi1);
    }
    lo0 = head_min<LPH>(lo0);
    hi0 = head_max<LPH>(hi0);
    if (D == 128) {
        lo1 = head_min<LPH>(lo1);
        hi1 = head_max<LPH>(hi1);
    } else {
        lo1 = lo0;
        hi1 = hi0;
    }
    if (is_q || !live) return;
    const int page = kv4_page(p.v, b, pos);
    if (page < 0) return;
    const int slot = pos & ((1 << p.v.page_shift) - 1);
    uint8_t* codes = (is_k ? p.v.kc : p.v.vc) + kv4_code_off<D>(p.v, page, kvh, slot);
    uint8_t* params = (is_k ? p.v.kp : p.v.vp) + kv4_param_off<D>(p.v, page, kvh, slot);
    const __half m0 = __float2half_rn(fminf(fmaxf(lo0, -kHalfMax), kHalfMax));
    const __half m1 = __float2half_rn(fminf(fmaxf(lo1, -kHalfMax), kHalfMax));
    const __half s0 = __float2half_rn(fminf(__fmul_rn(__fsub_rn(hi0, lo0), 1.f / 15.f), kKv4StepMax));
    const __half s1 = __float2half_rn(fminf(__fmul_rn(__fsub_rn(hi1, lo1), 1.f / 15.f), kKv4StepMax));
    const float fm0 = __half2float(m0), fm1 = __half2float(m1), fs0 = __half2float(s0), fs1 = __half2float(s1);
    const uint8_t b0 = (uint8_t)(kv4_code(x.x, fs0, fm0) | (kv4_code(x.y, fs0, fm0) << 4));
    const uint8_t b1 = (uint8_t)(kv4_code(y.x, fs1, fm1) | (kv4_code(y.y, fs1, fm1) << 4));
    if (D == 128) {  // words alternate between the groups
        codes[(l >> 2) * 8 + (l & 3)] = b0;
        codes[(l >> 2) * 8 + 4 + (l & 3)] = b1;
    } else {
        codes[l] = b0;
        codes[LPH + l] = b1;
    }
    if (l == 0) *reinterpret_cast<__half2*>(params) = __halves2half2(s0, m0);
    if (D == 128 && l == 1) *reinterpret_cast<__half2*>(params + 4) = __halves2half2(s1, m1);
}

struct Kv4GatherParams {
    Kv4View v;
    void* ko;
    void* vo;
    int64_t kos, vos;
};

// One thread per 32-bit word of codes (8 elements) of a row's k and v heads.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_gather_kernel(Kv4GatherParams p) {
    constexpr int WPR = D / 8, G = D / kKv4Group;  // words per head row, groups
    pdl_wait();
    pdl_trigger();
    const int wpr = (2 * p.v.nkv * WPR + 31) / 32;  // warps per row
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
    }
    if (item >= 2 * p.v.nkv * WPR) return;
    const int word = item % WPR, kvh = (item / WPR) % p.v.nkv, is_v = item / (WPR * p.v.nkv);
    const int grp = word % G, e0 = grp * kKv4Group + (word / G) * 8;
    float f[8] = {};
    if (page >= 0) {
        const uint32_t c = *reinterpret_cast<const uint32_t*>((is_v ? p.v.vc : p.v.kc) +
                                                              kv4_code_off<D>(p.v, page, kvh, slot) + 4 * word);
        const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(
                (is_v ? p.v.vp : p.v.kp) + kv4_param_off<D>(p.v, page, kvh, slot) + 4 * grp));
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __fadd_rn(__fmul_rn((float)((c >> (4 * i)) & 15u), sm.x), sm.y);
    }
    T* o = static_cast<T*>(is_v ? p.vo : p.ko) + row * (is_v ? p.vos : p.kos) + (int64_t)kvh * D + e0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) kv4_st2(o + i, f[i], f[i + 1]);
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
    const int64_t heads = a->n_q_heads + 2 * a->cache.n_kv_heads;
    const int64_t hpw = a->cache.head_dim == 64 ? 2 : 1;
    const int64_t blocks = ceil_div(a->batch.rows * ceil_div(heads, hpw), 4);
    AMCU_REQUIRE(blocks <= INT32_MAX, "amcu_kv4_append: too many rows");
    const dim3 grid((unsigned)blocks), block(128);
    const bool f32 = a->dtype == AMCU_F32;
    if (a->cache.head_dim == 64)
        f32 ? launch_pdl(kv4_append_kernel<float, 64>, grid, block, 0, as_stream(stream), p)
            : launch_pdl(kv4_append_kernel<__nv_bfloat16, 64>, grid, block, 0, as_stream(stream), p);
    else
        f32 ? launch_pdl(kv4_append_kernel<float, 128>, grid, block, 0, as_stream(stream), p)
            : launch_pdl(kv4_append_kernel<__nv_bfloat16, 128>, grid, block, 0, as_stream(stream), p);
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
    const int64_t wpr = ceil_div(2 * a->cache.n_kv_heads * a->cache.head_dim / 8, 32);
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
