// Causal GQA attention over the 4-bit paged KV cache.
//
// out[row, h] = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q . k_j - max), over
// the positions j <= pos of the row's sequence; k_j = m + s * code.
#include "kv4.cuh"

namespace amcu {

struct Kv4AttnParams {
    Kv4View v;
    const void* q;
    void* out;
    int64_t qs, os;
    int nq, grp;
    float scale;
};

// One warp per (row, q head): 32 keys at a time, one per lane, then the
// output's elements are shared out over the lanes.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_attn_simple_kernel(Kv4AttnParams p) {
    constexpr int G = D / kKv4Group, EPL = D / 32;
    __shared__ float qs[4][D];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, wi = threadIdx.x >> 5;
    const int64_t w = (int64_t)blockIdx.x * 4 + wi;
    if (w >= (int64_t)p.v.rows * p.nq) return;
    const int row = (int)(w / p.nq), h = (int)(w % p.nq), kvh = h / p.grp;
    const int b = kv4_find_seq(p.v, row);
    if (b < 0) return;
    const int pos = p.v.ctx_len[b] - p.v.row_start[b + 1] + row;
    const T* q = static_cast<const T*>(p.q) + row * p.qs + (int64_t)h * D;
    for (int e = lane; e < D; e += 32) qs[wi][e] = Act<T>::load(q[e]) * p.scale;
    __syncwarp();
    float mx = -INFINITY, sum = 0.f, acc[EPL] = {};
    for (int k0 = 0; k0 <= pos; k0 += 32) {
        const int key = k0 + lane;
        int page = -1;
        int64_t co = 0, po = 0;
        float s = -INFINITY;
        if (key <= pos) page = kv4_page(p.v, b, key);
        if (page >= 0) {
            const int slot = key & ((1 << p.v.page_shift) - 1);
            co = kv4_code_off<D>(p.v, page, kvh, slot);
            po = kv4_param_off<D>(p.v, page, kvh, slot);
            s = 0.f;
            for (int word = 0; word < D / 8; ++word) {
                const uint32_t c = *reinterpret_cast<const uint32_t*>(p.v.kc + co + 4 * word);
                const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(p.v.kp + po + 4 * (word % G)));
                const float* qe = &qs[wi][(word % G) * kKv4Group + (word / G) * 8];
                for (int i = 0; i < 8; ++i) s += qe[i] * ((float)((c >> (4 * i)) & 15u) * sm.x + sm.y);
            }
        }
        const float nm = fmaxf(mx, warp_max(s));
        const float corr = nm == -INFINITY ? 1.f : expf(mx - nm);
        const float pr = page >= 0 ? expf(s - nm) : 0.f;
        sum = sum * corr + warp_sum(pr);
        mx = nm;
        for (int i = 0; i < EPL; ++i) acc[i] *= corr;
        for (int j = 0; j < 32; ++j) {
            const float pj = __shfl_sync(0xffffffffu, pr, j);
            const int64_t cj = __shfl_sync(0xffffffffu, co, j), pj_off = __shfl_sync(0xffffffffu, po, j);
            if (!__shfl_sync(0xffffffffu, (int)(page >= 0), j)) continue;
            for (int i = 0; i < EPL; ++i) {
                const int e = i * 32 + lane, g = e / kKv4Group, r = e % kKv4Group;
                const uint8_t c = p.v.vc[cj + 4 * ((r / 8) * G + g) + (r % 8) / 2];
                const float2 sm = __half22float2(*reinterpret_cast<const __half2*>(p.v.vp + pj_off + 4 * g));
                acc[i] += pj * ((float)((c >> (4 * (r & 1))) & 15) * sm.x + sm.y);
            }
        }
    }
    T* o = static_cast<T*>(p.out) + row * p.os + (int64_t)h * D;
    for (int i = 0; i < EPL; ++i) o[i * 32 + lane] = Act<T>::store(sum > 0.f ? acc[i] / sum : 0.f);
}

}  // namespace amcu

using namespace amcu;

extern "C" size_t amcu_attn_kv4_workspace_bytes(const AmcuKv4AttentionArgs* a) {
    (void)a;
    return 0;
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
    if (a->batch.rows == 0 || a->batch.n_seq == 0) return AM_STATUS_OK;
    AMCU_REQUIRE(a->q && a->out, "amcu_attn_kv4: null pointer");
    p.q = a->q;
    p.out = a->out;
    p.qs = a->q_stride;
    p.os = a->out_stride;
    p.nq = (int)a->n_q_heads;
    p.grp = (int)(a->n_q_heads / a->cache.n_kv_heads);
    p.scale = a->scale > 0.f ? a->scale : 1.f / sqrtf((float)a->cache.head_dim);
    const int64_t blocks = ceil_div(a->batch.rows * a->n_q_heads, 4);
    AMCU_REQUIRE(blocks <= INT32_MAX, "amcu_attn_kv4: too many rows");
    const dim3 grid((unsigned)blocks), block(128);
    const bool f32 = a->dtype == AMCU_F32;
    if (a->cache.head_dim == 64)
        f32 ? launch_pdl(kv4_attn_simple_kernel<float, 64>, grid, block, 0, as_stream(stream), p)
            : launch_pdl(kv4_attn_simple_kernel<__nv_bfloat16, 64>, grid, block, 0, as_stream(stream), p);
    else
        f32 ? launch_pdl(kv4_attn_simple_kernel<float, 128>, grid, block, 0, as_stream(stream), p)
            : launch_pdl(kv4_attn_simple_kernel<__nv_bfloat16, 128>, grid, block, 0, as_stream(stream), p);
    return check_launch("amcu_attn_kv4");
}
