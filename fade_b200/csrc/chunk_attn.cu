// Attention of a step's new tokens over a paged FP16/BF16 cache.
//
// With s_j = sm_scale * q.k_j over the keys a query sees,
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  lse = m + log sum_j exp(s_j - m)
// in one pass over the keys, with the running maximum m.
#include <cmath>

#include "common.cuh"

namespace fade {

// One warp per (token, query head), channels over the lanes, keys one by one.
template <int DT, int D>
__global__ void __launch_bounds__(128) chunk_attn_kernel(const fade_chunk_desc d) {
    using T = typename Elem<DT>::T;
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t w = blockIdx.x * 4LL + (threadIdx.x >> 5);
    if (w >= d.T * d.Hq) return;
    const int64_t t = w / d.Hq, h = w % d.Hq, hk = h / (d.Hq / d.Hkv);
    int r = -1;
    for (int i = 0; i < d.R; ++i)
        if (d.cu_q[i] <= t && t < d.cu_q[i + 1]) r = i;
    if (r < 0) return;
    const int64_t kv = min((int64_t)d.kv_lens[r], d.table_width * d.page_size);
    const int64_t p = kv - d.cu_q[r + 1] + t;
    const int64_t j1 = d.causal ? min(kv, p + 1) : kv, j0 = d.window > 0 ? max((int64_t)0, p - d.window + 1) : 0;
    float q[E], acc[E], m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; ++e) {
        q[e] = Elem<DT>::to_f(static_cast<const T*>(d.q)[t * d.q_st + h * d.q_sh + lane * E + e]);
        acc[e] = 0.f;
    }
    for (int64_t j = j0; j < j1; ++j) {
        const int64_t page = d.block_table[r * d.table_stride + j / d.page_size], off = j % d.page_size;
        if (page < 0 || page >= d.n_pages) continue;
        const T* k = static_cast<const T*>(d.k_pool) + page * d.kp_sp + hk * d.kp_sh + off * d.kp_st + lane * E;
        const T* v = static_cast<const T*>(d.v_pool) + page * d.vp_sp + hk * d.vp_sh + off * d.vp_st + lane * E;
        float s = 0.f;
        for (int e = 0; e < E; ++e) s += q[e] * Elem<DT>::to_f(k[e]);
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        s *= (float)d.sm_scale;
        const float mn = fmaxf(m, s);
        const float a = m == mn ? 1.f : expf(m - mn), b = expf(s - mn);
        m = mn;
        l = l * a + b;
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * a + b * Elem<DT>::to_f(v[e]);
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    for (int e = 0; e < E; ++e)
        static_cast<T*>(d.out)[t * d.o_st + h * d.o_sh + lane * E + e] = Elem<DT>::from_f(acc[e] * inv);
    if (d.lse && lane == 0) d.lse[w] = m + logf(l);
}

static int check_desc(const fade_chunk_desc* d) {
    if (!d || d->R < 0 || d->T < 0 || d->Hq < 1 || d->Hkv < 1 || d->Hq % d->Hkv || d->table_width < 0 ||
        d->n_pages < 0 || d->window < 0 || !(d->sm_scale > 0.0) || std::isinf(d->sm_scale))
        return FADE_ERR_INVALID_ARG;
    if (d->dtype != FADE_F16 && d->dtype != FADE_BF16) return FADE_ERR_UNSUPPORTED;
    if ((d->D != 64 && d->D != 128) || d->Hq / d->Hkv > 128) return FADE_ERR_UNSUPPORTED;
    if (d->page_size != 16 && d->page_size != 32 && d->page_size != 64 && d->page_size != 128)
        return FADE_ERR_UNSUPPORTED;
    if (d->R > INT32_MAX / 2 || d->T > INT32_MAX / d->Hq || d->n_pages > INT32_MAX ||
        d->table_width > INT32_MAX / d->page_size)
        return FADE_ERR_UNSUPPORTED;
    return FADE_OK;
}

}  // namespace fade

using namespace fade;

extern "C" size_t fade_chunk_attn_workspace_size(const fade_chunk_desc* d) {
    return check_desc(d) == FADE_OK ? 256 : 0;
}

extern "C" int fade_chunk_attn(const fade_chunk_desc* d, void* workspace, size_t ws_bytes, void* stream) {
    const int bad = check_desc(d);
    if (bad != FADE_OK) return bad;
    if (d->T == 0 || d->R == 0) return FADE_OK;
    if (!d->q || !d->out || !d->cu_q || !d->kv_lens || (d->table_width > 0 && !d->block_table) ||
        (d->n_pages > 0 && (!d->k_pool || !d->v_pool)))
        return FADE_ERR_INVALID_ARG;
    const int64_t strides[] = {d->q_st, d->q_sh, d->o_st, d->o_sh, d->kp_sp, d->kp_sh, d->kp_st, d->vp_sp, d->vp_sh, d->vp_st};
    for (int64_t s : strides)
        if (s % 8) return FADE_ERR_ALIGN;
    if (!aligned16(d->q) || !aligned16(d->out) || !aligned16(d->k_pool) || !aligned16(d->v_pool)) return FADE_ERR_ALIGN;
    if (!workspace || ws_bytes < fade_chunk_attn_workspace_size(d)) return FADE_ERR_WORKSPACE;
    const unsigned grid = (unsigned)((d->T * d->Hq + 3) / 4);
    cudaStream_t st = as_stream(stream);
    if (d->dtype == FADE_F16) {
        if (d->D == 64) chunk_attn_kernel<FADE_F16, 64><<<grid, 128, 0, st>>>(*d);
        else chunk_attn_kernel<FADE_F16, 128><<<grid, 128, 0, st>>>(*d);
    } else {
        if (d->D == 64) chunk_attn_kernel<FADE_BF16, 64><<<grid, 128, 0, st>>>(*d);
        else chunk_attn_kernel<FADE_BF16, 128><<<grid, 128, 0, st>>>(*d);
    }
    FADE_LAUNCH_CHECK();
    return FADE_OK;
}
