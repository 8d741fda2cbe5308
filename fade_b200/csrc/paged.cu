// Page planning of a serving step and rotary positions with several axes,
// fused with the append of K and V to a paged cache.
#include "common.cuh"

namespace fade {

// ---------------------------------------------------------------------------
// Page planning
// ---------------------------------------------------------------------------
struct PlanParams {
    fade_plan_desc d;
    int page_log2;
};

// Inclusive sums of two counts over the block; `tot` receives the block's
// totals.  64-bit: lengths come from device memory and may be anything.
struct Sum2 {
    int64_t a, b;
};
__device__ __forceinline__ Sum2 block_scan(Sum2 v, Sum2* warp_sums, Sum2* tot) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (blockDim.x + 31) >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t a = __shfl_up_sync(~0u, v.a, o), b = __shfl_up_sync(~0u, v.b, o);
        if (lane >= o) v.a += a, v.b += b;
    }
    __syncthreads();   // warp_sums free again
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    Sum2 before{0, 0}, all{0, 0};
    for (int w = 0; w < nw; ++w) {
        if (w == warp) before = all;
        all.a += warp_sums[w].a;
        all.b += warp_sums[w].b;
    }
    *tot = all;
    return {v.a + before.a, v.b + before.b};
}

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int page_log2) {
    return (tokens + (1 << page_log2) - 1) >> page_log2;
}

// last r in [0, n) with start[r] <= x, for ascending starts (start[0] <= x)
__device__ __forceinline__ int row_of(const int32_t* start, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One block: lengths are scanned into shared memory (first token and first new
// page of every request), then tokens and new pages are dealt out to threads,
// which find their request by bisection.
__global__ void __launch_bounds__(1024) plan_step_kernel(const PlanParams p) {
    extern __shared__ int32_t starts[];          // [R] first token, [R] first new page
    __shared__ Sum2 warp_sums[32];
    const fade_plan_desc& d = p.d;
    const int R = (int)d.R, per = (R + blockDim.x - 1) / blockDim.x;
    int32_t* tok0 = starts;
    int32_t* new0 = starts + R;
    const int r0 = min(R, (int)threadIdx.x * per), r1 = min(R, r0 + per);
    Sum2 mine{0, 0};
    int bad = 0;
    for (int r = r0; r < r1; ++r) {
        const int64_t n = d.new_lens[r], c = d.kv_lens[r];
        if (n < 0 || c < 0) bad |= 1;
        if (pages_of(c + n, p.page_log2) > d.table_width || c + n > INT32_MAX) bad |= 2;
        mine.a += n;
        mine.b += pages_of(c + n, p.page_log2) - pages_of(c, p.page_log2);
    }
    Sum2 tot;
    const Sum2 incl = block_scan(mine, warp_sums, &tot);
    const int n_free = d.n_free[0];
    const bool neg = __syncthreads_or(bad & 1) || n_free < 0 || n_free > d.free_cap;
    const bool full = __syncthreads_or(bad & 2);
    const int status = neg ? FADE_PLAN_LENGTHS
                       : tot.a > d.total ? FADE_PLAN_TOKENS
                       : full ? FADE_PLAN_ROW_FULL
                       : tot.b > n_free ? FADE_PLAN_NO_PAGES
                                        : FADE_PLAN_OK;
    const bool ok = status == FADE_PLAN_OK;
    Sum2 at{incl.a - mine.a, incl.b - mine.b};
    for (int r = r0; r < r1; ++r) {
        const int n = d.new_lens[r], c = d.kv_lens[r];
        if (ok) {
            tok0[r] = (int)at.a;
            new0[r] = (int)at.b;
            at.a += n;
            at.b += pages_of((int64_t)c + n, p.page_log2) - pages_of(c, p.page_log2);
        }
        d.cu_q[r + 1] = ok ? (int)at.a : 0;
        d.kv_out[r] = ok ? c + n : c;
    }
    if (threadIdx.x == 0) {
        d.cu_q[0] = 0;
        d.n_free_out[0] = ok ? n_free - (int)tot.b : n_free;
        d.status[0] = status;
    }
    __syncthreads();
    const int live = ok ? (int)tot.a : 0;
    for (int64_t t = threadIdx.x; t < d.total; t += blockDim.x) {
        int pos = 0;
        int64_t slot = -1;
        if (t < live) {
            const int r = row_of(tok0, R, (int)t), c = d.kv_lens[r];
            pos = c + (int)t - tok0[r];
            const int j = pos >> p.page_log2, have = (int)pages_of(c, p.page_log2);
            const int page = j < have ? d.block_table[r * d.table_stride + j] : d.free_pages[n_free - 1 - new0[r] - (j - have)];
            slot = ((int64_t)page << p.page_log2) + (pos & ((1 << p.page_log2) - 1));
        }
        d.positions[t] = pos;
        d.slots[t] = slot;
    }
    const int fresh = ok ? (int)tot.b : 0;
    for (int k = threadIdx.x; k < fresh; k += blockDim.x) {
        const int r = row_of(new0, R, k);
        const int64_t j = pages_of(d.kv_lens[r], p.page_log2) + k - new0[r];
        d.block_table[r * d.table_stride + j] = d.free_pages[n_free - 1 - k];
    }
}

struct ReleaseParams {
    const uint8_t* rows;
    int32_t* kv_lens;
    const int32_t* block_table;
    int32_t* free_pages;
    int32_t* n_free;
    int32_t* status;
    int64_t table_width, table_stride, free_cap;
    int R, page_log2;
};

// One block, in place: every read of the lengths and of the stack's height
// precedes the barrier after which they change.
__global__ void __launch_bounds__(1024) release_rows_kernel(const ReleaseParams p) {
    extern __shared__ int32_t new0[];            // [R] first page a row gives back
    __shared__ Sum2 warp_sums[32];
    const int R = p.R, per = (R + blockDim.x - 1) / blockDim.x;
    const int r0 = min(R, (int)threadIdx.x * per), r1 = min(R, r0 + per);
    Sum2 mine{0, 0};
    int bad = 0;
    for (int r = r0; r < r1; ++r) {
        const int64_t n = p.rows[r] ? pages_of(p.kv_lens[r], p.page_log2) : 0;
        if (p.kv_lens[r] < 0) bad |= 1;
        if (n > p.table_width) bad |= 2;
        mine.a += n;
    }
    Sum2 tot;
    const Sum2 incl = block_scan(mine, warp_sums, &tot);
    const int n_free = p.n_free[0];
    const bool neg = __syncthreads_or(bad & 1) || n_free < 0;
    const bool full = __syncthreads_or(bad & 2);
    const int status = neg ? FADE_PLAN_LENGTHS
                       : full ? FADE_PLAN_ROW_FULL
                       : n_free + tot.a > p.free_cap ? FADE_PLAN_NO_PAGES
                                                     : FADE_PLAN_OK;
    if (threadIdx.x == 0) p.status[0] = status;
    if (status != FADE_PLAN_OK) return;
    int64_t at = incl.a - mine.a;
    for (int r = r0; r < r1; ++r) {
        new0[r] = (int)at;
        if (p.rows[r]) {
            at += pages_of(p.kv_lens[r], p.page_log2);
            p.kv_lens[r] = 0;
        }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < (int)tot.a; k += blockDim.x) {
        const int r = row_of(new0, R, k);
        p.free_pages[n_free + k] = p.block_table[r * p.table_stride + k - new0[r]];
    }
    if (threadIdx.x == 0) p.n_free[0] = n_free + (int)tot.a;
}

// ---------------------------------------------------------------------------
// Rotary positions with several axes (+ append)
// ---------------------------------------------------------------------------
__device__ __forceinline__ int rope_axis(const fade_rope_desc& d, int j) {
    if (d.interleaved) {
        const int a = j % (int)d.axes;
        return a != 0 && j < d.axes * d.sections[a] ? a : 0;
    }
    int a = 0;
    for (int64_t end = d.sections[0]; a + 1 < d.axes && j >= end; end += d.sections[a]) ++a;
    return a;
}

// One block per token: cos and sin of its rot/2 angles in shared memory, then
// one thread per channel pair or copied channel.
template <int DT>
__global__ void __launch_bounds__(256) rope_axes_kernel(const fade_rope_desc d, int page_log2) {
    using T = typename Elem<DT>::T;
    extern __shared__ float2 cs[];
    const int64_t t = blockIdx.x;
    const int half = (int)d.rot / 2, D = (int)d.D;
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
        const int64_t at = rope_axis(d, j) * d.pos_stride + t;
        const float pos = d.positions_64 ? (float)static_cast<const int64_t*>(d.positions)[at]
                                         : (float)static_cast<const int32_t*>(d.positions)[at];
        float s, c;
        sincosf(__fmul_rn(pos, d.inv_freq[j]), &s, &c);
        if (d.round_tables) s = Elem<DT>::rnd(s), c = Elem<DT>::rnd(c);
        cs[j] = make_float2(c, d.inverse ? -s : s);
    }
    __syncthreads();
    int64_t page = -1, off = 0;
    if (d.Hkv > 0) {
        const int64_t slot = d.slots[t];
        if (slot >= 0 && slot < d.n_pages << page_log2) page = slot >> page_log2, off = slot & (d.page_size - 1);
    }
    const int per = half + D - (int)d.rot;       // pairs, then copied channels
    auto turn = [&](const T* x, T* y, int u) {
        if (u < half) {
            const float a = Elem<DT>::to_f(x[u]), b = Elem<DT>::to_f(x[u + half]);
            const float c = cs[u].x, s = cs[u].y;
            y[u] = Elem<DT>::from_f(__fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)));
            y[u + half] = Elem<DT>::from_f(__fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s)));
        } else {
            y[u + half] = x[u + half];
        }
    };
    for (int i = threadIdx.x; i < d.Hq * per; i += blockDim.x) {
        const int64_t h = i / per;
        turn(static_cast<const T*>(d.q) + t * d.q_st + h * d.q_sh, static_cast<T*>(d.q_out) + t * d.qo_st + h * d.qo_sh,
             i % per);
    }
    if (page < 0) return;
    for (int i = threadIdx.x; i < d.Hkv * per; i += blockDim.x) {
        const int64_t h = i / per;
        turn(static_cast<const T*>(d.k) + t * d.k_st + h * d.k_sh,
             static_cast<T*>(d.k_pool) + page * d.kp_sp + h * d.kp_sh + off * d.kp_st, i % per);
    }
    for (int i = threadIdx.x; i < d.Hkv * D; i += blockDim.x) {
        const int64_t h = i / D;
        static_cast<T*>(d.v_pool)[page * d.vp_sp + h * d.vp_sh + off * d.vp_st + i % D] =
            static_cast<const T*>(d.v)[t * d.v_st + h * d.v_sh + i % D];
    }
}

static int log2_of(int64_t x) {
    int l = 0;
    while ((1LL << l) < x) ++l;
    return x > 0 && (1LL << l) == x ? l : -1;
}

}  // namespace fade

using namespace fade;

extern "C" int fade_plan_step(const fade_plan_desc* d, void* stream) {
    if (!d || d->R < 0 || d->total < 0 || d->table_width < 0 || d->free_cap < 0) return FADE_ERR_INVALID_ARG;
    if (!d->cu_q || !d->n_free || !d->n_free_out || !d->status) return FADE_ERR_INVALID_ARG;
    if (d->R > 0 && (!d->new_lens || !d->kv_lens || !d->kv_out || (!d->block_table && d->table_width > 0)))
        return FADE_ERR_INVALID_ARG;
    if (d->total > 0 && (!d->positions || !d->slots)) return FADE_ERR_INVALID_ARG;
    if (d->free_cap > 0 && !d->free_pages) return FADE_ERR_INVALID_ARG;
    if ((d->R > 0 && d->kv_out == d->kv_lens) || d->n_free_out == d->n_free) return FADE_ERR_INVALID_ARG;
    const int pl = log2_of(d->page_size);
    if (pl < 0 || pl > 20) return FADE_ERR_INVALID_ARG;
    if (d->R > FADE_PLAN_MAX_ROWS || d->total > INT32_MAX) return FADE_ERR_UNSUPPORTED;
    PlanParams p{*d, pl};
    const size_t smem = (size_t)d->R * 8;
    FADE_CUDA_TRY(cudaFuncSetAttribute(plan_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       FADE_PLAN_MAX_ROWS * 8));
    plan_step_kernel<<<1, 1024, smem, as_stream(stream)>>>(p);
    FADE_LAUNCH_CHECK();
    return FADE_OK;
}

extern "C" int fade_release_rows(const uint8_t* rows, int64_t R, int32_t* kv_lens, const int32_t* block_table,
                                 int64_t table_width, int64_t table_stride, int64_t page_size, int32_t* free_pages,
                                 int64_t free_cap, int32_t* n_free, int32_t* status, void* stream) {
    if (R < 0 || table_width < 0 || free_cap < 0 || !n_free || !status) return FADE_ERR_INVALID_ARG;
    if (R > 0 && (!rows || !kv_lens || (!block_table && table_width > 0))) return FADE_ERR_INVALID_ARG;
    if (free_cap > 0 && !free_pages) return FADE_ERR_INVALID_ARG;
    const int pl = log2_of(page_size);
    if (pl < 0 || pl > 20) return FADE_ERR_INVALID_ARG;
    if (R > FADE_PLAN_MAX_ROWS) return FADE_ERR_UNSUPPORTED;
    ReleaseParams p{rows, kv_lens, block_table, free_pages, n_free, status, table_width, table_stride, free_cap, (int)R, pl};
    FADE_CUDA_TRY(cudaFuncSetAttribute(release_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       FADE_PLAN_MAX_ROWS * 4));
    release_rows_kernel<<<1, 1024, (size_t)R * 4, as_stream(stream)>>>(p);
    FADE_LAUNCH_CHECK();
    return FADE_OK;
}

extern "C" int fade_rope_axes(const fade_rope_desc* d, void* stream) {
    if (!d || d->T < 0 || d->Hq < 0 || d->Hkv < 0 || d->D <= 0 || d->rot < 0) return FADE_ERR_INVALID_ARG;
    if (d->rot % 2) return FADE_ERR_ODD_DIM;
    if (d->rot > d->D || d->axes < 1 || d->axes > FADE_MAX_AXES) return FADE_ERR_INVALID_ARG;
    if (d->dtype != FADE_F16 && d->dtype != FADE_BF16 && d->dtype != FADE_F32) return FADE_ERR_INVALID_ARG;
    int64_t sum = 0;
    for (int a = 0; a < d->axes; ++a) {
        if (d->sections[a] < 0) return FADE_ERR_INVALID_ARG;
        sum += d->sections[a];
    }
    if (sum != d->rot / 2) return FADE_ERR_INVALID_ARG;
    if (d->D > 4096 || d->Hq > 4096 || d->Hkv > 4096 || d->T > INT32_MAX) return FADE_ERR_UNSUPPORTED;
    if (d->T == 0 || (d->Hq == 0 && d->Hkv == 0)) return FADE_OK;
    if ((d->rot > 0 && (!d->positions || !d->inv_freq)) || (d->Hq > 0 && (!d->q || !d->q_out)))
        return FADE_ERR_INVALID_ARG;
    int pl = 0;
    if (d->Hkv > 0) {
        pl = log2_of(d->page_size);
        if (pl < 0 || pl > 20 || d->n_pages < 0) return FADE_ERR_INVALID_ARG;
        if (!d->k || !d->v || !d->slots || (d->n_pages > 0 && (!d->k_pool || !d->v_pool))) return FADE_ERR_INVALID_ARG;
    }
    const size_t smem = (size_t)(d->rot / 2) * sizeof(float2);
    cudaStream_t st = as_stream(stream);
    if (d->dtype == FADE_F16) rope_axes_kernel<FADE_F16><<<(unsigned)d->T, 256, smem, st>>>(*d, pl);
    else if (d->dtype == FADE_BF16) rope_axes_kernel<FADE_BF16><<<(unsigned)d->T, 256, smem, st>>>(*d, pl);
    else rope_axes_kernel<FADE_F32><<<(unsigned)d->T, 256, smem, st>>>(*d, pl);
    FADE_LAUNCH_CHECK();
    return FADE_OK;
}
