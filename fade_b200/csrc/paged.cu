// Page planning of a serving step and rotary positions with several axes,
// fused with the append of K and V to a paged cache.
#include <algorithm>

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

// Every block scans the lengths into its shared memory (first token and first
// new page of every request), then takes its share of the tokens and new
// pages, bisecting for their requests; block 0 writes what there is once.  No
// block reads what another writes: slots in new pages come from the free list,
// not from the table.  Latency bound (a launch, two trips to L2, a scan): 64
// decodes 4.2 us, 2048 prompts of 131 k tokens 8.9 us (one block: 140 us).
__global__ void __launch_bounds__(1024) plan_step_kernel(const PlanParams p) {
    extern __shared__ int32_t starts[];          // [R] first token, [R] first new page
    __shared__ Sum2 warp_sums[32];
    const fade_plan_desc& d = p.d;
    const int R = (int)d.R, per = (R + blockDim.x - 1) / blockDim.x;
    int32_t* tok0 = starts;
    int32_t* new0 = starts + R;
    const int r0 = min(R, (int)threadIdx.x * per), r1 = min(R, r0 + per);
    const int n_free = d.n_free[0];
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
    const bool neg = __syncthreads_or(bad & 1) || n_free < 0 || n_free > d.free_cap;
    const bool full = __syncthreads_or(bad & 2);
    const int status = neg ? FADE_PLAN_LENGTHS
                       : tot.a > d.total ? FADE_PLAN_TOKENS
                       : full ? FADE_PLAN_ROW_FULL
                       : tot.b > n_free ? FADE_PLAN_NO_PAGES
                                        : FADE_PLAN_OK;
    const bool ok = status == FADE_PLAN_OK, first = blockIdx.x == 0;
    Sum2 at{incl.a - mine.a, incl.b - mine.b};
    for (int r = r0; r < r1; ++r) {
        const int n = d.new_lens[r], c = d.kv_lens[r];
        if (ok) {
            tok0[r] = (int)at.a;
            new0[r] = (int)at.b;
            at.a += n;
            at.b += pages_of((int64_t)c + n, p.page_log2) - pages_of(c, p.page_log2);
        }
        if (first) {
            d.cu_q[r + 1] = ok ? (int)at.a : 0;
            d.kv_out[r] = ok ? c + n : c;
        }
    }
    if (first && threadIdx.x == 0) {
        d.cu_q[0] = 0;
        d.n_free_out[0] = ok ? n_free - (int)tot.b : n_free;
        d.status[0] = status;
    }
    __syncthreads();
    const int live = ok ? (int)tot.a : 0, stride = gridDim.x * blockDim.x;
    for (int64_t t = blockIdx.x * blockDim.x + threadIdx.x; t < d.total; t += stride) {
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
    for (int k = blockIdx.x * blockDim.x + threadIdx.x; k < fresh; k += stride) {
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
// precedes the barrier after which they change.  Latency bound, and run when
// requests finish, not every step.
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
    const int axes = (int)d.axes;
    if (axes == 1) return 0;
    if (d.interleaved) {
        const int a = j % axes;
        return a != 0 && j < axes * (int)d.sections[a] ? a : 0;
    }
    int a = 0;
    for (int end = (int)d.sections[0]; a + 1 < axes && j >= end; end += (int)d.sections[a]) ++a;
    return a;
}

// two fp32 values per register pair, two products or sums per instruction
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 one_by_one(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t mul_two(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// (a, b) -> (a c - b s, b c + a s): the second product rounded, the first one
// and the sum in one operation
template <int DT, int VEC>
__device__ __forceinline__ void rotate_unit(typename Elem<DT>::T* a, typename Elem<DT>::T* b, const float* co, const float* si) {
    if constexpr (VEC == 1) {
        const float u0 = Elem<DT>::to_f(a[0]), u1 = Elem<DT>::to_f(b[0]);
        a[0] = Elem<DT>::from_f(__fmaf_rn(u0, co[0], __fmul_rn(u1, -si[0])));
        b[0] = Elem<DT>::from_f(__fmaf_rn(u1, co[0], __fmul_rn(u0, si[0])));
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const uint64_t u0 = two(Elem<DT>::to_f(a[j]), Elem<DT>::to_f(a[j + 1]));
            const uint64_t u1 = two(Elem<DT>::to_f(b[j]), Elem<DT>::to_f(b[j + 1]));
            const uint64_t c = two(co[j], co[j + 1]);
            const float2 y0 = one_by_one(fma_two(u0, c, mul_two(u1, two(-si[j], -si[j + 1]))));
            const float2 y1 = one_by_one(fma_two(u1, c, mul_two(u0, two(si[j], si[j + 1]))));
            a[j] = Elem<DT>::from_f(y0.x), a[j + 1] = Elem<DT>::from_f(y0.y);
            b[j] = Elem<DT>::from_f(y1.x), b[j + 1] = Elem<DT>::from_f(y1.y);
        }
    }
}

template <int BYTES> struct Packet;
template <> struct Packet<16> { using T = uint4; };
template <> struct Packet<8> { using T = uint2; };
template <> struct Packet<4> { using T = uint32_t; };
template <> struct Packet<2> { using T = uint16_t; };

// Place of frequency j in a token's table of rot/2 cosines, then rot/2 sines:
// packets of four of a unit apart by all units, so that neighbouring threads
// (neighbouring units) read neighbouring 16 bytes without bank conflicts.
template <int VEC>
__device__ __forceinline__ int table_at(int j, int turns) {
    return VEC < 4 ? j : (((j % VEC) / 4) * turns + j / VEC) * 4 + j % 4;
}

// A unit is VEC channels and their partners, or VEC copied channels, of up to
// kRopeHeads heads of q, k or v of a token: its cos and sin are read and its
// addresses made once for all of them, and their loads are in flight together.
// A block makes the cos and sin of `tokens` tokens, then its threads share out
// their units; the blocks of an SM hide one another's first phase.
// HBM bound: a token's rows are read and written once.  16384 tokens of 32 + 2
// x 8 heads of 128 bf16 channels, appended: 74 us, 5.5 TB/s of 403 MB.  With
// one head a unit 83 us (more address arithmetic), with four 76 us; three
// blocks per SM 78 us, five 79 us (spills); with loads under the making of the
// next tokens' tables 87 us and more (its registers cost blocks).
constexpr int kRopeHeads = 2;
constexpr int kRopeBlocks = 4;   // blocks per SM

template <int DT, int VEC>
__global__ void __launch_bounds__(256, kRopeBlocks)
    rope_axes_kernel(const __grid_constant__ fade_rope_desc d, int page_log2, int tokens) {
    using T = typename Elem<DT>::T;
    using P = typename Packet<VEC * sizeof(T)>::T;
    extern __shared__ __align__(16) float cs[];  // [tokens][rot]
    const int half = (int)d.rot / 2;
    const int64_t t0 = (int64_t)blockIdx.x * tokens;
    const int n_tok = (int)min((int64_t)tokens, d.T - t0);
    const int turns = half / VEC, per = turns + ((int)d.D - (int)d.rot) / VEC, per_v = (int)d.D / VEC;
    for (int a = threadIdx.x; a < n_tok * half; a += blockDim.x) {
        const int k = a / half, j = a - k * half;
        const int64_t at = rope_axis(d, j) * d.pos_stride + t0 + k;
        const float pos = d.positions_64 ? (float)static_cast<const int64_t*>(d.positions)[at]
                                         : (float)static_cast<const int32_t*>(d.positions)[at];
        float s, co;
        sincosf(__fmul_rn(pos, d.inv_freq[j]), &s, &co);
        if (d.round_tables) s = Elem<DT>::rnd(s), co = Elem<DT>::rnd(co);
        float* row = cs + k * 2 * half + table_at<VEC>(j, turns);
        row[0] = co;
        row[half] = d.inverse ? -s : s;
    }
    __syncthreads();
    const int bq = ((int)d.Hq + kRopeHeads - 1) / kRopeHeads, bk = ((int)d.Hkv + kRopeHeads - 1) / kRopeHeads;
    const int nq = bq * per, nk = bk * per, units = nq + nk + bk * per_v;
    for (int w = threadIdx.x; w < n_tok * units; w += blockDim.x) {
        const int k = w / units, u = w - k * units;
        const int64_t t = t0 + k;
        const int what = u < nq ? 0 : u < nq + nk ? 1 : 2;
        const int i = what == 0 ? u : what == 1 ? u - nq : u - nq - nk, n = what == 2 ? per_v : per;
        const int hb = i / n, x = i - hb * n, h0 = hb * kRopeHeads;
        const bool turn = what != 2 && x < turns;
        const int c = turn || what == 2 ? x * VEC : (int)d.rot + (x - turns) * VEC;   // first channel
        const int heads = min(kRopeHeads, (int)(what == 0 ? d.Hq : d.Hkv) - h0);
        P lo[kRopeHeads], hi[kRopeHeads];
        {
            const int64_t sh = what == 0 ? d.q_sh : what == 1 ? d.k_sh : d.v_sh;
            const T* src = (what == 0   ? static_cast<const T*>(d.q) + t * d.q_st
                            : what == 1 ? static_cast<const T*>(d.k) + t * d.k_st
                                        : static_cast<const T*>(d.v) + t * d.v_st) + h0 * sh + c;
#pragma unroll
            for (int g = 0; g < kRopeHeads; ++g) {
                if (g >= heads) continue;
                lo[g] = *reinterpret_cast<const P*>(src + g * sh);
                if (turn) hi[g] = *reinterpret_cast<const P*>(src + g * sh + half);
            }
        }
        int64_t sh = d.qo_sh;
        T* dst = static_cast<T*>(d.q_out) + t * d.qo_st;
        if (what != 0) {
            const int64_t slot = d.slots[t];
            if (slot < 0 || slot >= d.n_pages << page_log2) continue;   // padding
            const int64_t page = slot >> page_log2, off = slot & (d.page_size - 1);
            sh = what == 1 ? d.kp_sh : d.vp_sh;
            dst = what == 1 ? static_cast<T*>(d.k_pool) + page * d.kp_sp + off * d.kp_st
                            : static_cast<T*>(d.v_pool) + page * d.vp_sp + off * d.vp_st;
        }
        dst += h0 * sh + c;
        if (turn) {
            const float* row = cs + k * 2 * half;
            float co[VEC], si[VEC];
            if constexpr (VEC >= 4) {
#pragma unroll
                for (int j = 0; j < VEC; j += 4) {
                    *reinterpret_cast<float4*>(co + j) = *reinterpret_cast<const float4*>(row + table_at<VEC>(c + j, turns));
                    *reinterpret_cast<float4*>(si + j) =
                        *reinterpret_cast<const float4*>(row + half + table_at<VEC>(c + j, turns));
                }
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) co[j] = row[c + j], si[j] = row[half + c + j];
            }
#pragma unroll
            for (int g = 0; g < kRopeHeads; ++g)
                if (g < heads) rotate_unit<DT, VEC>(reinterpret_cast<T*>(&lo[g]), reinterpret_cast<T*>(&hi[g]), co, si);
        }
#pragma unroll
        for (int g = 0; g < kRopeHeads; ++g) {
            if (g >= heads) continue;
            *reinterpret_cast<P*>(dst + g * sh) = lo[g];
            if (turn) *reinterpret_cast<P*>(dst + g * sh + half) = hi[g];
        }
    }
}

template <int DT, int VEC>
static void launch_rope(const fade_rope_desc& d, int page_log2, cudaStream_t st) {
    // up to 8 tokens a block while every block slot of the GPU still has one
    const int64_t tokens = std::max<int64_t>(1, std::min<int64_t>(8, d.T / (148 * kRopeBlocks)));
    const int64_t per = d.rot / 2 / VEC + (d.D - d.rot) / VEC;
    const int64_t bq = (d.Hq + kRopeHeads - 1) / kRopeHeads, bk = (d.Hkv + kRopeHeads - 1) / kRopeHeads;
    const int64_t units = tokens * ((bq + bk) * per + bk * (d.D / VEC));
    const unsigned threads = units >= 256 ? 256 : (unsigned)((units + 31) / 32 * 32);
    rope_axes_kernel<DT, VEC><<<(unsigned)((d.T + tokens - 1) / tokens), threads, (size_t)(tokens * d.rot * 4), st>>>(
        d, page_log2, (int)tokens);
}

// The widest packet (16 bytes at most) that divides the rotated half, the
// copied channels and the head, and to which every pointer and stride in use
// is aligned.
template <int DT, int VEC>
static void launch_rope_widest(const fade_rope_desc& d, int page_log2, cudaStream_t st) {
    using T = typename Elem<DT>::T;
    if constexpr (VEC > 1) {
        bool ok = (d.rot / 2) % VEC == 0 && d.D % VEC == 0 && (d.D - d.rot) % VEC == 0;
        auto ptr = [&](const void* p) { ok = ok && reinterpret_cast<uintptr_t>(p) % (VEC * sizeof(T)) == 0; };
        auto stride = [&](int64_t s, int64_t n) { ok = ok && (n <= 1 || s % VEC == 0); };
        if (d.Hq > 0) {
            ptr(d.q), ptr(d.q_out);
            stride(d.q_st, d.T), stride(d.q_sh, d.Hq), stride(d.qo_st, d.T), stride(d.qo_sh, d.Hq);
        }
        if (d.Hkv > 0) {
            ptr(d.k), ptr(d.v), ptr(d.k_pool), ptr(d.v_pool);
            stride(d.k_st, d.T), stride(d.k_sh, d.Hkv), stride(d.v_st, d.T), stride(d.v_sh, d.Hkv);
            stride(d.kp_sp, d.n_pages), stride(d.kp_sh, d.Hkv), stride(d.kp_st, d.page_size);
            stride(d.vp_sp, d.n_pages), stride(d.vp_sh, d.Hkv), stride(d.vp_st, d.page_size);
        }
        if (!ok) return launch_rope_widest<DT, VEC / 2>(d, page_log2, st);
    }
    launch_rope<DT, VEC>(d, page_log2, st);
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
    if (smem > 40 * 1024)
        FADE_CUDA_TRY(cudaFuncSetAttribute(plan_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           FADE_PLAN_MAX_ROWS * 8));
    // threads for the longer of the scan and the tokens, a token each, up to one block per SM
    const int64_t work = d->R > d->total ? d->R : d->total;
    const int threads = work <= 256 ? 256 : 1024;
    const int64_t blocks = (d->total + threads - 1) / threads;
    plan_step_kernel<<<(unsigned)(blocks < 1 ? 1 : blocks > 148 ? 148 : blocks), threads, smem, as_stream(stream)>>>(p);
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
    if (R * 4 > 40 * 1024)
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
    if (d->D > 1024 || d->Hq > 4096 || d->Hkv > 4096 || d->T > INT32_MAX) return FADE_ERR_UNSUPPORTED;
    if (d->T == 0 || (d->Hq == 0 && d->Hkv == 0)) return FADE_OK;
    if ((d->rot > 0 && (!d->positions || !d->inv_freq)) || (d->Hq > 0 && (!d->q || !d->q_out)))
        return FADE_ERR_INVALID_ARG;
    // in place, or apart: a block reads what another one may have written otherwise
    const bool in_place = d->q == d->q_out && (d->T == 1 || d->q_st == d->qo_st) && (d->Hq == 1 || d->q_sh == d->qo_sh);
    if (!in_place && views_overlap(d->q, d->q_st, d->q_sh, d->q_out, d->qo_st, d->qo_sh, d->T, d->Hq, d->D,
                                   d->dtype == FADE_F32 ? 4 : 2))
        return FADE_ERR_INVALID_ARG;
    int pl = 0;
    if (d->Hkv > 0) {
        pl = log2_of(d->page_size);
        if (pl < 0 || pl > 20 || d->n_pages < 0) return FADE_ERR_INVALID_ARG;
        if (!d->k || !d->v || !d->slots || (d->n_pages > 0 && (!d->k_pool || !d->v_pool))) return FADE_ERR_INVALID_ARG;
    }
    cudaStream_t st = as_stream(stream);
    if (d->dtype == FADE_F16) launch_rope_widest<FADE_F16, 8>(*d, pl, st);
    else if (d->dtype == FADE_BF16) launch_rope_widest<FADE_BF16, 8>(*d, pl, st);
    else launch_rope_widest<FADE_F32, 4>(*d, pl, st);
    FADE_LAUNCH_CHECK();
    return FADE_OK;
}
