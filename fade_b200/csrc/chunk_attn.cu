// Attention of a step's new tokens over a paged FP16/BF16 cache.
//
// With s_j = sm_scale * q.k_j over the keys a query sees,
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  lse = m + log sum_j exp(s_j - m)
// in one pass over the keys: scores S = Q K^T and the sum O += P V run on the
// tensor cores with S, P and O in tensor memory, the running maximum m and the
// sum of the weights stay in fp32 registers.  P is rounded to the model dtype
// for its product (as K and V are stored); everything else is fp32 until the
// one rounding of the result.
//
// Rows.  The query heads of a kv head share its keys, so a row is (token, head
// of the group): row = token * g + head.  A half tile is 128 rows (the M of one
// MMA): tq = 128 / g tokens; a tile is two half tiles.  Each of two softmax
// warpgroups owns one *stream*: a score tile (128 rows x 128 keys), a weight
// tile over it and an output tile in tensor memory, one row per thread.
//   - more than tq tokens: stream s is half tile s, both walk all key blocks
//     and share every loaded K and V block;
//   - up to tq tokens (decodes, drafts, the end of a chunk): both streams hold
//     the same rows and take alternate key blocks; the two outputs are joined
//     at the end.
// While one stream's softmax runs, the tensor cores work on the other's.
//
// Work split.  Every (request, kv head, tile) costs its visible keys plus a
// constant; the sum is cut into equal parts, one per SM, wherever that falls
// in a tile's keys (to the block of 128).  A CTA walks its contiguous range of
// tiles; a tile that crosses a cut leaves partial outputs in the workspace,
// joined in order by a second kernel.  So ragged batches, the causal triangle
// and few long rows all fill the GPU alike, from lengths that only the device
// knows.
//
// Warps of a CTA: 0-3 and 4-7 softmax, 8 loads (TMA, one box per page), 9 and
// 11 MMA, 10 walks the tiles and posts the segments.
//
// What bounds it, bf16, 32 query and 8 kv heads of 128 channels:
//   - 4 chunks of 2048 tokens over 8192: 849-888 us, 1.16-1.21 PFLOP/s; tensor
//     pipe 63 % and exponential unit 63 % of the cycles, at a clock that power
//     pulls from 1.93 to 1.57 GHz.  A block of two half tiles takes about
//     3300 cycles against 2048 of its MMAs and 2048 of its exponentials: the
//     streams' turns at the exponential unit (1400 each) and the chain scores
//     - maximum - weights - weights x V are of one length.  Without turns
//     1026 us against 838; a quarter or half of the exponentials on the FMA pipe
//     instead (twelve instructions a pair) 930-1094 and 995-1199 us against
//     912-936.
//   - 16 decodes of up to 8192 tokens: 73.5 us, 5.4 TB/s: HBM while it streams
//     (5 TMA stages of 32 KB), the rest is start (5 us), join (4 us), uneven ends.
//   - 4 chunks of 1021 tokens, window 1024 (fp16): 100 us, 0.69 PFLOP/s: ten
//     blocks a tile, 2.5 us of output a tile, 10 us of joining.
//
// V of masked keys.  A weight of zero times a NaN or an infinity is NaN in the
// tensor core, so a V that only some rows of a tile see would reach them all.
// The output of a tile is checked as it is written; rows that are not finite
// are looked at again behind the join, and those with such a V among the keys
// their mask hides are computed anew, a warp a row, from the keys they see.
// Keys past the end of a cache are cleared in shared memory instead: what a
// page's rest holds is anything, and there it is the common case.
//
// Joining in the first kernel, by the CTA that completes a tile, took longer
// in every case (cold instructions, registers of the softmax).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>

#include "common.cuh"
#include "sm100.cuh"

namespace fade {

constexpr int kBlk = 128;              // keys per block
constexpr int kHalf = 128;             // rows of a half tile
constexpr int kCaThreads = 384;
constexpr int kCaSmemMax = 232448;     // 227 KB
// Cost of a tile: a key of one half tile is kCostOne (a block takes about
// 1.25 us: HBM, or the chain of a stream), of two half tiles kCostTwo (1.85 us),
// its start and end (first loads, output) kTileCost (about 2 us).
constexpr int kCostOne = 2, kCostTwo = 3;
constexpr int kTileCost = 384;
constexpr int kMinShare = 384;         // least work of a CTA: a block per stream, and a block of any tile
static_assert(kMinShare >= kCostTwo * kBlk, "every cut past a tile's start must move it by a block");
constexpr float kLazyMax = 8.f;        // weights may grow to 2^8 before the maximum is moved
constexpr uint32_t kCaPolls = 1u << 22;   // polls of a wait before it gives up, unless the host asks for fewer
constexpr uint32_t kSegPolls = 1u << 26;

struct Walk;

struct ChunkParams {
    const int32_t* block_table;
    const int32_t* cu_q;
    const int32_t* kv_lens;
    void* out;
    float* lse;
    int* err;
    int4* rec;          // [CTA][2]: the tile that begins in the CTA and crosses a cut; rows to look at again
    Walk* walks;        // [CTA]: the walk of its tiles, where rows are to be looked at again
    float2* part_ml;    // [CTA][continued tile, begun tile][256]: (maximum in the log2 domain, sum)
    float4* part_o;     // [CTA][2][D / 8][256][2]
    const void *q, *k_pool, *v_pool;
    int64_t table_stride, o_st, o_sh, q_st, q_sh, kp_sp, kp_sh, kp_st, vp_sp, vp_sh, vp_st;
    uint32_t tile_magic;   // division by the tokens of a tile
    int tile_shift;
    int R, T, Hq, Hkv, g, tq, page_log2, n_pages, table_width, causal, window, out32, fill_rest;
    float scale_log2, lazy;   // lazy: how far a score may exceed the running maximum
    uint32_t polls;           // of a wait before it gives up
};

// ---------------------------------------------------------------------------
// Work split: costs of tiles and their prefix sums
// ---------------------------------------------------------------------------
struct Req {
    int q0, qlen, kv, off;   // first token, tokens, keys, position of the first token
};
__device__ __forceinline__ Req load_req(const ChunkParams& p, int b) {
    Req r;
    const int c0 = p.cu_q[b], c1 = p.cu_q[b + 1];
    r.q0 = c0;
    r.qlen = c0 >= 0 && c1 <= p.T && c1 > c0 ? c1 - c0 : 0;
    r.kv = min(max(p.kv_lens[b], 0), p.table_width << p.page_log2);
    r.off = r.kv - r.qlen;
    return r;
}
// x / (tokens of a tile), for 0 <= x < 2^31
__device__ __forceinline__ uint32_t div_tile(const ChunkParams& p, uint32_t x) {
    return __umulhi(x, p.tile_magic) >> p.tile_shift;
}
// sum over i < n of clamp(a + i t, 0, L), t the tokens of a tile
__device__ __forceinline__ int64_t clamped_sum(const ChunkParams& p, int a, int L, int n) {
    const int t = 2 * p.tq;
    const int n0 = a >= 0 ? 0 : (int)min((uint32_t)n, div_tile(p, (uint32_t)(-a) + t - 1));
    const int n1 = a >= L ? 0 : (int)min((uint32_t)n, div_tile(p, (uint32_t)L - (uint32_t)a + t - 1));
    const int64_t m = max(n1 - n0, 0);
    return a * m + t * (((int64_t)n0 + n1 - 1) * m / 2) + (int64_t)L * (n - max(n1, n0));
}
__device__ __forceinline__ int tiles_of(const ChunkParams& p, const Req& r) {
    return (int)div_tile(p, (uint32_t)r.qlen + 2 * p.tq - 1);
}
// keys [lo, hi) that some row of a tile of n tokens from position pos on sees
__device__ __forceinline__ int keys_end(const ChunkParams& p, const Req& r, int pos, int n) {
    return p.causal ? min(max(pos + n, 0), r.kv) : r.kv;
}
__device__ __forceinline__ int keys_begin(const ChunkParams& p, int pos, int end) {
    return p.window > 0 ? min(max(pos - p.window + 1, 0), end) : 0;
}
// cost of the first n of a request's nt tiles (for one kv head)
__device__ __forceinline__ int64_t tiles_cost(const ChunkParams& p, const Req& r, int n, int nt) {
    const int t = 2 * p.tq;
    int64_t keys = p.causal ? clamped_sum(p, r.off + t, r.kv, n) : (int64_t)r.kv * n;
    if (p.window > 0) keys -= clamped_sum(p, r.off - p.window + 1, r.kv, n);
    int64_t c = (int64_t)kTileCost * n + kCostTwo * keys;
    if (n == nt && n > 0 && r.qlen - (n - 1) * t <= p.tq) {   // the last tile has one half tile only
        const int pos = r.off + (n - 1) * t, end = keys_end(p, r, pos, r.kv - pos);
        c -= (kCostTwo - kCostOne) * (end - keys_begin(p, pos, end));
    }
    return c;
}

// A tile, or the part of its key blocks that a CTA works on; handed from the
// walking warp to the others through shared memory.
struct __align__(16) Seg {
    int k0, k1;                // key blocks of this segment
    int n;                     // tokens of the tile; 0 ends the list
    int kv;                    // keys of the request
    int tok, pos;              // first token (in q) and its position
    int b, h;                  // request, kv head
    int lo_blk, hi_blk;        // key blocks of the whole tile
    int begins, unused;        // the tile begins in this CTA
};
constexpr int kSegSlots = 4;

// CTA c has the costs [first(c), first(c + 1)): `each`, and one more for the
// first `rest`.
__device__ __forceinline__ int64_t split_first(int64_t each, int rest, int c) { return each * c + min(c, rest); }

// The key block that a cut at cost y of a tile falls on.
struct Tile {
    int lo, hi, lo_blk, hi_blk, each, cost;
    __device__ __forceinline__ Tile(const ChunkParams& p, int pos, int n, int kv) {
        hi = p.causal ? min(max(pos + n, 0), kv) : kv;
        lo = keys_begin(p, pos, hi);
        lo_blk = lo / kBlk;
        hi_blk = hi > lo ? (hi + kBlk - 1) / kBlk : lo_blk;
        each = n > p.tq ? kCostTwo : kCostOne;
        cost = kTileCost + each * (hi - lo);
    }
    __device__ __forceinline__ int cut(int64_t y) const {
        if (y <= 0) return lo_blk;
        if (y >= cost) return hi_blk;
        return min(max((lo + max((int)y - kTileCost, 0) / each) / kBlk, lo_blk), hi_blk);
    }
};

struct Walk {
    Req r;
    int b, h, i, nt, cta, rest;
    int64_t pos, x0, x1, each; // cost position of the tile, range of the CTA
    int parts_from, parts_to, parts_n, parts_tok, parts_h, parts_b;   // the tile that begins here and crosses x1

    __device__ __forceinline__ bool next(const ChunkParams& p, Seg& s) {
        while (pos < x1) {
            const int t = 2 * p.tq, t0 = i * t;
            s.n = min(t, r.qlen - t0);
            s.kv = r.kv;
            s.tok = r.q0 + t0, s.pos = r.off + t0;
            s.b = b, s.h = h;
            const Tile tile(p, s.pos, s.n, r.kv);
            s.lo_blk = tile.lo_blk, s.hi_blk = tile.hi_blk;
            s.k0 = tile.cut(x0 - pos);
            s.k1 = tile.cut(x1 - pos);
            const bool begins = pos >= x0;
            s.begins = begins;
            if (begins && pos + tile.cost > x1) {   // the last tile here: which CTAs have a part of it?
                int from = cta;
                while (tile.cut(split_first(each, rest, from + 1) - pos) == tile.lo_blk && tile.lo_blk < tile.hi_blk) ++from;
                int to = from;
                while (tile.cut(split_first(each, rest, to + 1) - pos) < tile.hi_blk) ++to;
                parts_from = from, parts_to = to, parts_n = s.n, parts_tok = s.tok, parts_h = h, parts_b = b;
            }
            pos += tile.cost;
            if (++i == nt) {
                i = 0;
                if (++h == p.Hkv) {
                    h = 0;
                    while (pos < x1 && ++b < p.R) {
                        r = load_req(p, b);
                        if (r.qlen > 0) break;
                    }
                    nt = tiles_of(p, r);
                }
            }
            if (s.k1 > s.k0 || (s.lo_blk == s.hi_blk && begins)) return true;
        }
        return false;
    }
};

// ---------------------------------------------------------------------------
// Device helpers
// ---------------------------------------------------------------------------
// A wait of any call on this device gave up (captured calls have workspaces that nobody asks).
__device__ int g_gave_up;

// Waits are bounded.  One that runs out sets the CTA's flag and the error words,
// and every other wait of the CTA gives up after it.  The lanes of a warp may
// see that at different polls, so a warp goes on or stops by a vote of its
// lanes; a warp that stops starts no more copies or products, waits for those
// it has started (settle) and meets the others at the end of the kernel.
__device__ __forceinline__ void report(const ChunkParams& p) {
    atomicExch(p.err, 1);
    atomicExch(&g_gave_up, 1);
}
__device__ __forceinline__ bool ca_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, const ChunkParams& p) {
    for (uint32_t i = 0; i < p.polls; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255u) == 255u && *abort_flag) return false;
    }
    *abort_flag = 1;
    report(p);
    return false;
}
// the same answer for the whole warp
__device__ __forceinline__ bool ca_wait_all(uint32_t bar, uint32_t parity, volatile int* abort_flag, const ChunkParams& p) {
    return __all_sync(~0u, ca_wait(bar, parity, abort_flag, p));
}
// For what this warp has started itself: it ends by itself, given up or not.
__device__ __forceinline__ void settle(uint32_t bar, uint32_t parity, const ChunkParams& p) {
    for (uint32_t i = 0; i < kCaPolls; ++i)
        if (mbar_try_wait(bar, parity)) return;
    report(p);
}
__device__ __forceinline__ void mbar_arrive_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar),
                 "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
#define CA_R32(v, o)                                                                                              \
    "=r"(v[o + 0]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), \
        "=r"(v[o + 7]), "=r"(v[o + 8]), "=r"(v[o + 9]), "=r"(v[o + 10]), "=r"(v[o + 11]), "=r"(v[o + 12]),         \
        "=r"(v[o + 13]), "=r"(v[o + 14]), "=r"(v[o + 15]), "=r"(v[o + 16]), "=r"(v[o + 17]), "=r"(v[o + 18]),      \
        "=r"(v[o + 19]), "=r"(v[o + 20]), "=r"(v[o + 21]), "=r"(v[o + 22]), "=r"(v[o + 23]), "=r"(v[o + 24]),      \
        "=r"(v[o + 25]), "=r"(v[o + 26]), "=r"(v[o + 27]), "=r"(v[o + 28]), "=r"(v[o + 29]), "=r"(v[o + 30]),      \
        "=r"(v[o + 31])
#define CA_RW32(v, o)                                                                                             \
    "+r"(v[o + 0]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), "+r"(v[o + 4]), "+r"(v[o + 5]), "+r"(v[o + 6]), \
        "+r"(v[o + 7]), "+r"(v[o + 8]), "+r"(v[o + 9]), "+r"(v[o + 10]), "+r"(v[o + 11]), "+r"(v[o + 12]),         \
        "+r"(v[o + 13]), "+r"(v[o + 14]), "+r"(v[o + 15]), "+r"(v[o + 16]), "+r"(v[o + 17]), "+r"(v[o + 18]),      \
        "+r"(v[o + 19]), "+r"(v[o + 20]), "+r"(v[o + 21]), "+r"(v[o + 22]), "+r"(v[o + 23]), "+r"(v[o + 24]),      \
        "+r"(v[o + 25]), "+r"(v[o + 26]), "+r"(v[o + 27]), "+r"(v[o + 28]), "+r"(v[o + 29]), "+r"(v[o + 30]),      \
        "+r"(v[o + 31])
// 32 columns of this warp's 32 lanes; the values may be read after tc_wait_ld32 on them
template <int N>
__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t (&v)[N], int o) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : CA_R32(v, o)
        : "r"(taddr)
        : "memory");
}
template <int N>
__device__ __forceinline__ void tc_wait_ld32(uint32_t (&v)[N], int o) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : CA_RW32(v, o) : : "memory");
}
template <int N>
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&v)[N], int o) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(v[o + 0]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]),
        "r"(v[o + 7]), "r"(v[o + 8]), "r"(v[o + 9]), "r"(v[o + 10]), "r"(v[o + 11]), "r"(v[o + 12]), "r"(v[o + 13]),
        "r"(v[o + 14]), "r"(v[o + 15]), "r"(v[o + 16]), "r"(v[o + 17]), "r"(v[o + 18]), "r"(v[o + 19]),
        "r"(v[o + 20]), "r"(v[o + 21]), "r"(v[o + 22]), "r"(v[o + 23]), "r"(v[o + 24]), "r"(v[o + 25]),
        "r"(v[o + 26]), "r"(v[o + 27]), "r"(v[o + 28]), "r"(v[o + 29]), "r"(v[o + 30]), "r"(v[o + 31])
        : "memory");
}
// pairs of fp32 values in one instruction
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (DT == FADE_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// N results as N / 2 pairs.  An average of fp16 values lies within their range,
// but with its weights rounded it may pass 65504 by 2^-11 and would round to an
// infinity: finite results stay within the range.
template <int DT, int N>
__device__ __forceinline__ void pack_results(const float (&f)[N], uint32_t (&y)[N / 2]) {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) y[j] = pack2<DT>(f[2 * j], f[2 * j + 1]);
    if constexpr (DT == FADE_F16) {
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) top = fmaxf(top, fabsf(f[j]));
        if (top > 65504.f) {   // rare
            auto within = [](float x) { return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.f), 65504.f) : x; };
#pragma unroll
            for (int j = 0; j < N / 2; ++j) y[j] = pack2<DT>(within(f[2 * j]), within(f[2 * j + 1]));
        }
    }
}
// 32 bytes of a row: one store where every row is 32-byte aligned (a warp stores 32 rows, each its own cache line,
// and the lines, not the bytes, bound it)
template <int N>
__device__ __forceinline__ void st_row32(void* dst, const uint32_t (&v)[N], int o, int aligned) {
    if (aligned) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[o]), "r"(v[o + 1]),
                     "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
                     : "memory");
    } else {
        static_cast<uint4*>(dst)[0] = make_uint4(v[o], v[o + 1], v[o + 2], v[o + 3]);
        static_cast<uint4*>(dst)[1] = make_uint4(v[o + 4], v[o + 5], v[o + 6], v[o + 7]);
    }
}
// Instruction descriptor, kind::f16: f32 accumulator, A and B in the model dtype, M = 128, N columns;
// b_mn: B is MN-major.
template <int DT>
__host__ __device__ constexpr uint32_t ca_idesc(int n, bool b_mn) {
    return (1u << 4) | ((DT == FADE_BF16 ? 1u : 0u) << 7) | ((DT == FADE_BF16 ? 1u : 0u) << 10) |
           ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// Shared memory.  Q, K and V tiles are 128 rows of 128 bytes (64 channels) in
// the 128-byte swizzle, one such sub-tile per 64 channels.
template <int D>
struct CaLayout {
    static constexpr int SUB = 128 * 128;                  // a sub-tile
    static constexpr int TILE = SUB * (D / 64);            // 128 rows of D channels
    static constexpr int Q_OFF = 0;
    static constexpr int RING_OFF = 2 * TILE;
    static constexpr int NS = D == 128 ? 5 : 11;           // ring stages, one K or V block each
    static constexpr int ML_OFF = RING_OFF + NS * TILE;    // (m, l) of both streams
    static constexpr int BAR_OFF = ML_OFF + 2 * 128 * 8;
    static constexpr int N_BARS = 2 * NS + 23 + 2 * kSegSlots;
    static constexpr int MISC_OFF = BAR_OFF + 8 * N_BARS;  // tensor-memory slot, abort flag, output not finite
    static constexpr int SEG_OFF = (MISC_OFF + 16 + 15) / 16 * 16;
    static constexpr int SUM_OFF = SEG_OFF + kSegSlots * (int)sizeof(Seg);   // costs per warp
    static constexpr int WALK_OFF = SUM_OFF + kCaThreads / 32 * 8;          // the walk at its start
    static constexpr int BYTES = WALK_OFF + (int)sizeof(Walk);
    static_assert(BYTES <= kCaSmemMax, "chunk attention shared memory over the per-CTA limit");
};
constexpr int kColS = 0;      // two score tiles of 128 columns; the weights overlay the first 64 of each
constexpr int kColO = 256;    // two output tiles of D columns

template <int DT, int D>
__global__ void __launch_bounds__(kCaThreads, 1)
    chunk_attn_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                      const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ ChunkParams p) {
    using L = CaLayout<D>;
    using T = typename Elem<DT>::T;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sb = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid % 32;
    const int warp = __shfl_sync(~0u, tid / 32, 0);   // known to be the same for the whole warp
    const int cta = blockIdx.x, G = gridDim.x;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 8);
    volatile int* dirty = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 12);
    const uint32_t bars = sb + L::BAR_OFF;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (L::NS + s); };
    const uint32_t b1 = bars + 16u * L::NS;
    auto q_full = [&](int x) { return b1 + 8u * x; };
    auto q_empty = [&](int x) { return b1 + 8u * (2 + x); };
    auto s_full = [&](int x) { return b1 + 8u * (4 + x); };
    auto p_full = [&](int x) { return b1 + 8u * (6 + x); };
    auto o_full = [&](int x) { return b1 + 8u * (8 + x); };
    auto seg_full = [&](int x) { return b1 + 8u * (10 + x); };
    auto seg_empty = [&](int x) { return b1 + 8u * (10 + kSegSlots + x); };
    const uint32_t both = b1 + 8u * (10 + 2 * kSegSlots);   // the softmax warps meet
    auto h_full = [&](int x) { return b1 + 8u * (11 + 2 * kSegSlots + x); };   // weights of the block's first half
    auto turn = [&](int x, int w) { return b1 + 8u * (13 + 2 * kSegSlots + 4 * x + w); };   // warp w of stream x may take exponentials

    auto done = [&](int x) { return b1 + 8u * (21 + 2 * kSegSlots + x); };   // products of stream x, when its MMA warp ends

    if (sb & 1023u) {   // the swizzled tiles need 1 KB alignment
        if (tid == 0) {
            report(p);
            p.rec[cta * 2] = p.rec[cta * 2 + 1] = make_int4(0, 0, 0, 0);
        }
        return;
    }
    if (tid == 0) {
        *abort_flag = *dirty = 0;
        for (int s = 0; s < L::NS; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 2);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(q_full(x), 1);
            mbar_init(q_empty(x), 2);
            mbar_init(s_full(x), 1);
            mbar_init(p_full(x), 4);
            mbar_init(h_full(x), 4);
            mbar_init(o_full(x), 1);
            mbar_init(done(x), 1);
        }
        mbar_init(both, 8);
        for (int i = 0; i < 8; ++i) mbar_init(turn(i / 4, i % 4), 1);
        for (int x = 0; x < kSegSlots; ++x) {
            mbar_init(seg_full(x), 1);
            mbar_init(seg_empty(x), 11);   // loads, two MMA and eight softmax warps
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        tc_alloc(sb + L::MISC_OFF, 512);
        tc_relinquish();
    }

    // ---- costs of the requests, summed per warp (the walking warp finds this CTA's share) ----
    int64_t* sums = reinterpret_cast<int64_t*>(smem + L::SUM_OFF);
    const int per = (p.R + kCaThreads - 1) / kCaThreads;   // requests of a thread
    auto cost_of = [&](int first, int n) {
        int64_t c = 0;
        for (int b = first; b < min(first + n, p.R); ++b) {
            const Req r = load_req(p, b);
            const int nt = tiles_of(p, r);
            c += tiles_cost(p, r, nt, nt);
        }
        return c;
    };
    // prefix sums within the warps, where the first Q tile comes later
    int64_t* scan = reinterpret_cast<int64_t*>(smem + L::Q_OFF);
    {
        int64_t c = cost_of(tid * per, per);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(~0u, c, o);
            if (lane >= o) c += v;
        }
        scan[tid] = c;
        if (lane == 31) sums[warp] = c;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + L::MISC_OFF);
    griddep_launch_dependents();
    Seg* segs = reinterpret_cast<Seg*>(smem + L::SEG_OFF);
    Seg s;
    int seg = 0;
    uint32_t seg_phase = 0;
    // the next posted segment; every lane reads it, one says so
    auto next_seg = [&] {
        const bool ok = ca_wait_all(seg_full(seg), seg_phase, abort_flag, p);
        s = segs[seg];
        __syncwarp();
        if (lane == 0) mbar_arrive(seg_empty(seg));
        if (++seg == kSegSlots) seg = 0, seg_phase ^= 1u;
        return ok && s.n > 0;
    };

    // 384 threads x 168 registers at launch: 256 x 216 + 128 x 72 stay below that
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 8) {
            // ---------------------------- loads ----------------------------
            if (lane == 0) {
                asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_q)) : "memory");
                asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_k)) : "memory");
                asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_v)) : "memory");
            }
            const int ppb = kBlk >> p.page_log2;
            // lane = page of the block + ppb * sub-tile
            const int my_page = lane % ppb, my_sub = lane / ppb;
            const uint32_t my_dst = sb + L::RING_OFF + my_sub * L::SUB + ((my_page * 128) << p.page_log2);
            uint32_t q_phase = 3;   // bit x: parity to wait for on buffer x
            int flip = 0, stage = 0;
            uint32_t phase = 1;
            bool run = true;
            while (run && next_seg()) {
                if (s.k1 == s.k0) continue;
                const bool two = s.n > p.tq;
                for (int x = two ? 0 : flip; x < (two ? 2 : flip + 1); ++x) {
                    run = ca_wait_all(q_empty(x), (q_phase >> x) & 1u, abort_flag, p);
                    if (!run) break;
                    q_phase ^= 1u << x;
                    if (lane == 0) {
                        mbar_arrive_tx(q_full(x), 128u * (D / 64) * p.g * p.tq);
                        for (int c = 0; c < D / 64; ++c)
                            tma_load_3d(sb + L::Q_OFF + x * L::TILE + c * L::SUB, &tmap_q, c * 64, s.h * p.g,
                                        s.tok + (two ? x * p.tq : 0), q_full(x));
                    }
                }
                if (!two) flip ^= 1;
                // page ids, 32 entries at a time: this group and the next
                const int32_t* row = p.block_table + s.b * p.table_stride;
                const int n_pg = (s.kv + (1 << p.page_log2) - 1) >> p.page_log2;
                auto entry = [&](int at) {
                    const int id = at < n_pg ? row[at] : p.n_pages;
                    return (uint32_t)id < (uint32_t)p.n_pages ? id : p.n_pages;   // beyond the pool: zeros
                };
                int base = s.k0 * ppb & ~31;
                int cur = entry(base + lane), nxt = entry(base + 32 + lane);
                for (int kb = s.k0; run && kb < s.k1; ++kb) {
                    if (kb * ppb >= base + 32) {
                        base += 32;
                        cur = nxt;
                        nxt = entry(base + 32 + lane);
                    }
                    const int id = __shfl_sync(~0u, cur, (kb * ppb + my_page) & 31);
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        run = ca_wait_all(empty(stage), phase, abort_flag, p);
                        if (!run) break;
                        if (lane == 0) mbar_arrive_tx(full(stage), L::TILE);
                        __syncwarp();
                        if (my_sub < D / 64)
                            tma_load_4d(my_dst + stage * L::TILE, kv ? &tmap_v : &tmap_k, my_sub * 64, 0, s.h, id,
                                        full(stage));
                        if (++stage == L::NS) stage = 0, phase ^= 1u;
                    }
                }
            }
            // every copy has landed before the CTA may exit, and where nothing gave up has been used
            for (int i = 0; i < L::NS; ++i) settle(full(i), i < stage ? phase ^ 1u : phase, p);
            for (int x = 0; x < 2; ++x) settle(q_full(x), (q_phase >> x) & 1u, p);
            for (int i = 0; i < L::NS; ++i) {
                ca_wait(empty(stage), phase, abort_flag, p);
                if (++stage == L::NS) stage = 0, phase ^= 1u;
            }
        } else if (warp == 9 || warp == 11) {
            // ---------------------- MMA, a warp per stream ----------------------
            // Waits and commits take a warp about as long as half of a block's
            // MMAs, so each stream has its own.  The whole warp walks the loop
            // (addresses and descriptors stay in uniform registers), one lane
            // issues.  Both warps go through every fill of every buffer, also
            // where only the other one uses it (two arrivals free a buffer):
            // a warp that skipped fills could mistake one for another.
            const int st = warp == 9 ? 0 : 1;
            const bool elected = elect_one();
            bool run = true, lead = elected;     // lead: this lane issues
            constexpr uint32_t IQK = ca_idesc<DT>(kBlk, false), IPV = ca_idesc<DT>(D, true);
            const uint64_t q_desc = tc_desc(sb + L::Q_OFF, 16, 1024, 2);
            const uint64_t k_desc = tc_desc(sb + L::RING_OFF, 16, 1024, 2);
            const uint64_t v_desc = tc_desc(sb + L::RING_OFF, L::SUB, 1024, 2);
            const uint32_t ts = tmem + kColS + 128 * st, to = tmem + kColO + D * st;
            uint32_t q_phase = 0, p_phase = 0;   // bit x of q_phase: parity to wait for on buffer x
            int flip = 0, stage = 0;             // next ring stage: K, V, K, V, ... of the blocks
            uint32_t phase = 0;
            auto wait = [&](uint32_t bar, uint32_t parity) {
                run = run && ca_wait_all(bar, parity, abort_flag, p);
                lead = elected && run;
            };
            auto landed = [&] { wait(full(stage), phase); };
            auto advance = [&] {
                if (++stage == L::NS) stage = 0, phase ^= 1u;
            };
            auto pass = [&] {   // a block of the other stream
                for (int i = 0; i < 2; ++i) {
                    landed();
                    if (lead) mbar_arrive(empty(stage));
                    advance();
                }
                __syncwarp();
            };
            while (run && next_seg()) {
                const int nb = s.k1 - s.k0;
                if (nb == 0) continue;
                const bool two = s.n > p.tq;
                if (two || flip == 0) wait(q_full(0), q_phase & 1u);
                if (two || flip == 1) wait(q_full(1), q_phase >> 1);
                const int x = two ? st : flip;   // Q buffer
                q_phase ^= two ? 3u : 1u << flip;
                if (!two) flip ^= 1;
                const int mine = two ? nb : (nb + 1 - st) / 2;
                if (lead && two) mbar_arrive(q_empty(st ^ 1));
                if (lead && mine == 0) mbar_arrive(q_empty(x));
                const uint64_t a = q_desc + (uint32_t)(x * (L::TILE >> 4));
                auto scores = [&](bool last) {   // of the block whose K is next in the ring
                    const uint64_t b = k_desc + (uint32_t)(stage * (L::TILE >> 4));
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const uint32_t o = (i >> 2) * (L::SUB >> 4) + (i & 3) * 2;
                        tc_mma_ss(ts, a + o, b + o, IQK, i > 0 ? 1u : 0u);
                    }
                    tc_commit(s_full(st));
                    tc_commit(empty(stage));
                    if (last) tc_commit(q_empty(x));
                };
                if (!two && st == 1) pass();
                if (mine > 0) {
                    landed();
                    tc_fence_after();
                    if (lead) scores(mine == 1);
                    __syncwarp();
                    advance();
                }
                for (int j = 0; run && j < mine; ++j) {
                    const bool more = j + 1 < mine, now = two && more;   // the next scores follow at once
                    landed();
                    const uint64_t b = v_desc + (uint32_t)(stage * (L::TILE >> 4));
                    const uint32_t v_empty = empty(stage);
                    advance();
                    if (now) landed();
                    wait(h_full(st), p_phase);
                    tc_fence_after();
                    if (lead) {
                        tc_mma_ts(to, ts, b, IPV, j > 0 ? 1u : 0u);
#pragma unroll
                        for (int i = 1; i < kBlk / 32; ++i) tc_mma_ts(to, ts + 8 * i, b + (uint32_t)(i * 128), IPV, 1u);
                    }
                    __syncwarp();
                    wait(p_full(st), p_phase);
                    p_phase ^= 1u;
                    tc_fence_after();
                    if (lead) {
#pragma unroll
                        for (int i = kBlk / 32; i < kBlk / 16; ++i)
                            tc_mma_ts(to, ts + 8 * i, b + (uint32_t)(i * 128), IPV, 1u);
                        if (now) scores(j + 2 == mine);
                        if (!more) tc_commit(o_full(st));
                        tc_commit(v_empty);
                    }
                    __syncwarp();
                    if (now) advance();
                    if (!two) {
                        if (2 * j + st + 1 < nb) pass();
                        if (more) {
                            landed();
                            tc_fence_after();
                            if (lead) scores(j + 2 == mine);
                            __syncwarp();
                            advance();
                        }
                    }
                }
            }
            // the products have ended before tensor memory is given back and the CTA exits
            if (elected) tc_commit(done(st));
            __syncwarp();
            settle(done(st), 0, p);
        } else if (warp == 10) {
            // ------------------------ tiles, in order ------------------------
            // Range of this CTA: [x0, x1) of the total cost W, of which the
            // first CTAs take one more when it does not divide.
            Walk walk;
            int64_t W = 0;
#pragma unroll
            for (int w = 0; w < kCaThreads / 32; ++w) W += sums[w];
            W *= p.Hkv;
            const int n_cta = W == 0 ? 0 : (int)min((int64_t)G, max((int64_t)1, W / kMinShare));
            // (a 64-bit division costs several times a 32-bit one)
            const int64_t each = n_cta == 0 ? 0 : W >> 32 ? W / n_cta : (int64_t)((uint32_t)W / (uint32_t)n_cta);
            const int rest = (int)(W - each * n_cta);
            walk.cta = cta, walk.each = each, walk.rest = rest, walk.parts_from = walk.parts_to = 0;
            walk.x0 = cta < n_cta ? split_first(each, rest, cta) : 0;
            walk.x1 = cta < n_cta ? split_first(each, rest, cta + 1) : 0;
            walk.pos = 0;
            if (cta < n_cta) {
                // the warp's, the lane's, the request and the tile that x0 lies in
                int64_t at = 0;
                int w = 0;
                for (; w + 1 < kCaThreads / 32 && walk.x0 >= at + sums[w] * p.Hkv; ++w) at += sums[w] * p.Hkv;
                const int64_t incl = scan[w * 32 + lane] * p.Hkv;
                const int who = __ffs(__ballot_sync(~0u, walk.x0 < at + incl)) - 1;
                const int64_t before = who > 0 ? scan[w * 32 + who - 1] : 0, here = scan[w * 32 + who] - before;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                at += before * p.Hkv;
                walk.b = (w * 32 + who) * per;
                int64_t c;
                for (;; ++walk.b) {
                    walk.r = load_req(p, walk.b);
                    walk.nt = tiles_of(p, walk.r);
                    c = per == 1 ? here : tiles_cost(p, walk.r, walk.nt, walk.nt);
                    if (walk.x0 < at + c * p.Hkv || walk.b + 1 >= p.R) break;
                    at += c * p.Hkv;
                }
                // a kv head's tiles cost c
                walk.h = 0;
                while (walk.h + 1 < p.Hkv && walk.x0 >= at + c) at += c, ++walk.h;
                walk.i = 0;
                for (int span = walk.nt; span > 1;) {   // 32 parts of the remaining tiles
                    const int step = (span + 31) / 32, i = walk.i + lane * step;
                    const bool below = lane * step < span && at + tiles_cost(p, walk.r, i, walk.nt) <= walk.x0;
                    const int k = __popc(__ballot_sync(~0u, below)) - 1;
                    span = min(step, span - k * step);
                    walk.i += k * step;
                }
                walk.pos = at + (walk.i > 0 ? tiles_cost(p, walk.r, walk.i, walk.nt) : 0);
            }
            if (lane == 0) {
                *reinterpret_cast<Walk*>(smem + L::WALK_OFF) = walk;
                bool more = true, run = true;
                while (more) {
                    more = walk.next(p, s);
                    if (!more) s.n = 0;
                    // a segment may take long: look for a free slot now and then
                    for (uint32_t i = 0; run && !mbar_try_wait(seg_empty(seg), seg_phase ^ 1u); ++i) {
                        if (i + 1 == kSegPolls) *abort_flag = 1, report(p);
                        run = !*abort_flag;
                        __nanosleep(200);
                    }
                    if (!run) break;   // the slot may be in use
                    segs[seg] = s;
                    mbar_arrive(seg_full(seg));
                    if (++seg == kSegSlots) seg = 0, seg_phase ^= 1u;
                }
                if (!run) walk.parts_from = walk.parts_to = 0;
                p.rec[cta * 2] = make_int4(walk.parts_from, walk.parts_to, walk.parts_n, walk.parts_tok);
                p.rec[cta * 2 + 1] = make_int4(walk.parts_h, 0, walk.parts_b, 0);
            }
            __syncwarp();
        }
    } else {
        // ----------------------------- softmax -----------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int st = warp / 4, row = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;            // this warp's 32 lanes of tensor memory
        const uint32_t ts = tmem + lanes + kColS + 128 * st, to = tmem + lanes + kColO + D * st;
        const float sl = p.scale_log2;
        float2* ml = reinterpret_cast<float2*>(smem + L::ML_OFF);
        const int tok = row / p.g;                                    // token within the half tile
        uint32_t s_phase = 0, o_phase = 0, ring = 0, meetings = 0, turn_phase = st ^ 1;
        const uint32_t my_turn = turn(st, warp & 3), their_turn = turn(st ^ 1, warp & 3);
        auto meet = [&] {   // a bounded wait, so that no warp is left behind when another gave up
            __syncwarp();
            if (lane == 0) mbar_arrive(both);
            ca_wait(both, meetings & 1u, abort_flag, p);
            ++meetings;
            __syncwarp();
        };
        auto release = [&] {
            __syncwarp();
            if (lane == 0) mbar_arrive(seg_empty(seg));
            if (++seg == kSegSlots) seg = 0, seg_phase ^= 1u;
        };
        while (true) {
            // the segment stays in its slot until this warp is through with it
            if (!ca_wait_all(seg_full(seg), seg_phase, abort_flag, p)) break;
            const Seg& g = segs[seg];
            const int n = g.n;
            if (n <= 0) break;
            const bool two = n > p.tq;
            const int k0 = g.k0, k1 = g.k1;
            const int t = (two ? st * p.tq : 0) + tok;                // token within the tile
            const bool valid = tok < p.tq && t < n;
            const bool warp_on = __any_sync(~0u, valid);
            float m = -INFINITY, l = 0.f;
            int blocks = 0;
            bool ok = true;
            {
                // keys of this row: [kmin, kend); blocks that every row of the half tile sees whole: [free0, free1)
                const int kv = g.kv, first = g.pos + (two ? st * p.tq : 0);
                const int kend = p.causal ? min(first + tok + 1, kv) : kv;
                const int kmin = p.window > 0 ? first + tok - p.window + 1 : 0;
                const int free1 = max(p.causal ? min(first + 1, kv) : kv, 0) / kBlk;
                const int free0 = p.window > 0 ? (max(first + p.tq - p.window, 0) + kBlk - 1) / kBlk : 0;
                const int step = two ? 1 : 2;
                for (int kb = k0 + (two ? 0 : st); kb < k1; kb += step, ++blocks) {
                    ok = ca_wait_all(s_full(st), s_phase, abort_flag, p);
                    if (!ok) break;
                    s_phase ^= 1u;
                    tc_fence_after();
                    // keys past the end of the cache: their V rows (the rest of a page) may hold anything
                    auto clear_rest = [&] {
                        if (kb * kBlk + kBlk <= kv) return;
                        if (!two || st == 0) {
                            const uint32_t vp = ring + 2u * (kb - k0) + 1u;
                            ca_wait(full(vp % L::NS), (vp / L::NS) & 1u, abort_flag, p);
                            const int keep = kv - kb * kBlk;
                            uint8_t* v = smem + L::RING_OFF + (vp % L::NS) * L::TILE;
                            for (int i = row; i < (kBlk - keep) * (D / 8); i += 128) {
                                const int r = keep + i / (D / 8), c = i % (D / 8);
                                *reinterpret_cast<uint4*>(v + (c / 8) * L::SUB + r * 128 + (c % 8) * 16) =
                                    make_uint4(0u, 0u, 0u, 0u);
                            }
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        }
                        if (two) meet();
                    };
                    // The two warps of a scheduler share its exponential unit: taking turns keeps the streams
                    // half a block apart, so that one's MMAs run under the other's exponentials.
                    auto take_turn = [&] {
                        if (!two) return;
                        ca_wait(my_turn, turn_phase, abort_flag, p);
                        turn_phase ^= 1u;
                        __syncwarp();
                    };
                    auto pass_turn = [&] {
                        if (two && lane == 0) mbar_arrive(their_turn);
                    };
                    auto post = [&](uint32_t bar) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar);
                    };
                    if (!warp_on) {
                        clear_rest();
                        take_turn();
                        pass_turn();
                        post(h_full(st));
                        post(p_full(st));
                        continue;
                    }
                    uint32_t x[128];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tc_ld32(ts + 32 * c, x, 32 * c);
#pragma unroll
                    for (int c = 0; c < 4; ++c) tc_wait_ld32(x, 32 * c);
                    if (kb >= free1 || kb < free0) {
                        const int je = kend - kb * kBlk, jm = kmin - kb * kBlk;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {   // 32 keys as a bit mask: [jm, je)
                            const uint32_t below = je >= 32 * c + 32 ? ~0u : je > 32 * c ? (1u << (je - 32 * c)) - 1u : 0u;
                            const uint32_t from = jm <= 32 * c ? ~0u : jm < 32 * c + 32 ? ~0u << (jm - 32 * c) : 0u;
                            const uint32_t keep = below & from;
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!(keep >> j & 1u)) x[32 * c + j] = 0xff800000u;
                        }
                    }
                    float mx[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) mx[c] = fmaxf(__uint_as_float(x[c]), __uint_as_float(x[8 + c]));
#pragma unroll
                    for (int j = 16; j < 128; j += 16)
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            mx[c] = max3(mx[c], __uint_as_float(x[j + c]), __uint_as_float(x[j + 8 + c]));
                    const float bm = fmaxf(max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[4]), max3(mx[5], mx[6], mx[7]));
                    const bool need = bm > m + p.lazy;
                    if (__any_sync(~0u, need)) {
                        const float mn = need ? bm : m;
                        const float a = need ? ex2((m - mn) * sl) : 1.f;
                        m = mn;
                        l *= a;
                        if (blocks > 0) {   // the output so far, in tensor memory, to the new maximum
#pragma unroll
                            for (int c = 0; c < D; c += 16) {
                                uint32_t o[16];
                                tc_ld16(to + c, o);
#pragma unroll
                                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * a);
                                tc_st16(to + c, o);
                            }
                        }
                    }
                    clear_rest();
                    take_turn();
                    const float off = m == -INFINITY ? 0.f : m * sl;
                    const uint64_t sl2 = pair(sl, sl), off2 = pair(-off, -off);
                    uint64_t sum[4] = {0, 0, 0, 0};
                    // weights, rounded, into the place of the scores
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const int k = 64 * c + 2 * j;
                            const uint64_t y = fma2(pair(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), sl2, off2);
                            float a, b;
                            unpair(y, a, b);
                            a = ex2(a), b = ex2(b);
                            sum[j & 3] = add2(sum[j & 3], pair(a, b));
                            w[j] = pack2<DT>(a, b);
                        }
                        if (c == 1) pass_turn();
                        tc_st32(ts + 32 * c, w, 0);
                        tc_wait_st();
                        post(c == 0 ? h_full(st) : p_full(st));
                    }
                    float a, b;
                    unpair(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), a, b);
                    l += a + b;
                }
            }
            if (!ok) break;
            const int nb = k1 - k0;
            ring += 2u * nb;
            const int64_t orow = (int64_t)g.tok + t;
            const int hq = g.h * p.g + row % p.g;
            T* orow_p = static_cast<T*>(p.out) + orow * p.o_st + (int64_t)hq * p.o_sh;
            if (nb == 0 && valid && (two || st == 0)) {   // no key is visible
                for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(orow_p + c) = make_uint4(0u, 0u, 0u, 0u);
                if (p.lse) p.lse[orow * p.Hq + hq] = -INFINITY;
            }
            const bool whole = k0 == g.lo_blk && k1 == g.hi_blk;
            const int slot = cta * 2 + g.begins;
            release();
            if (nb == 0) continue;
            if (blocks > 0) {
                if (!ca_wait_all(o_full(st), o_phase, abort_flag, p)) break;
                o_phase ^= 1u;
            }
            __syncwarp();
            tc_fence_after();
            // ---- this stream's rows, or both streams' halves of the channels ----
            float e0 = 1.f, e1 = 0.f;   // factors of the outputs of streams 0 and 1
            float mlog = m * sl;        // -inf while no key was seen
            if (!two) {
                ml[st * 128 + row] = make_float2(mlog, l);
                tc_fence_before();
                meet();
                tc_fence_after();
                const float2 a = ml[row], b = ml[128 + row];
                mlog = fmaxf(a.x, b.x);
                e0 = a.x == -INFINITY ? 0.f : ex2(a.x - mlog);
                e1 = b.x == -INFINITY ? 0.f : ex2(b.x - mlog);
                l = a.y * e0 + b.y * e1;
            }
            const float inv = !whole ? 1.f : l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
            const int prow = two ? st * 128 + row : row;
            const int c0 = two ? 0 : st * (D / 2), c1 = two ? D : c0 + D / 2;
            uint64_t zero = 0;          // NaN once an output is not finite
            if (warp_on) {
                const uint32_t t0 = tmem + lanes + kColO + (two ? D * st : 0);
                for (int c = c0; c < c1; c += 32) {
                    uint32_t o[32], o1[32];
                    tc_ld32(t0 + c, o, 0);
                    const bool more = !two && nb > 1;
                    if (more) tc_ld32(t0 + D + c, o1, 0);
                    tc_wait_ld32(o, 0);
                    float f[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(o[j]) * e0;
                    if (more) {
                        tc_wait_ld32(o1, 0);
#pragma unroll
                        for (int j = 0; j < 32; ++j) f[j] += __uint_as_float(o1[j]) * e1;
                    }
                    if (valid && whole) {
                        uint32_t y[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) zero = fma2(pair(f[2 * j], f[2 * j + 1]), 0, zero);
#pragma unroll
                        for (int j = 0; j < 32; ++j) f[j] *= inv;
                        pack_results<DT>(f, y);
#pragma unroll
                        for (int j = 0; j < 16; j += 8) st_row32(orow_p + c + 2 * j, y, j, p.out32);
                    } else if (valid) {   // [channel / 8][row][8]: consecutive rows next to each other
                        uint32_t y[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) y[j] = __float_as_uint(f[j]);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            st_row32(p.part_o + (((int64_t)slot * (D / 8) + c / 8 + j) * 256 + prow) * 2, y, 8 * j, 1);
                    }
                    __syncwarp();
                }
            }
            float z0, z1;
            unpair(zero, z0, z1);
            if (!(z0 + z1 == 0.f)) *dirty = 1;
            if (valid && (two || st == 0)) {
                if (!whole) p.part_ml[slot * 256 + prow] = make_float2(mlog, l);
                else if (p.lse) p.lse[orow * p.Hq + hq] = l == 0.f ? -INFINITY : 0.69314718056f * (mlog + __log2f(l));
            }
            tc_fence_before();
            if (!two) meet();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tc_dealloc(tmem, 512);
    if (tid == 0 && *dirty) {
        p.walks[cta] = *reinterpret_cast<Walk*>(smem + L::WALK_OFF);
        reinterpret_cast<int*>(p.rec + cta * 2 + 1)[1] = 1;
    }
}

// A warp looks again at the output of one row, which sees the keys [kmin, kend)
// of the [lo, hi) that its tile went through.  If it is not finite and a V of
// the tile's other keys is not, it is computed anew; from its last key, because
// a request gone bad is bad from some token on, and with every channel in
// question reached by a key that the row does see (or by a score), the row
// stays as it is.
template <int DT, int D>
__device__ __forceinline__ void mend_row(const ChunkParams& p, int b, int h, int hq, int64_t t, int kmin, int kend, int lo,
                                      int hi) {
    using T = typename Elem<DT>::T;
    constexpr int N = D / 32;                              // channels of a lane
    const int lane = threadIdx.x % 32;
    T* out = static_cast<T*>(p.out) + t * p.o_st + (int64_t)hq * p.o_sh + lane * N;
    auto finite = [](const T* x) {
        bool ok = true;
#pragma unroll
        for (int c = 0; c < N; ++c) ok &= isfinite(Elem<DT>::to_f(x[c]));
        return ok;
    };
    if (__all_sync(~0u, finite(out))) return;
    const int32_t* row = p.block_table + b * p.table_stride;
    const T* kp = static_cast<const T*>(p.k_pool) + h * p.kp_sh + lane * N;
    const T* vp = static_cast<const T*>(p.v_pool) + h * p.vp_sh + lane * N;
    const int in_page = (1 << p.page_log2) - 1;
    bool bad = false;
    for (int j = lo; j < hi; ++j) {
        if (j >= kmin && j < kend) {
            j = kend - 1;
            continue;
        }
        const int64_t id = row[j >> p.page_log2];
        if (id >= 0 && id < p.n_pages) bad |= !finite(vp + id * p.vp_sp + (j & in_page) * p.vp_st);
    }
    if (!__any_sync(~0u, bad)) return;
    const T* qp = static_cast<const T*>(p.q) + t * p.q_st + (int64_t)hq * p.q_sh + lane * N;
    float m = -INFINITY, l = 0.f, acc[N], q[N];
    uint32_t open = 0;                                     // channels not finite, no such V seen yet
#pragma unroll
    for (int c = 0; c < N; ++c) {
        acc[c] = 0.f, q[c] = Elem<DT>::to_f(qp[c]);
        if (!isfinite(Elem<DT>::to_f(out[c]))) open |= 1u << c;
    }
    for (int j = kend - 1; j >= kmin; --j) {
        const int64_t id = row[j >> p.page_log2];
        const bool in = id >= 0 && id < p.n_pages;         // beyond the pool: zeros
        float s = 0.f, v[N];
#pragma unroll
        for (int c = 0; c < N; ++c) {
            s += in ? q[c] * Elem<DT>::to_f(kp[id * p.kp_sp + (j & in_page) * p.kp_st + c]) : 0.f;
            v[c] = in ? Elem<DT>::to_f(vp[id * p.vp_sp + (j & in_page) * p.vp_st + c]) : 0.f;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        s *= p.scale_log2;
#pragma unroll
        for (int c = 0; c < N; ++c)
            if (!isfinite(v[c])) open &= ~(1u << c);
        if (s != s || !__any_sync(~0u, open != 0)) return;
        const float mn = fmaxf(m, s), off = mn == -INFINITY ? 0.f : mn;
        const float a = ex2(m - off), w = ex2(s - off);
        m = mn;
        l = l * a + w;
#pragma unroll
        for (int c = 0; c < N; ++c) acc[c] = acc[c] * a + w * v[c];
    }
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
#pragma unroll
    for (int c = 0; c < N; ++c) acc[c] *= inv;
    uint32_t y[N / 2];
    pack_results<DT>(acc, y);
#pragma unroll
    for (int c = 0; c < N / 2; ++c) reinterpret_cast<uint32_t*>(out)[c] = y[c];
}
// The rows q0, q0 + step, ... below end of a tile
template <int DT, int D>
__device__ __forceinline__ void mend_tile(const ChunkParams& p, const Seg& s, int q0, int step, int end) {
    for (int q = q0; q < end; q += step) {
        const int pos = s.pos + q / p.g;
        const int kend = p.causal ? min(max(pos + 1, 0), s.kv) : s.kv;
        const int kmin = p.window > 0 ? min(max(pos - p.window + 1, 0), kend) : 0;
        mend_row<DT, D>(p, s.b, s.h, s.h * p.g + q % p.g, (int64_t)s.tok + q / p.g, kmin, kend, s.lo_blk * kBlk,
                        min(s.hi_blk * kBlk, s.kv));
    }
}

// The rows of the tile begun in CTA c that this block has joined, `rows` at a time,
// and the tiles that the CTA wrote itself, their rows over the blocks of a column
// of the grid
template <int DT, int D>
__device__ __forceinline__ void mend(const ChunkParams& p, int c, int rows) {
    const int warps = blockDim.x / 32, warp = threadIdx.x / 32;
    const int4 rec = p.rec[c * 2], more = p.rec[c * 2 + 1];
    Seg s;
    if (rec.y > rec.x) {
        const Req r = load_req(p, more.z);
        s.n = rec.z, s.tok = rec.w, s.b = more.z, s.h = more.x, s.kv = r.kv;
        s.pos = r.off + s.tok - r.q0;
        const Tile tile(p, s.pos, s.n, r.kv);
        s.lo_blk = tile.lo_blk, s.hi_blk = tile.hi_blk;
        const int end = s.n * p.g;
        for (int q = blockIdx.y * rows; q < end; q += gridDim.y * rows)
            mend_tile<DT, D>(p, s, q + warp, warps, min(q + rows, end));
    }
    if (!more.y) return;
    Walk walk = p.walks[c];
    while (walk.next(p, s))
        if (s.k0 == s.lo_blk && s.k1 == s.hi_blk && s.k1 > s.k0)
            mend_tile<DT, D>(p, s, blockIdx.y * warps + warp, gridDim.y * warps, s.n * p.g);
}

// Joins the parts of the tiles that cross a cut, in the order of the cuts.  A
// block per CTA of the first kernel and slice of rows; a thread per row and
// sixteen channels (four loads a part in flight, 32 bytes stored), rows
// fastest, so that a warp reads neighbouring rows.
// Mending is inlined and capped at three blocks per SM (80 registers): when it
// was added, 16 decodes went from 74.0 to 75.6 us; as calls, which need a stack,
// to 76.3, without the cap to 77.3.  A second loop for few rows, with less per
// thread and more parts in flight, costs more in cold instructions than it
// saves (75.6 against 74.4).
constexpr int kJoinThreads = 256;

template <int DT, int D>
__global__ void __launch_bounds__(kJoinThreads, 3) chunk_join_kernel(const __grid_constant__ ChunkParams p) {
    constexpr int kRows = kJoinThreads / (D / 16);
    // Rows past the last request, which no tile has: by blocks of their own, which wait for nothing (as a part of
    // every block 16 decodes took 1.5 us longer).
    if (p.fill_rest && blockIdx.x == gridDim.x - 1) {
        for (int t = min(max(p.cu_q[p.R], 0), p.T) + blockIdx.y; t < p.T; t += gridDim.y) {
            auto* row = static_cast<typename Elem<DT>::T*>(p.out) + (int64_t)t * p.o_st;
            if (p.fill_rest & 1)
                for (int i = threadIdx.x; i < p.Hq * (D / 8); i += kJoinThreads)
                    *reinterpret_cast<uint4*>(row + (int64_t)(i / (D / 8)) * p.o_sh + i % (D / 8) * 8) =
                        make_uint4(0u, 0u, 0u, 0u);
            if ((p.fill_rest & 2) && p.lse)
                for (int i = threadIdx.x; i < p.Hq; i += kJoinThreads) p.lse[(int64_t)t * p.Hq + i] = -INFINITY;
        }
        return;
    }
    griddep_wait();
    const int c = blockIdx.x;
    const int4 rec = p.rec[c * 2], more = p.rec[c * 2 + 1];
    const int from = rec.x, to = rec.y;
    if (to <= from && !more.y) return;
    const int h = more.x, c4 = threadIdx.x / kRows * 4;
    bool bad = false;
    const int rows = to > from ? rec.z * p.g : 0;          // half tiles at rows 0 and 128 of the parts
    for (int q = blockIdx.y * kRows + threadIdx.x % kRows; q < rows; q += gridDim.y * kRows) {
        const int row = q < p.tq * p.g ? q : 128 + q - p.tq * p.g;
        float m = -INFINITY, l = 0.f;
        float4 acc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int e = from; e <= to; ++e) {
            const int slot = e == c ? e * 2 + 1 : e * 2;
            const float2 ml = p.part_ml[slot * 256 + row];
            float4 v[4];
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                const float4* src = p.part_o + (((int64_t)slot * (D / 8) + (c4 + j) / 2) * 256 + row) * 2;
                asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                             : "=f"(v[j].x), "=f"(v[j].y), "=f"(v[j].z), "=f"(v[j].w), "=f"(v[j + 1].x),
                               "=f"(v[j + 1].y), "=f"(v[j + 1].z), "=f"(v[j + 1].w)
                             : "l"(src));
            }
            const float mn = fmaxf(m, ml.x);
            const float a = m == mn ? 1.f : ex2(m - mn), b = ml.x == -INFINITY ? 0.f : ex2(ml.x - mn);
            m = mn;
            l = l * a + ml.y * b;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[j].x = acc[j].x * a + v[j].x * b;
                acc[j].y = acc[j].y * a + v[j].y * b;
                acc[j].z = acc[j].z * a + v[j].z * b;
                acc[j].w = acc[j].w * a + v[j].w * b;
            }
        }
        const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
        const int64_t t = (int64_t)rec.w + q / p.g;
        const int hq = h * p.g + q % p.g;
        uint32_t y[8];
        float f[16];
        float zero = 0.f;                                  // NaN if an output is not finite
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[4 * j] = acc[j].x * inv, f[4 * j + 1] = acc[j].y * inv;
            f[4 * j + 2] = acc[j].z * inv, f[4 * j + 3] = acc[j].w * inv;
            zero = fmaf(acc[j].x, 0.f, fmaf(acc[j].y, 0.f, fmaf(acc[j].z, 0.f, fmaf(acc[j].w, 0.f, zero))));
        }
        pack_results<DT>(f, y);
        bad |= !(zero == 0.f);
        st_row32(static_cast<typename Elem<DT>::T*>(p.out) + t * p.o_st + (int64_t)hq * p.o_sh + c4 * 4, y, 0, p.out32);
        if (p.lse && c4 == 0) p.lse[t * p.Hq + hq] = l == 0.f ? -INFINITY : 0.69314718056f * (m + __log2f(l));
    }
    if (__syncthreads_or(bad || more.y)) mend<DT, D>(p, c, kRows);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static std::atomic<int64_t> g_wait_polls{kCaPolls};

static PFN_cuTensorMapEncodeTiled_v12000 ca_encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

static int check_desc(const fade_chunk_desc* d) {
    if (!d || d->R < 0 || d->T < 0 || d->Hq < 1 || d->Hkv < 1 || d->Hq % d->Hkv || d->table_width < 0 ||
        d->n_pages < 0 || d->window < 0 || !(d->sm_scale >= 1e-45) ||   // times log2(e) an fp32 number that is not 0
        !(d->sm_scale <= 1e30))
        return FADE_ERR_INVALID_ARG;
    if (d->dtype != FADE_F16 && d->dtype != FADE_BF16) return FADE_ERR_UNSUPPORTED;
    if ((d->D != 64 && d->D != 128) || d->Hq / d->Hkv > 128) return FADE_ERR_UNSUPPORTED;
    if (d->page_size != 16 && d->page_size != 32 && d->page_size != 64 && d->page_size != 128)
        return FADE_ERR_UNSUPPORTED;
    // 32-bit positions: sums of two lengths stay below 2^31
    const int64_t most = 1LL << 29;
    if (d->R > most || d->T > most || d->Hq > (1 << 20) || d->n_pages > INT32_MAX - 1 ||
        d->table_width > most / d->page_size)
        return FADE_ERR_UNSUPPORTED;
    return FADE_OK;
}

// [T, Hq, D] or [pages, heads, tokens, D] in 64-channel boxes, 128-byte swizzle
static int make_map(CUtensorMap* m, int dtype, const void* base, int rank, const cuuint64_t* dims,
                    const int64_t* strides, const cuuint32_t* box) {
    auto enc = ca_encode_fn();
    if (!enc) return FADE_ERR_CUDA;
    cuuint64_t bytes[3];
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    for (int i = 0; i < rank - 1; ++i) {
        if (strides[i] < 0) return FADE_ERR_INVALID_ARG;
        bytes[i] = (cuuint64_t)strides[i] * 2;
    }
    const bool ok = encoded([&] {
        return enc(m, dtype == FADE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                   const_cast<void*>(base), dims, bytes, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
    return ok ? FADE_OK : FADE_ERR_ALIGN;
}

constexpr int kWalkBytes = 128;   // of a CTA in the workspace
static_assert(sizeof(Walk) <= kWalkBytes);
static size_t ws_bytes_for(int G, int64_t D) {
    return 256 + (size_t)G * (32 + kWalkBytes) + (size_t)G * 2 * 256 * 8 + (size_t)G * 2 * 256 * D * 4;
}

template <int DT, int D>
static int launch_chunk(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const ChunkParams& p, int G,
                        cudaStream_t st) {
    auto k = chunk_attn_kernel<DT, D>;
    static std::atomic<uint64_t> ready{0};   // devices whose kernel has its shared memory granted
    int dev = 0;
    FADE_CUDA_TRY(cudaGetDevice(&dev));
    if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
        FADE_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, CaLayout<D>::BYTES));
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    k<<<G, kCaThreads, CaLayout<D>::BYTES, st>>>(tq, tk, tv, p);
    FADE_LAUNCH_CHECK();
    // Blocks for the rows that a tile can have, eight slices at most: they start as the first kernel's CTAs, which
    // leave no registers beside them, end, and more would queue.  One column more for the rows past the last request.
    const int64_t rows = std::min<int64_t>(256, (int64_t)p.T * p.g);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(G + (p.fill_rest ? 1 : 0),
                       (unsigned)std::min<int64_t>(8, (rows * (D / 16) + kJoinThreads - 1) / kJoinThreads));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    FADE_CUDA_TRY(cudaLaunchKernelEx(&cfg, chunk_join_kernel<DT, D>, p));
    return FADE_OK;
}

}  // namespace fade

using namespace fade;

extern "C" size_t fade_chunk_attn_workspace_size(const fade_chunk_desc* d) {
    if (check_desc(d) != FADE_OK) return 0;
    const int G = fade_sm_count();
    return ws_bytes_for(G > 0 ? G : 148, d->D);
}

extern "C" int fade_chunk_attn(const fade_chunk_desc* desc, void* workspace, size_t ws_bytes, void* stream) {
    const int bad = check_desc(desc);
    if (bad != FADE_OK) return bad;
    // the stride of a dimension of one is never stepped and may be anything: dense ones in their place
    fade_chunk_desc dense = *desc;
    const fade_chunk_desc* d = &dense;
    if (d->Hq == 1) dense.q_sh = dense.o_sh = d->D;
    if (d->T == 1) dense.q_st = dense.o_st = d->Hq * d->D;
    if (d->Hkv == 1) dense.kp_sh = dense.vp_sh = d->page_size * d->D;
    if (d->n_pages <= 1) dense.kp_sp = dense.vp_sp = d->Hkv * d->page_size * d->D;
    if (d->T == 0 || d->R == 0) return FADE_OK;
    if (!d->q || !d->out || !d->cu_q || !d->kv_lens || (d->table_width > 0 && !d->block_table) ||
        (d->n_pages > 0 && (!d->k_pool || !d->v_pool)))
        return FADE_ERR_INVALID_ARG;
    const int64_t strides[] = {d->q_st, d->q_sh, d->o_st, d->o_sh, d->kp_sp, d->kp_sh, d->kp_st, d->vp_sp, d->vp_sh, d->vp_st};
    for (int64_t s : strides)
        if (s % 8) return FADE_ERR_ALIGN;
    if (!aligned16(d->q) || !aligned16(d->out) || !aligned16(d->k_pool) || !aligned16(d->v_pool)) return FADE_ERR_ALIGN;
    if (!workspace || ws_bytes < fade_chunk_attn_workspace_size(d)) return FADE_ERR_WORKSPACE;
    if (views_overlap(d->q, d->q_st, d->q_sh, d->out, d->o_st, d->o_sh, d->T, d->Hq, d->D, 2)) return FADE_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(workspace) % 32) return FADE_ERR_ALIGN;   // 32-byte loads and stores of the parts
    const int G = fade_sm_count();
    if (G <= 0) return FADE_ERR_CUDA;
    ChunkParams p = {};
    p.block_table = d->block_table;
    p.cu_q = d->cu_q;
    p.kv_lens = d->kv_lens;
    p.out = d->out;
    p.lse = d->lse;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.err = reinterpret_cast<int*>(ws);
    p.rec = reinterpret_cast<int4*>(ws + 256);
    p.walks = reinterpret_cast<Walk*>(ws + 256 + (size_t)G * 32);
    p.part_ml = reinterpret_cast<float2*>(ws + 256 + (size_t)G * (32 + kWalkBytes));
    p.part_o = reinterpret_cast<float4*>(ws + 256 + (size_t)G * (32 + kWalkBytes) + (size_t)G * 2 * 256 * 8);
    p.table_stride = d->table_stride;
    p.o_st = d->o_st;
    p.o_sh = d->o_sh;
    p.q = d->q;
    p.q_st = d->q_st;
    p.q_sh = d->q_sh;
    p.k_pool = d->k_pool;
    p.kp_sp = d->kp_sp;
    p.kp_sh = d->kp_sh;
    p.kp_st = d->kp_st;
    p.v_pool = d->v_pool;
    p.vp_sp = d->vp_sp;
    p.vp_sh = d->vp_sh;
    p.vp_st = d->vp_st;
    p.R = (int)d->R;
    p.T = (int)d->T;
    p.Hq = (int)d->Hq;
    p.Hkv = (int)d->Hkv;
    p.g = p.Hq / p.Hkv;
    p.tq = kHalf / p.g;
    // floor(x / t) = floor(x m / 2^(31 + s)) for x < 2^31 with s = ceil(log2 t), m = floor(2^(31 + s) / t) + 1
    const uint32_t tile = 2 * p.tq;
    int up = 0;
    while ((1u << up) < tile) ++up;
    p.tile_magic = (uint32_t)(((uint64_t)1 << (31 + up)) / tile + 1);
    p.tile_shift = up - 1;
    while ((1 << p.page_log2) < d->page_size) ++p.page_log2;
    p.n_pages = (int)d->n_pages;
    p.table_width = d->n_pages > 0 ? (int)d->table_width : 0;
    p.causal = d->causal != 0;
    p.fill_rest = (int)(d->fill_rest & 3);
    p.window = d->window >= (1LL << 29) ? 0 : (int)d->window;   // as long as the longest cache: hides nothing
    p.out32 = reinterpret_cast<uintptr_t>(d->out) % 32 == 0 && d->o_st % 16 == 0 && d->o_sh % 16 == 0;
    p.scale_log2 = (float)(d->sm_scale * 1.4426950408889634);
    p.lazy = std::min(kLazyMax / p.scale_log2, 1e30f);   // finite: the first maximum always replaces -inf
    p.polls = (uint32_t)g_wait_polls.load(std::memory_order_relaxed);
    CUtensorMap tq, tk, tv;
    const cuuint64_t qd[3] = {(cuuint64_t)d->D, (cuuint64_t)d->Hq, (cuuint64_t)d->T};
    const int64_t qs[2] = {d->q_sh, d->q_st};
    const cuuint32_t qb[3] = {64, (cuuint32_t)p.g, (cuuint32_t)p.tq};
    int st = make_map(&tq, (int)d->dtype, d->q, 3, qd, qs, qb);
    if (st != FADE_OK) return st;
    // without a pool every table entry lies beyond it; the maps then describe q's memory and read nothing
    const void* kb = d->n_pages > 0 ? d->k_pool : d->q;
    const void* vb = d->n_pages > 0 ? d->v_pool : d->q;
    const cuuint64_t kd[4] = {(cuuint64_t)d->D, (cuuint64_t)d->page_size, (cuuint64_t)d->Hkv,
                              (cuuint64_t)(d->n_pages > 0 ? d->n_pages : 1)};
    const int64_t ks[3] = {d->kp_st, d->kp_sh, d->kp_sp}, vs[3] = {d->vp_st, d->vp_sh, d->vp_sp};
    const cuuint32_t kbox[4] = {64, (cuuint32_t)d->page_size, 1, 1};
    if ((st = make_map(&tk, (int)d->dtype, kb, 4, kd, ks, kbox)) != FADE_OK) return st;
    if ((st = make_map(&tv, (int)d->dtype, vb, 4, kd, vs, kbox)) != FADE_OK) return st;
    cudaStream_t s = as_stream(stream);
    std::lock_guard<std::mutex> lock(workspace_mutex(workspace));
    if (d->dtype == FADE_F16)
        return d->D == 64 ? launch_chunk<FADE_F16, 64>(tq, tk, tv, p, G, s)
                          : launch_chunk<FADE_F16, 128>(tq, tk, tv, p, G, s);
    return d->D == 64 ? launch_chunk<FADE_BF16, 64>(tq, tk, tv, p, G, s)
                      : launch_chunk<FADE_BF16, 128>(tq, tk, tv, p, G, s);
}

extern "C" int fade_chunk_attn_check(void* stream) {
    void* word = nullptr;
    FADE_CUDA_TRY(cudaGetSymbolAddress(&word, g_gave_up));
    int h = 0;
    cudaStream_t s = as_stream(stream);
    FADE_CUDA_TRY(cudaMemcpyAsync(&h, word, sizeof(int), cudaMemcpyDeviceToHost, s));
    FADE_CUDA_TRY(cudaStreamSynchronize(s));
    if (h == 0) return FADE_OK;
    FADE_CUDA_TRY(cudaMemsetAsync(word, 0, sizeof(int), s));
    FADE_CUDA_TRY(cudaStreamSynchronize(s));
    return FADE_ERR_TIMEOUT;
}

extern "C" int fade_set_wait_polls(int64_t polls) {
    if (polls > kCaPolls) return FADE_ERR_INVALID_ARG;
    g_wait_polls.store(polls < 0 ? kCaPolls : polls, std::memory_order_relaxed);
    return FADE_OK;
}
