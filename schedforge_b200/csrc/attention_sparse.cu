// Decode attention over selected blocks of a paged cache.
//
// For each block of the cache and each key element the smallest and largest value are kept beside the pool
// (sfb_k_paged_kv_bounds).  sum_d max(q_d low_d, q_d high_d) then bounds every logit of the block from above at a
// sixteenth of the keys' bytes (16-token blocks), and the blocks with the largest bounds are attended to.
// Three steps: scores (memory-bound on the bounds), selection (one CTA per (sequence, K/V head)), attention over the
// list (step_attention).  Ranks follow from the scores, so they count in 64 bits, where a different order of summation
// cannot swap two blocks that are not equal for all purposes.  64-bit arithmetic for all blocks would take longer than
// their bytes (two products an element and head: 537 million at eight sequences of 128 thousand tokens), so the pass
// over all blocks sums in 32 bits, and only blocks whose rank those sums leave open are scored again.
#include <algorithm>

#include "cache_ops.cuh"
#include "mma_sync.cuh"
#include "ptx_sm100.cuh"
#include "select.cuh"

namespace sfb {
namespace {

__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
}
__device__ __forceinline__ void load4(const bf16* p, float (&v)[4]) {
    const uint2 f = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(f.x << 16); v[1] = __uint_as_float(f.x & 0xffff0000u);
    v[2] = __uint_as_float(f.y << 16); v[3] = __uint_as_float(f.y & 0xffff0000u);
}

template <class T>
__global__ void __launch_bounds__(128)
bounds_kernel(const __grid_constant__ PagedView kv, const int* __restrict__ start_len, T* __restrict__ bounds, int vec) {
    const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    const int end = kv.length(b), start = max(0, start_len[b]);
    if (start >= end) return;
    const int last = kv.block_of(end - 1);
    for (int block = kv.block_of(start) + blockIdx.x * 4 + warp; block <= last; block += gridDim.x * 4) {
        const int64_t row = kv.row(b, kvh, block * kv.block_tokens);
        if (row < 0) continue;
        const int live = min(kv.block_tokens, end - block * kv.block_tokens);
        const T* keys = static_cast<const T*>(kv.k_pool) + row * kv.dim;
        T* dst = bounds + row / kv.block_tokens * 2 * kv.dim;
        if (vec) {   // four elements a lane, every token's load in flight
            for (int d = lane * 4; d < kv.dim; d += 128) {
                float lo[4] = {INFINITY, INFINITY, INFINITY, INFINITY}, hi[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 16
                for (int t = 0; t < live; ++t) {
                    float v[4];
                    load4(keys + static_cast<int64_t>(t) * kv.dim + d, v);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { lo[e] = fminf(lo[e], v[e]); hi[e] = fmaxf(hi[e], v[e]); }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    dst[d + e] = from_float<T>(lo[e]);
                    dst[kv.dim + d + e] = from_float<T>(hi[e]);
                }
            }
            continue;
        }
        for (int d = lane; d < kv.dim; d += 32) {
            float lo = INFINITY, hi = -INFINITY;
#pragma unroll 8
            for (int t = 0; t < live; ++t) {
                const float v = to_float(keys[static_cast<int64_t>(t) * kv.dim + d]);
                lo = fminf(lo, v);
                hi = fmaxf(hi, v);
            }
            dst[d] = from_float<T>(lo);
            dst[kv.dim + d] = from_float<T>(hi);
        }
    }
}

struct ScoreParams {
    PagedView kv;
    const void *q, *bounds;
    float* scores;        // [batch * kv_heads][score_stride], summed in 32 bits
    float* sizes;         // [batch * kv_heads][gridDim.x]: the largest |bound| among the blocks of a CTA
    int q_heads, score_stride, batch_blocks, cta_blocks, heads;   // heads: K/V heads a CTA takes
};

// Any layout: one warp per block, lane owns every 32nd element.
template <class T>
__global__ void __launch_bounds__(128)
score_kernel(const __grid_constant__ ScoreParams p) {
    __shared__ float size_of[4];
    const PagedView& kv = p.kv;
    const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    const int ctx = kv.length(b);
    const int blocks = ctx > 0 ? kv.block_of(ctx - 1) + 1 : 0;
    const int group = p.q_heads / kv.kv_heads;
    const T* q = static_cast<const T*>(p.q) + (static_cast<size_t>(b) * p.q_heads + kvh * group) * kv.dim;
    const size_t row = static_cast<size_t>(b) * kv.kv_heads + kvh;
    float size = 0.0F;
    for (int block = blockIdx.x * 16 + warp; block < min(blocks, (static_cast<int>(blockIdx.x) + 1) * 16); block += 4) {
        const int page = kv.table[static_cast<size_t>(b) * kv.max_blocks + block];
        float best = __uint_as_float(0x7fc00000u);  // NaN: ranks last
        if (page >= 0 && page < kv.num_blocks) {
            const T* lo = static_cast<const T*>(p.bounds) + (static_cast<int64_t>(page) * kv.kv_heads + kvh) * 2 * kv.dim;
            const T* hi = lo + kv.dim;
            for (int g = 0; g < group; ++g) {
                float s = 0.0F;
                for (int d = lane; d < kv.dim; d += 32) {
                    const float qv = to_float(q[g * kv.dim + d]), l = to_float(lo[d]), h = to_float(hi[d]);
                    s = fmaf(qv, qv > 0.0F ? h : l, s);
                    size = fmaxf(size, fmaxf(fabsf(l), fabsf(h)));
                }
                s = warp_sum(s);
                best = fmaxf(best, s);  // (fmaxf ignores NaN)
            }
        } else if (lane == 0) {
            atomicOr(kv.status, kCodeDecodeBounds);
        }
        if (lane == 0) p.scores[row * p.score_stride + block] = best;
    }
    size = warp_max(size);
    if (lane == 0) size_of[warp] = size;
    __syncthreads();
    if (threadIdx.x == 0)
        p.sizes[row * gridDim.x + blockIdx.x] = fmaxf(fmaxf(size_of[0], size_of[1]), fmaxf(size_of[2], size_of[3]));
}

// Sums of N values over LPR lanes: every step halves the values a lane still carries as long as there are several, so
// that N values cost N - 1 exchanges instead of N log2(LPR).  Lane `sub` ends with the values of index
// sub * N / LPR ... (all lanes of a run of LPR / N with the same one where N < LPR).
template <int N, int LPR>
__device__ __forceinline__ void spread_sums(float (&v)[N], int sub) {
    int n = N;
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) {
        if (n > 1) {
            n >>= 1;
            const bool upper = (sub & o) != 0;
#pragma unroll
            for (int i = 0; i < N / 2; ++i)
                if (i < n) {
                    const float keep = upper ? v[i + n] : v[i], send = upper ? v[i] : v[i + n];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
                }
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
        }
    }
}

// dim % 8 == 0 and 16-byte aligned rows.  Each of a CTA's four warps works on its own through the blocks of the CTA's
// range: batches of about 8 KB of bounds come into its part of shared memory by bulk copies (one per block: low and
// high are contiguous), three batches in flight, so 96 KB per CTA and two CTAs per SM whatever the warps do.
// LPR lanes share a block, eight elements each, 32 / LPR blocks at once and four times over.  With q+ = max(q, 0) and
// q- = min(q, 0) the bound is q+ . high + q- . low: two fused multiply-adds an element and no selection.
constexpr int kScoreRows = 4, kScoreStages = 3, kScoreWarps = 4, kScoreBatchBytes = 8192;
constexpr uint32_t kCodeScore = 0x20;

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <class T, int LPR, int GC>
__global__ void __launch_bounds__(kScoreWarps * 32)
score_vec_kernel(const __grid_constant__ ScoreParams p) {
    constexpr int RPW = 32 / LPR, N = kScoreRows * GC, kPass = RPW * kScoreRows;   // blocks a warp scores at once
    constexpr int kLeft = N > LPR ? N / LPR : 1;        // values a lane ends with
    extern __shared__ __align__(16) uint8_t score_smem[];   // [warps][stages][batch][2 * dim]
    __shared__ uint64_t bars[kScoreWarps][kScoreStages];
    __shared__ uint32_t abort_word;
    __shared__ float size_of[kScoreWarps];
    const PagedView& kv = p.kv;
    const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LPR, rg = lane / LPR;
    const int group = p.q_heads / kv.kv_heads, batch = p.batch_blocks;
    const uint32_t block_bytes = static_cast<uint32_t>(2 * kv.dim * sizeof(T));
    if (lane == 0) {
        for (int s = 0; s < kScoreStages; ++s) ptx::mbar_init(ptx::smem_u32(&bars[warp][s]), 1);
        if (warp == 0) abort_word = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async();
    }
    grid_dependency_wait();
    __syncthreads();
    const int ctx = kv.length(b);
    const int blocks = ctx > 0 ? kv.block_of(ctx - 1) + 1 : 0;
    const size_t row = static_cast<size_t>(b) * kv.kv_heads + kvh;
    const int last = min(blocks, (static_cast<int>(blockIdx.x) + 1) * p.cta_blocks);
    const int begin = blockIdx.x * p.cta_blocks + warp * batch;      // batches go round the warps
    const int step = kScoreWarps * batch;
    const int* table = kv.table + static_cast<size_t>(b) * kv.max_blocks;
    uint8_t* mine = score_smem + static_cast<size_t>(warp) * kScoreStages * batch * block_bytes;
    const bool inside = sub * 8 < kv.dim;

    // lane i brings block i of a batch (batch <= 32); -1: no such block in the pool
    const auto page_of = [&](int base) -> int {
        const int block = base + lane;
        if (lane >= batch || block >= last) return -2;
        const int page = table[block];
        if (page >= 0 && page < kv.num_blocks) return page;
        atomicOr(kv.status, kCodeDecodeBounds);
        return -1;
    };
    const auto issue = [&](int stage, int page) {
        const uint32_t bar = ptx::smem_u32(&bars[warp][stage]);
        const int n = __popc(__ballot_sync(0xffffffffu, page >= 0));
        if (lane == 0) ptx::mbar_expect_tx(bar, n * block_bytes);
        __syncwarp();
        if (page >= 0)
            bulk_load(ptx::smem_u32(mine + (static_cast<size_t>(stage) * batch + lane) * block_bytes),
                      static_cast<const T*>(p.bounds) + (static_cast<int64_t>(page) * kv.kv_heads + kvh) * 2 * kv.dim, block_bytes, bar);
    };
    unsigned there[kScoreStages];       // lanes whose block exists, per stage
#pragma unroll
    for (int s = 0; s < kScoreStages; ++s) {
        const int page = begin + s * step < last ? page_of(begin + s * step) : -2;
        there[s] = __ballot_sync(0xffffffffu, page >= 0);
        if (begin + s * step < last) issue(s, page);
    }
    float pos[GC][8], neg[GC][8], size = 0.0F;
    const auto load_heads = [&](int g0) {
#pragma unroll
        for (int g = 0; g < GC; ++g) {
            Raw8<T> raw;   // (heads past the group repeat its last: the largest score does not change)
            if (inside) raw.load(static_cast<const T*>(p.q) + (static_cast<size_t>(b) * p.q_heads + kvh * group + min(g0 + g, group - 1)) * kv.dim + sub * 8);
            else raw.zero();
            raw.get(pos[g]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                neg[g][e] = fminf(pos[g][e], 0.0F);
                pos[g][e] = fmaxf(pos[g][e], 0.0F);
            }
        }
    };
    load_heads(0);
    int stage = 0, phase = 0;
    for (int base = begin; base < last; base += step) {
        const int ahead = base + kScoreStages * step;
        const int next_page = ahead < last ? page_of(ahead) : -2;     // in flight while this batch is scored
        if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bars[warp][stage]), phase, &abort_word, kv.status, kCodeScore))) break;
        unsigned present = 0;
#pragma unroll
        for (int s = 0; s < kScoreStages; ++s)
            if (s == stage) present = there[s];
        const uint8_t* rows = mine + static_cast<size_t>(stage) * batch * block_bytes;
        for (int pass = 0; pass < batch && base + pass < last; pass += kPass) {
            float best[kLeft];
#pragma unroll 1
            for (int g0 = 0; g0 < group; g0 += GC) {
                if (group > GC) load_heads(g0);
                float s[N];
#pragma unroll
                for (int u = 0; u < kScoreRows; ++u) {
                    const int i = pass + u * RPW + rg;
                    Raw8<T> lo, hi;
                    if (inside && (present >> i & 1u)) {
                        const T* src = reinterpret_cast<const T*>(rows + static_cast<size_t>(i) * block_bytes) + sub * 8;
                        lo.load(src);
                        hi.load(src + kv.dim);
                    } else {
                        lo.zero();
                        hi.zero();
                    }
                    float l[8], h[8];
                    lo.get(l);
                    hi.get(h);
#pragma unroll
                    for (int e = 0; e < 8; ++e) size = fmaxf(size, fmaxf(fabsf(l[e]), fabsf(h[e])));
#pragma unroll
                    for (int g = 0; g < GC; ++g) {
                        float a = 0.0F;
#pragma unroll
                        for (int e = 0; e < 8; ++e) a = fmaf(neg[g][e], l[e], fmaf(pos[g][e], h[e], a));
                        s[u * GC + g] = a;
                    }
                }
                spread_sums<N, LPR>(s, sub);
                // index = block * GC + head: the largest over the heads, first among a lane's own values
                float top[kLeft];
                constexpr int kOwn = kLeft < GC ? kLeft : GC;     // heads a lane holds of one block
#pragma unroll
                for (int i = 0; i < kLeft; ++i) {
                    top[i] = s[i];
#pragma unroll
                    for (int k = 1; k < kOwn; ++k) top[i] = fmaxf(top[i], s[i / kOwn * kOwn + (i + k) % kOwn]);
                }
                constexpr int kFirst = N < LPR ? LPR / N : 1;     // lane distance of two heads
#pragma unroll
                for (int o = kFirst; o < kFirst * (GC / kOwn); o <<= 1)
#pragma unroll
                    for (int i = 0; i < kLeft; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
                for (int i = 0; i < kLeft; ++i) best[i] = g0 == 0 ? top[i] : fmaxf(best[i], top[i]);
            }
            // the first lane (and value) of every block writes its score
#pragma unroll
            for (int i = 0; i < kLeft; ++i) {
                const int index = N >= LPR ? sub * kLeft + i : sub / (LPR / N);
                const bool first = index % GC == 0 && (N >= LPR || sub % (LPR / N) == 0);
                const int at = pass + index / GC * RPW + rg;
                if (first && at < batch && base + at < last)
                    p.scores[row * p.score_stride + base + at] = present >> at & 1u ? best[i] : __uint_as_float(0x7fc00000u);
            }
        }
        __syncwarp();
        if (ahead < last) {
            const unsigned now = __ballot_sync(0xffffffffu, next_page >= 0);
#pragma unroll
            for (int s = 0; s < kScoreStages; ++s)
                if (s == stage) there[s] = now;
            issue(stage, next_page);
        }
        if (++stage == kScoreStages) { stage = 0; phase ^= 1; }
    }
    size = warp_max(size);
    if (lane == 0) size_of[warp] = size;
    __syncthreads();
    if (abort_word)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);  // let copies in flight land before the CTA exits
    if (threadIdx.x == 0)
        p.sizes[row * gridDim.x + blockIdx.x] = fmaxf(fmaxf(size_of[0], size_of[1]), fmaxf(size_of[2], size_of[3]));
}

// bf16, dim % 16 == 0: the products on the tensor path.  16 blocks are the rows of A (low and high side by side are
// 2 dim columns), q- and q+ of up to eight heads the columns of B: 2 dim / 16 instructions replace 4 dim multiply-adds a
// block and head.  A CTA takes `heads` K/V heads of a sequence at once (all of them up to eight): their bounds lie side by
// side, so a block is one copy of heads * 4 dim bytes (4 KB at eight heads of 128; copies of one head's 512 bytes ran at
// 3.8 TB/s).  A copy warp keeps three stages of 16 * (warps / heads) blocks in flight; each of the other warps takes one head
// of 16 blocks of every stage.  Rows are 16 bytes further apart than their length, so that ldmatrix meets no bank twice.
template <int KS>   // steps of 16 columns in one half: dim / 16
struct ScoreMma {
    static constexpr int D = KS * 16;
    static constexpr int kWarps = KS <= 8 ? 8 : 4;       // that compute
    static constexpr int kMaxBlocks = kWarps * 16;       // per stage
};

template <int KS>
__global__ void __launch_bounds__((ScoreMma<KS>::kWarps + 1) * 32)
score_mma_kernel(const __grid_constant__ ScoreParams p) {
    using Sh = ScoreMma<KS>;
    constexpr int D = Sh::D, kWarps = Sh::kWarps, kWords = (Sh::kMaxBlocks + 31) / 32;
    extern __shared__ __align__(16) uint8_t score_smem[];   // [stages][stage blocks][heads * 4 D + 16]
    __shared__ uint64_t full_bar[kScoreStages], empty_bar[kScoreStages];
    __shared__ unsigned there[kScoreStages][kWords];        // blocks of the stage that exist
    __shared__ uint32_t abort_word;
    __shared__ float size_of[kWarps];
    const PagedView& kv = p.kv;
    const int heads = p.heads, subs = kWarps / heads, stage_blocks = subs * 16;
    const uint32_t copy_bytes = heads * 4 * D, row_bytes = copy_bytes + 16;
    const int b = blockIdx.z, head0 = blockIdx.y * heads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3;
    const int group = p.q_heads / kv.kv_heads;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kScoreStages; ++s) {
            ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), heads * subs);
        }
        abort_word = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async();
    }
    grid_dependency_wait();
    __syncthreads();
    const int ctx = kv.length(b);
    const int blocks = ctx > 0 ? kv.block_of(ctx - 1) + 1 : 0;
    const int begin = blockIdx.x * p.cta_blocks, last = min(blocks, begin + p.cta_blocks);
    float size = 0.0F;
    if (warp == kWarps) {
        // ---------------------------------------------------------------- copies: lane i brings blocks i, i + 32, ...
        const int* table = kv.table + static_cast<size_t>(b) * kv.max_blocks;
        int next[kWords];
        const auto fetch = [&](int base) {
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                const int at = lane + 32 * j;
                next[j] = -2;
                if (at < stage_blocks && base + at < last) {
                    const int page = table[base + at];
                    next[j] = page >= 0 && page < kv.num_blocks ? page : -1;
                    if (next[j] < 0) atomicOr(kv.status, kCodeDecodeBounds);
                }
            }
        };
        fetch(begin);
        int n = 0;
        for (int base = begin; base < last; base += stage_blocks, ++n) {
            int page[kWords];
            unsigned count = 0, present[kWords];
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                page[j] = next[j];
                present[j] = __ballot_sync(0xffffffffu, page[j] >= 0);
                count += __popc(present[j]);
            }
            fetch(base + stage_blocks);      // in flight while this stage waits
            const int s = n % kScoreStages;
            if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&empty_bar[s]), ((n / kScoreStages) & 1) ^ 1, &abort_word, kv.status, kCodeScore))) break;
            const uint32_t bar = ptx::smem_u32(&full_bar[s]);
            if (lane == 0) {
#pragma unroll
                for (int j = 0; j < kWords; ++j) there[s][j] = present[j];
                ptx::mbar_expect_tx(bar, count * copy_bytes);
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < kWords; ++j)
                if (page[j] >= 0)
                    bulk_load(ptx::smem_u32(score_smem + (static_cast<size_t>(s) * stage_blocks + lane + 32 * j) * row_bytes),
                              static_cast<const bf16*>(p.bounds) + (static_cast<int64_t>(page[j]) * kv.kv_heads + head0) * 2 * D, copy_bytes, bar);
        }
    } else if (warp < heads * subs) {
        const int kvh = head0 + warp % heads, sub = warp / heads;
        const size_t row = static_cast<size_t>(b) * kv.kv_heads + kvh;
        // B fragments: columns are heads, rows k: q- for the low half, q+ for the high half
        uint32_t qb[2 * KS][2];
        const auto load_heads = [&](int g0) {
            const int g = g0 + (lane >> 2);
            const bf16* q = static_cast<const bf16*>(p.q) + (static_cast<size_t>(b) * p.q_heads + kvh * group + min(g, group - 1)) * D;
            const __nv_bfloat162 zero = __floats2bfloat162_rn(0.0F, 0.0F);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(q + 16 * k + 8 * h + 2 * quad);
                    const __nv_bfloat162 neg = __hmin2_nan(v, zero), pos = __hmax2_nan(v, zero);   // (a NaN in q reaches every score)
                    qb[k][h] = *reinterpret_cast<const uint32_t*>(&neg);
                    qb[KS + k][h] = *reinterpret_cast<const uint32_t*>(&pos);
                }
        };
        load_heads(0);
        __nv_bfloat162 most = __floats2bfloat162_rn(0.0F, 0.0F);
        int n = 0;
        for (int base = begin; base < last; base += stage_blocks, ++n) {
            const int s = n % kScoreStages;
            if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&full_bar[s]), (n / kScoreStages) & 1, &abort_word, kv.status, kCodeScore))) break;
            const int first = base + sub * 16;
            if (first < last) {
                const unsigned present = there[s][sub >> 1] >> ((sub & 1) * 16);
                const uint32_t rows = ptx::smem_u32(score_smem) + (s * stage_blocks + sub * 16 + (lane & 15)) * row_bytes +
                                      (warp % heads) * 4 * D + (lane >> 4) * 16;
                float best[2] = {-INFINITY, -INFINITY};   // rows lane / 4 and lane / 4 + 8
#pragma unroll 1
                for (int g0 = 0; g0 < group; g0 += 8) {
                    if (group > 8) load_heads(g0);
                    float c[2][4] = {};   // two chains: even and odd steps
#pragma unroll
                    for (int k = 0; k < 2 * KS; ++k) {
                        uint32_t a[4];
                        ldmatrix_x4(rows + k * 32, a);
                        mma_bf16(c[k & 1], a, qb[k][0], qb[k][1]);
                        if (g0 == 0) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const bool ok = present >> ((lane >> 2) + 8 * (i & 1)) & 1u;   // (a row that was not loaded holds anything)
                                const uint32_t word = ok ? a[i] & 0x7fff7fffu : 0u;
                                most = __hmax2(most, *reinterpret_cast<const __nv_bfloat162*>(&word));
                            }
                        }
                    }
                    // columns 2 quad and 2 quad + 1 of the heads
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float x = g0 + 2 * quad < group ? c[0][2 * r] + c[1][2 * r] : -INFINITY;
                        const float y = g0 + 2 * quad + 1 < group ? c[0][2 * r + 1] + c[1][2 * r + 1] : -INFINITY;
                        best[r] = fmaxf(best[r], fmaxf(x, y));
                    }
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    best[r] = fmaxf(best[r], __shfl_xor_sync(0xffffffffu, best[r], 1));
                    best[r] = fmaxf(best[r], __shfl_xor_sync(0xffffffffu, best[r], 2));
                    const int at = (lane >> 2) + 8 * r;
                    if (quad == 0 && first + at < last)
                        p.scores[row * p.score_stride + first + at] = present >> at & 1u ? best[r] : __uint_as_float(0x7fc00000u);
                }
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&empty_bar[s]));
        }
        size = warp_max(fmaxf(__low2float(most), __high2float(most)));
    }
    if (warp < kWarps && lane == 0) size_of[warp] = size;
    __syncthreads();
    if (abort_word)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);  // let copies in flight land before the CTA exits
    if (threadIdx.x < heads) {
        float most = 0.0F;
        for (int i = threadIdx.x; i < heads * subs; i += heads) most = fmaxf(most, size_of[i]);
        p.sizes[(static_cast<size_t>(b) * kv.kv_heads + head0 + threadIdx.x) * gridDim.x + blockIdx.x] = most;
    }
}

// How the scores are taken: by which kernel, blocks per batch and per CTA, and the error of a score relative to
// sum |q_d| * largest |bound|.
enum ScoreKind { kScoreAny, kScoreVec, kScoreMma };
struct ScoreShape {
    ScoreKind kind;
    int lanes, batch, cta_blocks, heads;
    float error;
};
ScoreShape score_shape(const sfb_sparse_args& a, int blocks) {
    ScoreShape s{kScoreAny, 0, 0, 16, 1, 9.5367431640625e-7F};   // 2^-20: at most 8 + 5 roundings of 2^-24
    if (!aligned16(a.bounds) || !aligned16(a.q)) return s;
    if (a.dtype == SFB_BF16 && a.head_dim % 16 == 0) {
        s.kind = kScoreMma;
        s.error = 6.103515625e-5F;   // 2^-14: 2 dim <= 512 products, each addition good to 2^-23 at least
        const int warps = a.head_dim <= 128 ? 8 : 4;
        s.heads = a.kv_heads < warps ? a.kv_heads : warps;
        while (a.kv_heads % s.heads != 0) --s.heads;
        s.batch = warps / s.heads * 16;
        // one round of CTAs (two per SM below 128 elements a head) as long as that leaves a stage for each; ranges of at most
        // 2048 blocks even out ragged contexts
        const int64_t slots = (a.head_dim <= 64 ? 2LL : 1LL) * sm_count(), groups = static_cast<int64_t>(a.batch) * (a.kv_heads / s.heads);
        const int64_t each = slots / groups > 0 ? slots / groups : 1;
        int range = ceil_div(blocks, static_cast<int>(each < blocks ? each : blocks));
        if (range > 2048) range = 2048;
        s.cta_blocks = ceil_div(range, s.batch) * s.batch;
        return s;
    } else if (a.dtype == SFB_F32 && a.head_dim % 8 == 0) {
        s.kind = kScoreVec;
        s.lanes = a.head_dim <= 64 ? 8 : a.head_dim <= 128 ? 16 : 32;
        const int pass = 32 / s.lanes * kScoreRows;
        s.batch = kScoreBatchBytes / (2 * a.head_dim * 4);
        if (s.batch > 32) s.batch = 32;
        s.batch = s.batch / pass * pass;
    } else {
        return s;
    }
    // ranges of at least one batch a warp, longer while there are enough of them for four rounds of two CTAs per SM
    const int64_t rows = static_cast<int64_t>(a.batch) * a.kv_heads;
    const int64_t ctas = 8LL * sm_count() / rows > 0 ? 8LL * sm_count() / rows : 1;
    const int round = kScoreWarps * s.batch;
    s.cta_blocks = ceil_div(ceil_div(blocks, static_cast<int>(ctas < blocks ? ctas : blocks)), round) * round;
    return s;
}

// Three stages of at most 128 blocks and heads of 128, or 64 of 256, elements: 4 * dim + 16 bytes for each at most.
constexpr int kScoreSmemLimit = kScoreStages * 128 * (4 * 128 + 16);
static_assert(kScoreSmemLimit >= kScoreStages * 64 * (4 * 256 + 16) && kScoreSmemLimit >= kScoreStages * kScoreWarps * kScoreBatchBytes, "scores");

template <class Kernel>
sfb_status launch_score(Kernel kernel, int threads, size_t smem, dim3 grid, const ScoreParams& p, cudaStream_t stream) {
    // (the same limit for every shape, since another thread may be launching the kernel)
    if (smem > 0) SFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kScoreSmemLimit));
    SFB_CUDA(launch_dependent(kernel, grid, dim3(threads), smem, stream, p));
    return check_launch("sparse_scores");
}

sfb_status launch_scores(const ScoreParams& p, const ScoreShape& shape, int batch, int dtype, cudaStream_t stream) {
    const PagedView& kv = p.kv;
    const int group = p.q_heads / kv.kv_heads;
    const dim3 grid(ceil_div(p.score_stride, shape.cta_blocks), kv.kv_heads, batch);
    if (shape.kind == kScoreAny)
        return dtype == SFB_F32 ? launch_score(score_kernel<float>, 128, 0, grid, p, stream) : launch_score(score_kernel<bf16>, 128, 0, grid, p, stream);
    if (shape.kind == kScoreMma) {
        const size_t smem = static_cast<size_t>(kScoreStages) * shape.batch * (shape.heads * 4 * kv.dim + 16);
        const dim3 grid(ceil_div(p.score_stride, shape.cta_blocks), kv.kv_heads / shape.heads, batch);
        switch (kv.dim / 16) {
#define SFB_SCORE_CASE(KS) case KS: return launch_score(score_mma_kernel<KS>, (ScoreMma<KS>::kWarps + 1) * 32, smem, grid, p, stream);
            SFB_SCORE_CASE(1) SFB_SCORE_CASE(2) SFB_SCORE_CASE(3) SFB_SCORE_CASE(4) SFB_SCORE_CASE(5) SFB_SCORE_CASE(6) SFB_SCORE_CASE(7)
            SFB_SCORE_CASE(8) SFB_SCORE_CASE(9) SFB_SCORE_CASE(10) SFB_SCORE_CASE(11) SFB_SCORE_CASE(12) SFB_SCORE_CASE(13)
            SFB_SCORE_CASE(14) SFB_SCORE_CASE(15) SFB_SCORE_CASE(16)
#undef SFB_SCORE_CASE
        }
    }
    const size_t smem = sizeof(float) * 2 * kv.dim * static_cast<size_t>(shape.batch) * kScoreStages * kScoreWarps;
    const auto by_group = [&](auto k1, auto k2, auto k4) -> sfb_status {
        return group == 1 ? launch_score(k1, 128, smem, grid, p, stream) : group == 2 ? launch_score(k2, 128, smem, grid, p, stream) : launch_score(k4, 128, smem, grid, p, stream);
    };
    if (shape.lanes == 8) return by_group(score_vec_kernel<float, 8, 1>, score_vec_kernel<float, 8, 2>, score_vec_kernel<float, 8, 4>);
    if (shape.lanes == 16) return by_group(score_vec_kernel<float, 16, 1>, score_vec_kernel<float, 16, 2>, score_vec_kernel<float, 16, 4>);
    return by_group(score_vec_kernel<float, 32, 1>, score_vec_kernel<float, 32, 2>, score_vec_kernel<float, 32, 4>);
}

constexpr int kSelectThreads = 1024;

struct SelectParams {
    PagedView kv;
    const void *q, *bounds;
    const float *scores, *sizes;
    double* exact;        // [batch * kv_heads][score_stride]
    int* selected;
    int q_heads, score_stride, size_count, blocks_per_size, budget, sink, recent, cached;
    float error;
};

// Inverse of order_key(float).
__device__ __forceinline__ float score_of_key(uint64_t key) {
    const uint32_t image = static_cast<uint32_t>(key);
    return __uint_as_float(image >> 31 ? image & 0x7fffffffu : ~image);
}

// Score of one block in 64 bits, by one warp: a lane's elements of low and high are read once for all heads.
template <class T>
__device__ double exact_score(const SelectParams& p, int b, int kvh, int block) {
    const PagedView& kv = p.kv;
    const int lane = threadIdx.x & 31, group = p.q_heads / kv.kv_heads;
    const int page = kv.table[static_cast<size_t>(b) * kv.max_blocks + block];
    double best = __longlong_as_double(0x7ff8000000000000ll);  // NaN: ranks last
    if (page < 0 || page >= kv.num_blocks) return best;
    const T* q = static_cast<const T*>(p.q) + (static_cast<size_t>(b) * p.q_heads + kvh * group) * kv.dim;
    const T* low = static_cast<const T*>(p.bounds) + (static_cast<int64_t>(page) * kv.kv_heads + kvh) * 2 * kv.dim;
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        lo[i] = d < kv.dim ? to_float(low[d]) : 0.0F;
        hi[i] = d < kv.dim ? to_float(low[kv.dim + d]) : 0.0F;
    }
    for (int g0 = 0; g0 < group; g0 += 4) {
        double s[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            s[g] = 0.0;
            const T* qg = q + min(g0 + g, group - 1) * kv.dim;   // (heads past the group repeat its last)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = lane + 32 * i;
                const float qv = d < kv.dim ? to_float(qg[d]) : 0.0F;
                if (qv != 0.0F) s[g] += static_cast<double>(qv) * static_cast<double>(qv > 0.0F ? hi[i] : lo[i]);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int g = 0; g < 4; ++g) s[g] += __shfl_xor_sync(0xffffffffu, s[g], o);
#pragma unroll
        for (int g = 0; g < 4; ++g) best = fmax(best, s[g]);  // (fmax ignores NaN)
    }
    return best;
}

// The scores of the pass before are sums in 32 bits, each within
//   err = error * (largest |q|_1 of the heads) * (largest |bound|)
// of the exact one (score_shape).  Any value t with k scores at or above
// it and fewer than k (or at most k) above it then decides every block but those within 2 err of t: those are
// scored again in 64 bits and ranked by that.  Typically none to a handful; equal blocks, or bounds so large that err is
// not finite, send more through the second pass, never a wrong one through the first.
template <class T>
__global__ void __launch_bounds__(kSelectThreads)
select_kernel(const __grid_constant__ SelectParams p) {
    __shared__ SelectShared sh;
    __shared__ float most[2][kSelectThreads / 32];
    __shared__ int counts[2];
    const PagedView& kv = p.kv;
    const int b = blockIdx.y, kvh = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    const int ctx = kv.length(b), group = p.q_heads / kv.kv_heads;
    // the error of the 32-bit scores
    float norm = 0.0F, size = 0.0F;
    for (int g = warp; g < group; g += kSelectThreads / 32) {
        const T* q = static_cast<const T*>(p.q) + (static_cast<size_t>(b) * p.q_heads + kvh * group + g) * kv.dim;
        float s = 0.0F;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < kv.dim) s += fabsf(to_float(q[lane + 32 * i]));
        s = warp_sum(s);
        norm = s > norm || s != s ? s : norm;
    }
    const int n = ctx > 0 ? kv.block_of(ctx - 1) + 1 : 0;
    const size_t row = static_cast<size_t>(b) * kv.kv_heads + kvh;
    int* out = p.selected + row * p.budget;
    const int k = min(p.budget, n);
    if (k == n) {  // everything is kept
        for (int i = threadIdx.x; i < p.budget; i += kSelectThreads) out[i] = i < n ? i : -1;
        return;
    }
    extern __shared__ uint32_t keys[];
    const float* scores = p.scores + row * p.score_stride;
    double* exact = p.exact + row * p.score_stride;
    const int recent_from = n - p.recent, sink = p.sink;
    const auto forced = [&](int i) { return i < sink || i >= recent_from; };
    for (int i = threadIdx.x; i < (n + p.blocks_per_size - 1) / p.blocks_per_size; i += kSelectThreads)
        size = fmaxf(size, p.sizes[row * p.size_count + i]);
    size = warp_max(size);
    if (p.cached) {
#pragma unroll 8
        for (int i = threadIdx.x; i < n; i += kSelectThreads) keys[i] = forced(i) ? kForced : static_cast<uint32_t>(order_key(scores[i]));
    }
    if (lane == 0) { most[0][warp] = norm; most[1][warp] = size; }
    if (threadIdx.x < 2) counts[threadIdx.x] = 0;
    __syncthreads();
    {
        const float a = lane < kSelectThreads / 32 ? most[0][lane] : 0.0F;
        norm = __any_sync(0xffffffffu, a != a) ? __uint_as_float(0x7fc00000u) : warp_max(a);
        size = warp_max(lane < kSelectThreads / 32 ? most[1][lane] : 0.0F);
    }
    const int n_forced = min(sink, n) + min(p.recent, n) - max(0, min(sink, n) - max(recent_from, 0));
    // 2 err: relative to the largest sum of products there can be, and 1e-34 for products below the normal numbers.  Where
    // that sum could leave the range (or is NaN) a 32-bit score says nothing, and every block is ranked in 64 bits.
    const float reach = norm * size;
    const float err2 = reach < 1e37F ? 2.0F * p.error * reach + 1e-34F : INFINITY;
    const bool zeros = norm == 0.0F || size == 0.0F;   // (then every score is exactly zero)
    if (p.cached && k > n_forced) {
        const bool settled = select_mask<kSelectThreads, false>(
            sh, keys, n, k - n_forced,
            [&](uint32_t& low, uint32_t& high) {   // whatever the tolerance lets change places with the k-th (NaN, infinity: all)
                const float from = score_of_key(low) - err2, to = score_of_key(high) + err2;
                low = from > -INFINITY ? static_cast<uint32_t>(order_key(from)) : 1u;
                high = to < INFINITY ? static_cast<uint32_t>(order_key(to)) : kForced - 1;
            },
            [&](int j) -> uint64_t { return order_key(exact_score<T>(p, b, kvh, sh.near[j])); });
        if (settled) {
            walk_bits<kSelectThreads>(sh.scan, (n + 31) / 32, [&](int w, unsigned& take, unsigned& none) { take = sh.words[w]; none = 0; },
                                      [&](int i, int rank) { if (rank < k) out[rank] = i; }, [](int, int) {});
            for (int i = k + threadIdx.x; i < p.budget; i += kSelectThreads) out[i] = -1;
            return;
        }
    }
    // class of a block: 2 kept, 0 left out, 1 to be ranked in 64 bits
    float above = INFINITY, below = INFINITY;
    if (k > n_forced) {
        const Threshold first = select_threshold<kSelectThreads>(
            sh, n, k - n_forced, [&](int i) -> uint64_t { return forced(i) ? 0 : order_key(scores[i]); });
        const float t = score_of_key(first.low);
        above = t + err2;
        below = t - err2;
    }
    const bool open = k > n_forced;
    const auto classify = [&](int i) -> int {
        if (forced(i)) return 2;
        if (!open) return 0;
        const float v = scores[i];
        return v > above ? 2 : (v < below ? 0 : 1);   // (NaN anywhere: 1)
    };
    int near = 0, kept = 0;
    for (int i = threadIdx.x; i < n; i += kSelectThreads) {
        const int c = classify(i);
        near += c == 1;
        kept += c == 2;
    }
    near = __reduce_add_sync(0xffffffffu, near);
    kept = __reduce_add_sync(0xffffffffu, kept);
    if (lane == 0) {
        atomicAdd(&counts[0], near);
        atomicAdd(&counts[1], kept);
    }
    __syncthreads();
    const int room = k - counts[1];       // near blocks still to be kept
    Threshold last{0, 0};
    if (room > 0 && room < counts[0]) {
        for (int i0 = warp * 32; i0 < n; i0 += kSelectThreads) {
            unsigned todo = __ballot_sync(0xffffffffu, i0 + lane < n && classify(i0 + lane) == 1);
            while (todo) {
                const int i = i0 + __ffs(todo) - 1;
                todo &= todo - 1;
                const double v = zeros ? 0.0 : exact_score<T>(p, b, kvh, i);
                if (lane == 0) exact[i] = v;
            }
        }
        __syncthreads();
        last = select_threshold<kSelectThreads>(sh, n, room, [&](int i) -> uint64_t { return classify(i) == 1 ? order_key(exact[i]) : 0; });
    }
    const bool ranked = room > 0 && room < counts[0];
    walk_ranks<kSelectThreads>(sh.walk, n,
        [&](int i) {
            const int c = classify(i);
            if (c == 2 || (c == 1 && room > 0 && !ranked)) return 1;
            if (c == 0 || room <= 0) return 0;
            const uint64_t v = order_key(exact[i]);
            if (last.cut == 0) return v >= last.low ? 1 : 0;
            return v > last.low ? 1 : (v == last.low ? 2 : 0);
        },
        [&](int i, bool take, bool tie, int rank, int ties) {   // ties: the first last.cut of them, lowest indices first
            const int at = rank + min(ties, last.cut);
            if ((take || (tie && ties < last.cut)) && at < k) out[at] = i;
        });
    for (int i = k + threadIdx.x; i < p.budget; i += kSelectThreads) out[i] = -1;
}

struct SparseLayout {
    int score_stride, size_count;
    StepPlan step;
    size_t scores, sizes, partials, total;   // exact scores come first
};

SparseLayout sparse_layout(const sfb_sparse_args& a, bool wide) {
    SparseLayout l{};
    const int covered = a.max_blocks * a.block_tokens;
    const int limit = a.max_context < covered ? a.max_context : covered;
    const int blocks = limit > 0 ? ceil_div(limit, a.block_tokens) : 1;
    l.score_stride = blocks;
    const int64_t kept = a.budget_blocks < blocks ? a.budget_blocks : blocks;
    l.step = step_plan(a.dtype, a.head_dim, a.head_dim_value, a.batch, a.q_heads, a.kv_heads, static_cast<int>(kept * a.block_tokens),
                       a.block_tokens, a.num_blocks, a.splits, wide);
    const size_t rows = static_cast<size_t>(a.batch) * a.kv_heads;
    l.size_count = ceil_div(blocks, 16);     // no scoring kernel takes fewer blocks a CTA
    l.scores = round_up16(sizeof(double) * rows * blocks);
    l.sizes = l.scores + round_up16(sizeof(float) * rows * blocks);
    l.partials = l.sizes + round_up16(sizeof(float) * rows * l.size_count);
    l.total = l.partials + l.step.bytes;
    return l;
}

sfb_status check_sparse(const sfb_sparse_args* a) {
    SFB_REQUIRE(a, "sparse decode: null arguments");
    SFB_TRY(check_cache(a->k_pool, a->v_pool, a->block_table, a->batch, a->kv_heads, a->head_dim, a->head_dim_value,
                        a->block_tokens, a->max_blocks, a->num_blocks, a->dtype, "sparse decode"));
    SFB_REQUIRE(a->q_heads > 0 && a->q_heads % a->kv_heads == 0, "invalid grouped-query attention configuration");
    SFB_REQUIRE(a->max_context > 0, "sparse decode: max_context must be positive");
    SFB_REQUIRE(a->budget_blocks > 0 && a->sink_blocks >= 0 && a->recent_blocks >= 0 &&
                    static_cast<int64_t>(a->sink_blocks) + a->recent_blocks <= a->budget_blocks,
                "sparse decode: the sink and recent blocks have to fit into the budget");
    return SFB_OK;
}

}  // namespace
}  // namespace sfb

using namespace sfb;

extern "C" {

sfb_status sfb_k_paged_kv_bounds(const sfb_bounds_args* a, sfb_stream stream) {
    SFB_REQUIRE(a && a->bounds && a->start_len && a->end_len, "block bounds: null tensor");
    SFB_TRY(check_cache(a->k_pool, a->k_pool, a->block_table, a->batch, a->kv_heads, a->head_dim, a->head_dim,
                        a->block_tokens, a->max_blocks, a->num_blocks, a->dtype, "block bounds"));
    SFB_REQUIRE(a->max_tokens > 0, "block bounds: max_tokens must be positive");
    const PagedView kv = make_view(a->k_pool, a->k_pool, a->block_table, a->end_len, a->kv_heads, a->head_dim, a->head_dim,
                                   a->block_tokens, a->max_blocks, a->num_blocks, a->max_blocks * a->block_tokens);
    const int vec = a->head_dim % 4 == 0 && aligned16(a->k_pool);
    const int64_t touched = a->max_tokens / a->block_tokens + 2;
    const int64_t spread = touched < a->max_blocks ? touched : a->max_blocks;
    const dim3 grid(static_cast<unsigned>(ceil_div64(spread, 4)), a->kv_heads, a->batch);
    if (a->dtype == SFB_F32)
        SFB_CUDA(launch_dependent(bounds_kernel<float>, grid, dim3(128), 0, as_stream(stream), kv, a->start_len, static_cast<float*>(a->bounds), vec));
    else
        SFB_CUDA(launch_dependent(bounds_kernel<bf16>, grid, dim3(128), 0, as_stream(stream), kv, a->start_len, static_cast<bf16*>(a->bounds), vec));
    return check_launch("paged_kv_bounds");
}

size_t sfb_attention_sparse_workspace(const sfb_sparse_args* a) {
    if (check_sparse(a) != SFB_OK) return 0;
    return std::max(sparse_layout(*a, true).total, sparse_layout(*a, false).total);   // (the addresses may not be set yet)
}

sfb_status sfb_k_attention_decode_sparse(const sfb_sparse_args* a, sfb_stream stream) {
    SFB_TRY(check_sparse(a));
    SFB_REQUIRE(a->q && a->bounds && a->context_len && a->out && a->selected && a->workspace, "sparse decode: null tensor");
    SFB_REQUIRE(aligned16(a->workspace), "sparse decode: the workspace has to be 16-byte aligned");
    const SparseLayout l = sparse_layout(*a, aligned16(a->k_pool) && aligned16(a->v_pool) && aligned16(a->q));
    const PagedView kv = make_view(a->k_pool, a->v_pool, a->block_table, a->context_len, a->kv_heads, a->head_dim, a->head_dim_value,
                                   a->block_tokens, a->max_blocks, a->num_blocks, a->max_context);
    cudaStream_t s = as_stream(stream);
    char* ws = static_cast<char*>(a->workspace);
    double* exact = reinterpret_cast<double*>(ws);
    float *scores = reinterpret_cast<float*>(ws + l.scores), *sizes = reinterpret_cast<float*>(ws + l.sizes);
    const ScoreShape shape = score_shape(*a, l.score_stride);
    {
        const ScoreParams p{kv, a->q, a->bounds, scores, sizes, a->q_heads, l.score_stride, shape.batch, shape.cta_blocks, shape.heads};
        SFB_TRY(launch_scores(p, shape, a->batch, a->dtype, s));
    }
    {
        const SelectParams p{kv, a->q, a->bounds, scores, sizes, exact, a->selected, a->q_heads, l.score_stride,
                             ceil_div(l.score_stride, shape.cta_blocks), shape.cta_blocks, a->budget_blocks, a->sink_blocks, a->recent_blocks, l.score_stride <= kMaskItems, shape.error};
        const dim3 grid(a->kv_heads, a->batch);
        const size_t smem = p.cached ? sizeof(float) * l.score_stride : 0;
        const auto go = [&](auto kernel) -> sfb_status {
            SFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(uint32_t) * kMaskItems)));
            SFB_CUDA(launch_dependent(kernel, grid, dim3(kSelectThreads), smem, s, p));
            return SFB_OK;
        };
        SFB_TRY(a->dtype == SFB_F32 ? go(select_kernel<float>) : go(select_kernel<bf16>));
        SFB_TRY(check_launch("sparse_select"));
    }
    StepParams p{};
    p.kv = kv; p.q = a->q; p.out = a->out;
    p.part = step_partials(l.step, a->batch, a->q_heads, a->head_dim_value, ws + l.partials);
    p.selected = a->selected; p.budget = a->budget_blocks;
    p.batch = a->batch; p.q_heads = a->q_heads; p.chunk_blocks = l.step.chunk_blocks;
    p.scale_log2 = (a->scale > 0.0F ? a->scale : 1.0F / sqrtf(static_cast<float>(a->head_dim))) * 1.4426950408889634F;
    SFB_TRY(step_attention(p, l.step, a->dtype, s));
    if (step_joined(l.step)) return SFB_OK;
    return merge_partials({p.part, kv, a->out, nullptr, a->batch, a->q_heads, 1, a->head_dim_value, 1, 0}, a->dtype, s);
}

}  // extern "C"
