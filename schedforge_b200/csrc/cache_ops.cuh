// Shared pieces of the serving operators over the paged cache: guarded cache access, the bookkeeping of cut work and the
// joining of partial results.
//
// The kernels are launched with launch_dependent() and wait for the kernel before at once; none announces its dependents
// early: blocks that came in ahead of time only took room from the ones they waited for (one eviction step 11.8 us with
// griddepcontrol.launch_dependents at the start of its kernels, 9.2 us without).
#pragma once

#include "attention_decode.cuh"
#include "common.cuh"

namespace sfb {

// One paged cache as every operator sees it.  limit: the longest context that the tables, the workspace and
// max_context cover.
struct PagedView {
    const void *k_pool, *v_pool;
    const int *table, *lens;
    int kv_heads, dim, dim_v, block_tokens, block_shift, max_blocks, num_blocks, limit;  // block_shift < 0: not a power of two
    uint32_t* status;

    __device__ __forceinline__ int length(int b) const {
        int n = lens[b];
        if (n < 0 || n > limit) {
            n = n < 0 ? 0 : limit;
            if (threadIdx.x == 0) atomicOr(status, kCodeDecodeBounds);
        }
        return n;
    }
    __device__ __forceinline__ int block_of(int position) const {
        return block_shift >= 0 ? position >> block_shift : position / block_tokens;
    }
    // Row of position `position` of sequence b and K/V head `head` in the [blocks][heads][tokens] pool; -1 where the
    // table names no block of the pool.
    __device__ __forceinline__ int64_t row(int b, int head, int position) const { return row_in(page(b, position), head, position); }
    __device__ __forceinline__ int page(int b, int position) const { return table[static_cast<size_t>(b) * max_blocks + block_of(position)]; }
    __device__ __forceinline__ int64_t row_in(int page, int head, int position) const {
        const int block = block_of(position);
        if (page < 0 || page >= num_blocks) {
            atomicOr(status, kCodeDecodeBounds);
            return -1;
        }
        return (static_cast<int64_t>(page) * kv_heads + head) * block_tokens + (position - block * block_tokens);
    }
};

inline int shift_of(int n) {
    for (int s = 0; s < 31; ++s)
        if (n == 1 << s) return s;
    return -1;
}

// Checks what all operators share.
sfb_status check_cache(const void* k_pool, const void* v_pool, const int* table, int batch, int kv_heads, int dim, int dim_v,
                       int block_tokens, int max_blocks, int num_blocks, int dtype, const char* what);

PagedView make_view(const void* k_pool, const void* v_pool, const int* table, const int* lens, int kv_heads, int dim, int dim_v,
                    int block_tokens, int max_blocks, int num_blocks, int max_context);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline size_t round_up16(size_t n) { return (n + 15) & ~size_t(15); }

// ---- partial results -------------------------------------------------------------------------------------------------
// A query row's attention may be cut along the keys; each piece leaves its maximum (base-2 units), its sum and its
// numerator.  Two arrangements: a fixed number of splits per row, or, where every CTA takes an equal range of all rows'
// work, the pieces of CTAs first..last of the row's (sequence, K/V head) pair, piece = CTA + pair.
struct Partials {
    float* ml;         // maximum and sum of index i at ml[i * ml_step]
    float* o;          // numerator of index i at o[i * o_step]
    int2* span;        // first and last CTA of every pair; nullptr: fixed splits
    int splits, ml_step, o_step;
};
constexpr int kPieceHeads = 8;    // query heads per pair in the arrangement by CTAs
constexpr int kMaxPieces = 512;   // pieces of one row (the joining kernels keep a factor for each)

// ---- one query token per sequence --------------------------------------------------------------------------------
// Attention of the query heads of one K/V head over the blocks of a list (selected != nullptr) or over the whole
// context.  logits != nullptr: the scaled logit of every position is kept there (base-2 units), and every row leaves a
// partial result.
struct StepParams {
    PagedView kv;
    const void* q;
    void* out;
    Partials part;
    float* logits;          // [batch, q_heads, logit_stride]
    const int* selected;    // [batch, kv_heads, budget]
    int64_t logit_stride;
    int budget;
    int batch, q_heads, chunk_blocks;
    float scale_log2;
};

// How a step is cut; decided by type, sizes and the wanted splits alone, so that the workspace can be sized without
// the tensors.
struct StepPlan {
    bool mma;            // attention_step_mma.cu: even ranges; else attention_step.cu: fixed splits
    int ctas, splits, chunk_blocks;
    int64_t pairs;
    size_t bytes;        // of the partial results
};
StepPlan step_plan(int dtype, int dim, int dim_v, int batch, int q_heads, int kv_heads, int tokens, int block_tokens, int num_blocks,
                   int wanted, bool wide);
Partials step_partials(const StepPlan& plan, int batch, int q_heads, int dim_v, void* workspace);
sfb_status step_attention(const StepParams& p, const StepPlan& plan, int dtype, cudaStream_t stream);
sfb_status step_mma(const StepParams& p, const StepPlan& plan, cudaStream_t stream);
inline bool step_joined(const StepPlan& plan) { return !plan.mma && plan.splits == 1; }   // nothing is left to join

// ---- joining --------------------------------------------------------------------------------------------------------
// Rows are (b, q_head, node); nodes == 1 and node_count == nullptr for single-token decode.
struct MergeParams {
    Partials part;
    PagedView kv;            // lengths and heads
    void* out;
    const int* node_count;
    int batch, q_heads, nodes, dim_v, token_major;
    int chunk;               // keys of a split, the last split the rest; only the splits that have keys left a piece.  0: all did
};
sfb_status merge_partials(const MergeParams& p, int dtype, cudaStream_t stream);

#ifdef __CUDACC__
// Eight consecutive elements of a 16-byte aligned row.
template <class T> struct Raw8;
template <> struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.0F, 0.0F, 0.0F, 0.0F); }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
};
template <> struct Raw8<bf16> {
    uint4 a;
    __device__ __forceinline__ void load(const bf16* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void zero() { a = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Where the pieces of query row (b, head) lie: indices first + i * step, i < count.  ctx: the sequence's length.
struct RowPieces {
    size_t first;
    int step, count;
};
__device__ __forceinline__ RowPieces row_pieces(const Partials& part, int kv_heads, int q_heads, int b, int head, int ctx) {
    if (!part.span) return {(static_cast<size_t>(b) * q_heads + head) * part.splits, 1, part.splits};
    const int group = q_heads / kv_heads, chunks = (group + kPieceHeads - 1) / kPieceHeads;
    const int in_group = head % group;
    const size_t pair = (static_cast<size_t>(b) * kv_heads + head / group) * chunks + in_group / kPieceHeads;
    const int2 span = part.span[pair];
    if (ctx == 0) return {0, 0, 0};   // (nobody wrote the span; its load need not wait for the length)
    return {(span.x + pair) * kPieceHeads + in_group % kPieceHeads, kPieceHeads, min(span.y - span.x + 1, kMaxPieces)};
}

// Maximum and 1 / sum of a row (0 for an empty one) out of its pieces, by one warp; factors != nullptr: the factor of
// every piece.  Up to 64 pieces are read once, all at the same time.
__device__ __forceinline__ float2 row_statistics(const Partials& part, const RowPieces& r, float* factors) {
    const int lane = threadIdx.x & 31;
    const auto read = [&](int i) -> float2 {
        const float* at = part.ml + (r.first + static_cast<size_t>(i) * r.step) * part.ml_step;
        return i < r.count ? make_float2(at[0], at[1]) : make_float2(-INFINITY, 0.0F);
    };
    const float2 a = read(lane), b = read(lane + 32);
    float top = fmaxf(a.x, b.x);
    for (int i = lane + 64; i < r.count; i += 32) top = fmaxf(top, read(i).x);
    top = warp_max(top);
    if (top == -INFINITY) top = 0.0F;
    const float fa = a.x == -INFINITY ? 0.0F : exp2_fast(a.x - top), fb = b.x == -INFINITY ? 0.0F : exp2_fast(b.x - top);
    float sum = a.y * fa + b.y * fb;
    for (int i = lane + 64; i < r.count; i += 32) {
        const float2 v = read(i);
        sum += v.x == -INFINITY ? 0.0F : v.y * exp2_fast(v.x - top);
    }
    sum = warp_sum(sum);
    const float inv = sum == 0.0F ? 0.0F : 1.0F / sum;
    if (factors) {
        if (lane < r.count) factors[lane] = fa * inv;
        if (lane + 32 < r.count) factors[lane + 32] = fb * inv;
        for (int i = lane + 64; i < r.count; i += 32) {
            const float2 v = read(i);
            factors[i] = v.x == -INFINITY ? 0.0F : exp2_fast(v.x - top) * inv;
        }
    }
    return make_float2(top, inv);
}

// The range of CTA blockIdx.x when the work units of `batch` sequences (count(b) units for each of their `subs` pairs)
// are laid end to end and cut into gridDim.x equal ranges (a multiple of `granule` units each).  One whole warp calls it.  out: sequence, pair inside
// it, unit inside the pair, units of this CTA (0: none), units of a full range.
template <class Count>
__device__ __forceinline__ void even_range(int batch, int64_t subs, int granule, Count count, int* out) {
    const int lane = threadIdx.x & 31;
    const int first_count = lane < batch ? count(lane) : 0;   // (the only ones up to 32 sequences)
    int64_t total = __reduce_add_sync(0xffffffffu, first_count);
    for (int b0 = 32; b0 < batch; b0 += 32) total += __reduce_add_sync(0xffffffffu, b0 + lane < batch ? count(b0 + lane) : 0);
    total *= subs;
    int64_t per = (total + gridDim.x - 1) / gridDim.x;
    per = (per + granule - 1) / granule * granule;
    if (per < granule) per = granule;
    const int64_t first = blockIdx.x * per;
    const int64_t mine = first < total ? (total - first < per ? total - first : per) : 0;
    if (mine > 0) {
        int64_t before = 0;
        for (int b0 = 0; b0 < batch; b0 += 32) {
            const int n = b0 == 0 ? first_count : (b0 + lane < batch ? count(b0 + lane) : 0);
            int sum = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            const int64_t end = before + sum * subs, begin = end - n * subs;
            const bool here = n > 0 && begin <= first && first < end;
            if (here) {
                out[0] = b0 + lane;
                out[1] = static_cast<int>((first - begin) / n);
                out[2] = static_cast<int>((first - begin) % n);
            }
            if (__any_sync(0xffffffffu, here)) break;
            before += __shfl_sync(0xffffffffu, sum, 31) * subs;
        }
    }
    if (lane == 0) {
        out[3] = static_cast<int>(mine);
        out[4] = static_cast<int>(per);
    }
}

#endif

}  // namespace sfb
