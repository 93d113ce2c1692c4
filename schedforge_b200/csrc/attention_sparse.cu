// Decode attention over selected blocks of a paged cache.
//
// For each block of the cache and each key element the smallest and largest value are kept beside the pool
// (sfb_k_paged_kv_bounds).  sum_d max(q_d low_d, q_d high_d) then bounds every logit of the block from above at a
// sixteenth of the keys' bytes (16-token blocks), and the blocks with the largest bounds are attended to.
// Three steps: scores (memory-bound on the bounds), selection (one CTA per (sequence, K/V head)), attention over the
// list (step_attention).  Scores are summed in 64 bits: ranks follow from them, and with 64 bits a different order of
// summation cannot swap two blocks that are not equal for all purposes.
#include "cache_ops.cuh"
#include "select.cuh"

namespace sfb {
namespace {

template <class T>
__global__ void __launch_bounds__(128)
bounds_kernel(const __grid_constant__ PagedView kv, const int* __restrict__ start_len, T* __restrict__ bounds) {
    const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependents_may_launch();
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
    double* scores;       // [batch * kv_heads][score_stride]
    int q_heads, score_stride;
};

// One warp per block; lane owns every 32nd element.
template <class T>
__global__ void __launch_bounds__(256)
score_kernel(const __grid_constant__ ScoreParams p) {
    const PagedView& kv = p.kv;
    const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependents_may_launch();
    grid_dependency_wait();
    const int ctx = kv.length(b);
    const int blocks = ctx > 0 ? kv.block_of(ctx - 1) + 1 : 0;
    const int group = p.q_heads / kv.kv_heads;
    const T* q = static_cast<const T*>(p.q) + (static_cast<size_t>(b) * p.q_heads + kvh * group) * kv.dim;
    for (int block = blockIdx.x * 8 + warp; block < blocks; block += gridDim.x * 8) {
        const int page = kv.table[static_cast<size_t>(b) * kv.max_blocks + block];
        double best = __longlong_as_double(0x7ff8000000000000ll);  // NaN: ranks last
        if (page >= 0 && page < kv.num_blocks) {
            const T* lo = static_cast<const T*>(p.bounds) + (static_cast<int64_t>(page) * kv.kv_heads + kvh) * 2 * kv.dim;
            const T* hi = lo + kv.dim;
            for (int g = 0; g < group; ++g) {
                double s = 0.0;
                for (int d = lane; d < kv.dim; d += 32) {
                    const float qv = to_float(q[g * kv.dim + d]);
                    s += static_cast<double>(qv) * static_cast<double>(to_float(qv > 0.0F ? hi[d] : lo[d]));
                }
                s = warp_sum(s);
                best = fmax(best, s);  // (fmax ignores NaN)
            }
        } else if (lane == 0) {
            atomicOr(kv.status, kCodeDecodeBounds);
        }
        if (lane == 0) p.scores[(static_cast<size_t>(b) * kv.kv_heads + kvh) * p.score_stride + block] = best;
    }
}

constexpr int kSelectThreads = 512;

struct SelectParams {
    PagedView kv;
    const double* scores;
    int* selected;
    int score_stride, budget, sink, recent;
};

__global__ void __launch_bounds__(kSelectThreads)
select_kernel(const __grid_constant__ SelectParams p) {
    __shared__ SelectShared sh;
    const PagedView& kv = p.kv;
    const int b = blockIdx.y, kvh = blockIdx.x;
    grid_dependents_may_launch();
    grid_dependency_wait();
    const int ctx = kv.length(b);
    const int n = ctx > 0 ? kv.block_of(ctx - 1) + 1 : 0;
    const size_t row = static_cast<size_t>(b) * kv.kv_heads + kvh;
    int* out = p.selected + row * p.budget;
    const int k = min(p.budget, n);
    if (k == n) {  // everything is kept
        for (int i = threadIdx.x; i < p.budget; i += kSelectThreads) out[i] = i < n ? i : -1;
        return;
    }
    const double* scores = p.scores + row * p.score_stride;
    const int recent_from = n - p.recent, sink = p.sink;
    const auto key = [&](int i) -> uint64_t { return i < sink || i >= recent_from ? ~0ull : order_key(scores[i]); };
    const Threshold t = select_threshold<kSelectThreads>(sh, n, k, key);
    int written = 0, ties = 0;
    for (int i0 = 0; i0 < n; i0 += kSelectThreads) {
        const int i = i0 + threadIdx.x;
        const uint64_t v = i < n ? key(i) : 0;
        const bool tie = i < n && t.cut != 0 && v == t.low;
        const bool above = i < n && (t.cut != 0 ? v > t.low : v >= t.low);
        int above_rank, tie_rank, above_total, tie_total;
        flag_ranks<kSelectThreads>(sh.scan, above, tie, above_rank, tie_rank, above_total, tie_total);
        const int tie_room = t.cut - ties;                   // ties still to be kept, lowest indices first
        const int at = written + above_rank + min(tie_rank, max(tie_room, 0));
        if (above || (tie && tie_rank < tie_room)) out[at] = i;
        written += above_total + min(tie_total, max(tie_room, 0));
        ties += tie_total;
    }
    for (int i = k + threadIdx.x; i < p.budget; i += kSelectThreads) out[i] = -1;
}

struct SparseLayout {
    int score_stride, splits, chunk_blocks;
    size_t scores, partials, total;
};

SparseLayout sparse_layout(const sfb_sparse_args& a) {
    SparseLayout l{};
    const int covered = a.max_blocks * a.block_tokens;
    const int limit = a.max_context < covered ? a.max_context : covered;
    const int blocks = limit > 0 ? ceil_div(limit, a.block_tokens) : 1;
    l.score_stride = blocks;
    const int64_t kept = a.budget_blocks < blocks ? a.budget_blocks : blocks;
    l.splits = step_splits(a.batch, a.kv_heads, static_cast<int>(kept * a.block_tokens), a.block_tokens, a.splits, &l.chunk_blocks);
    l.scores = round_up16(sizeof(double) * static_cast<size_t>(a.batch) * a.kv_heads * blocks);
    l.partials = sizeof(float) * static_cast<size_t>(a.batch) * a.q_heads * l.splits * (a.head_dim_value + 2);
    l.total = l.scores + l.partials;
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
    const int64_t touched = a->max_tokens / a->block_tokens + 2;
    const int64_t spread = touched < a->max_blocks ? touched : a->max_blocks;
    const dim3 grid(static_cast<unsigned>(ceil_div64(spread, 4)), a->kv_heads, a->batch);
    if (a->dtype == SFB_F32)
        SFB_CUDA(launch_dependent(bounds_kernel<float>, grid, dim3(128), 0, as_stream(stream), kv, a->start_len, static_cast<float*>(a->bounds)));
    else
        SFB_CUDA(launch_dependent(bounds_kernel<bf16>, grid, dim3(128), 0, as_stream(stream), kv, a->start_len, static_cast<bf16*>(a->bounds)));
    return check_launch("paged_kv_bounds");
}

size_t sfb_attention_sparse_workspace(const sfb_sparse_args* a) {
    if (check_sparse(a) != SFB_OK) return 0;
    return sparse_layout(*a).total;
}

sfb_status sfb_k_attention_decode_sparse(const sfb_sparse_args* a, sfb_stream stream) {
    SFB_TRY(check_sparse(a));
    SFB_REQUIRE(a->q && a->bounds && a->context_len && a->out && a->selected && a->workspace, "sparse decode: null tensor");
    SFB_REQUIRE(aligned16(a->workspace), "sparse decode: the workspace has to be 16-byte aligned");
    const SparseLayout l = sparse_layout(*a);
    const PagedView kv = make_view(a->k_pool, a->v_pool, a->block_table, a->context_len, a->kv_heads, a->head_dim, a->head_dim_value,
                                   a->block_tokens, a->max_blocks, a->num_blocks, a->max_context);
    cudaStream_t s = as_stream(stream);
    char* ws = static_cast<char*>(a->workspace);
    {
        const ScoreParams p{kv, a->q, a->bounds, reinterpret_cast<double*>(ws), a->q_heads, l.score_stride};
        const dim3 grid(ceil_div(l.score_stride, 8), a->kv_heads, a->batch);
        if (a->dtype == SFB_F32) SFB_CUDA(launch_dependent(score_kernel<float>, grid, dim3(256), 0, s, p));
        else SFB_CUDA(launch_dependent(score_kernel<bf16>, grid, dim3(256), 0, s, p));
        SFB_TRY(check_launch("sparse_scores"));
    }
    {
        const SelectParams p{kv, reinterpret_cast<const double*>(ws), a->selected, l.score_stride, a->budget_blocks, a->sink_blocks,
                             a->recent_blocks};
        SFB_CUDA(launch_dependent(select_kernel, dim3(a->kv_heads, a->batch), dim3(kSelectThreads), 0, s, p));
        SFB_TRY(check_launch("sparse_select"));
    }
    StepParams p{};
    p.kv = kv; p.q = a->q; p.out = a->out; p.partials = reinterpret_cast<float*>(ws + l.scores);
    p.selected = a->selected; p.budget = a->budget_blocks;
    p.batch = a->batch; p.q_heads = a->q_heads; p.splits = l.splits; p.chunk_blocks = l.chunk_blocks;
    p.scale_log2 = (a->scale > 0.0F ? a->scale : 1.0F / sqrtf(static_cast<float>(a->head_dim))) * 1.4426950408889634F;
    SFB_TRY(step_attention(p, a->dtype, s));
    if (l.splits == 1) return SFB_OK;
    return merge_partials({p.partials, a->out, nullptr, a->batch, a->q_heads, 1, a->head_dim_value, l.splits, 1}, a->dtype, s);
}

}  // extern "C"
