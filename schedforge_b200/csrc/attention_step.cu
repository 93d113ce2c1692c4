// Single-token attention over a paged cache, CUDA-core form: any type, head dimension up to 256, block size and group.
//
// One CTA handles one (sequence, K/V head, up to eight query heads, split).  A key row is read by LPR lanes, eight
// elements each, so that a warp has 32 / LPR rows in flight, four times over (twice where four float32 or eight bf16 heads
// leave too few registers for four CTAs an SM: 295 -> 240 us for 16 ragged float32 sequences to 8192 tokens, 32/8 heads of
// 128); the blocks of the next rows are looked up a round ahead.  Every lane group runs its own online softmax over the
// rows it meets (no synchronisation while streaming), and the groups, warps and splits are joined by the log-sum-exp rule.  All heads of the CTA share each K and V byte.  Memory-bound for small groups; the K/V bytes
// are read once per eight query heads.
#include "cache_ops.cuh"

namespace sfb {
namespace {

constexpr int kWarps = 4;

// Eight elements of a row: lane `sub` of LPR owns [8 * sub, 8 * sub + 8) (VEC: dim % 8 == 0 and 16-byte aligned rows),
// or every LPR-th element.
template <class T, int LPR, bool VEC>
struct Piece {
    Raw8<T> raw;
    float f[8];
    __device__ __forceinline__ void load(const T* row, int sub, int dim, bool live) {
        if constexpr (VEC) {
            if (live && 8 * sub < dim) raw.load(row + 8 * sub);
            else raw.zero();
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = sub + LPR * i;
                f[i] = live && d < dim ? to_float(row[d]) : 0.0F;
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (VEC) raw.get(v);
        else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = f[i];
        }
    }
};

template <class T, int LPR, int G, bool VEC>
__global__ void __launch_bounds__(kWarps * 32)
step_kernel(const __grid_constant__ StepParams p) {
    constexpr int RPW = 32 / LPR, kRows = G * sizeof(T) >= 16 ? 2 : 4;
    extern __shared__ float merge_smem[];  // [kWarps][G][dim_v + 2]
    const PagedView& kv = p.kv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LPR, rg = lane / LPR;
    const int group = p.q_heads / kv.kv_heads;
    const int split = blockIdx.x, b = blockIdx.z;
    const int chunks = (group + G - 1) / G;
    const int kvh = blockIdx.y / chunks, head0 = kvh * group + (blockIdx.y % chunks) * G;
    const int heads = min(G, (kvh + 1) * group - head0);
    grid_dependency_wait();
    const int ctx = kv.length(b);
    const int* list = p.selected ? p.selected + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.budget : nullptr;
    const int blocks = ctx > 0 ? kv.block_of(ctx - 1) + 1 : 0;
    const int entries = list ? min(p.budget, blocks) : blocks;
    const int e0 = min(entries, split * p.chunk_blocks), e1 = min(entries, e0 + p.chunk_blocks);
    const int rows = (e1 - e0) * kv.block_tokens;

    float q[G][8], o[G][8], m[G], l[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        Piece<T, LPR, VEC> piece;
        piece.load(static_cast<const T*>(p.q) + (static_cast<size_t>(b) * p.q_heads + head0 + (g < heads ? g : 0)) * kv.dim, sub, kv.dim, g < heads);
        piece.get(q[g]);
#pragma unroll
        for (int i = 0; i < 8; ++i) { q[g][i] *= p.scale_log2; o[g][i] = 0.0F; }
        m[g] = -INFINITY;
        l[g] = 0.0F;
    }
    // block and position (-1: none) of the warp's rows base + u * RPW + rg, read one round ahead
    int next_page[kRows], next_position[kRows];
    const auto locate = [&](int base) {
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            const int r = base + u * RPW + rg;
            next_page[u] = -1;
            next_position[u] = -1;
            if (r >= rows) continue;
            const int e = kv.block_of(r);
            const int logical = list ? list[e0 + e] : e0 + e;
            // (a list entry of -1 ends the list; it cannot be met before `entries`, but is not followed either)
            const int at = logical * kv.block_tokens + (r - e * kv.block_tokens);
            if (logical < 0 || at >= ctx) continue;
            next_position[u] = at;
            next_page[u] = kv.page(b, at);
        }
    };
    locate(warp * RPW * kRows);
    for (int base = warp * RPW * kRows; base < rows; base += kWarps * RPW * kRows) {
        Piece<T, LPR, VEC> kp[kRows], vp[kRows];
        int position[kRows];
        bool live[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            position[u] = next_position[u];
            const int64_t at = position[u] >= 0 ? kv.row_in(next_page[u], kvh, position[u]) : -1;
            live[u] = at >= 0;
            kp[u].load(static_cast<const T*>(kv.k_pool) + (live[u] ? at : 0) * kv.dim, sub, kv.dim, live[u]);
            vp[u].load(static_cast<const T*>(kv.v_pool) + (live[u] ? at : 0) * kv.dim_v, sub, kv.dim_v, live[u]);
            if (position[u] >= 0 && !live[u] && p.logits && sub < heads)   // a position whose block is missing weighs nothing
                p.logits[(static_cast<size_t>(b) * p.q_heads + head0 + sub) * p.logit_stride + position[u]] = -INFINITY;
        }
        locate(base + kWarps * RPW * kRows);
        float x[kRows][G];
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            float f[8];
            kp[u].get(f);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float s = 0.0F;
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fmaf(q[g][i], f[i], s);
                x[u][g] = s;
            }
        }
#pragma unroll
        for (int w = 1; w < LPR; w <<= 1)
#pragma unroll
            for (int u = 0; u < kRows; ++u)
#pragma unroll
                for (int g = 0; g < G; ++g) x[u][g] += __shfl_xor_sync(0xffffffffu, x[u][g], w);
        if (p.logits) {
#pragma unroll
            for (int u = 0; u < kRows; ++u)
#pragma unroll
                for (int g = 0; g < G; ++g)
                    if (live[u] && sub == g % LPR && g < heads)
                        p.logits[(static_cast<size_t>(b) * p.q_heads + head0 + g) * p.logit_stride + position[u]] = x[u][g];
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float top = m[g];
#pragma unroll
            for (int u = 0; u < kRows; ++u)
                if (live[u]) top = fmaxf(top, x[u][g]);
            const float alpha = top == -INFINITY ? 1.0F : exp2f(m[g] - top);
            m[g] = top;
            l[g] *= alpha;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[g][i] *= alpha;
#pragma unroll
            for (int u = 0; u < kRows; ++u) {
                x[u][g] = live[u] && x[u][g] != -INFINITY ? exp2f(x[u][g] - top) : 0.0F;
                l[g] += x[u][g];
            }
        }
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
            float f[8];
            vp[u].get(f);
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 8; ++i) o[g][i] = fmaf(x[u][g], f[i], o[g][i]);
        }
    }
    // lane groups of the warp
#pragma unroll
    for (int w = LPR; w < 32; w <<= 1)
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float other = __shfl_xor_sync(0xffffffffu, m[g], w);
            const float top = fmaxf(m[g], other);
            const float mine = m[g] == -INFINITY ? 0.0F : exp2f(m[g] - top);
            l[g] = l[g] * mine;
            l[g] += __shfl_xor_sync(0xffffffffu, l[g], w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                o[g][i] *= mine;
                o[g][i] += __shfl_xor_sync(0xffffffffu, o[g][i], w);
            }
            m[g] = top;
        }
    const int record = kv.dim_v + 2;
    if (rg == 0) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float* rec = merge_smem + (warp * G + g) * record;
            if (sub == 0) { rec[0] = m[g]; rec[1] = l[g]; }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = VEC ? 8 * sub + i : sub + LPR * i;
                if (d < kv.dim_v) rec[2 + d] = o[g][i];
            }
        }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < heads * record; idx += kWarps * 32) {
        const int g = idx / record, c = idx % record;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, merge_smem[(w * G + g) * record]);
        float sum = 0.0F, value = 0.0F;
        if (top != -INFINITY) {
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float* rec = merge_smem + (w * G + g) * record;
                const float f = rec[0] == -INFINITY ? 0.0F : exp2f(rec[0] - top);
                sum += rec[1] * f;
                value += rec[c] * f;
            }
        }
        const size_t row = static_cast<size_t>(b) * p.q_heads + head0 + g;
        if (p.part.splits == 1 && !p.logits) {
            if (c >= 2) static_cast<T*>(p.out)[row * kv.dim_v + c - 2] = from_float<T>(sum == 0.0F ? 0.0F : value / sum);
        } else {
            p.part.ml[(row * p.part.splits + split) * record + c] = c == 0 ? top : c == 1 ? sum : value;
        }
    }
}

template <class T, int LPR, bool VEC>
sfb_status launch_step(const StepParams& p, cudaStream_t stream) {
    const int group = p.q_heads / p.kv.kv_heads;
    const auto go = [&](auto kernel, int g) -> sfb_status {
        const size_t smem = sizeof(float) * kWarps * g * (p.kv.dim_v + 2);
        const dim3 grid(p.part.splits, p.kv.kv_heads * ceil_div(group, g), p.batch);
        SFB_CUDA(launch_dependent(kernel, grid, dim3(kWarps * 32), smem, stream, p));
        return check_launch("attention_step");
    };
    if (group == 1) return go(step_kernel<T, LPR, 1, VEC>, 1);
    if (group == 2) return go(step_kernel<T, LPR, 2, VEC>, 2);
    if (group <= 4) return go(step_kernel<T, LPR, 4, VEC>, 4);
    return go(step_kernel<T, LPR, 8, VEC>, 8);
}

template <class T>
sfb_status step_typed(const StepParams& p, cudaStream_t stream) {
    const PagedView& kv = p.kv;
    const bool vec = kv.dim % 8 == 0 && kv.dim_v % 8 == 0 && aligned16(p.q) && aligned16(kv.k_pool) && aligned16(kv.v_pool);
    const int widest = kv.dim > kv.dim_v ? kv.dim : kv.dim_v;
    if (!vec) return launch_step<T, 32, false>(p, stream);
    if (widest <= 64) return launch_step<T, 8, true>(p, stream);
    if (widest <= 128) return launch_step<T, 16, true>(p, stream);
    return launch_step<T, 32, true>(p, stream);
}

// Pieces of a row cut into splits of `chunk` keys.
__device__ __forceinline__ int split_pieces(const MergeParams& p, int b) {
    if (p.chunk == 0) return p.part.splits;
    const int keys = p.kv.length(b) + min(p.node_count ? p.node_count[b] : p.nodes, p.nodes);
    return min(p.part.splits, (keys + p.chunk - 1) / p.chunk);
}

// One CTA per output row; thread = output element (strided), the two halves of the CTA take alternate pieces.
template <class T>
__global__ void __launch_bounds__(256) merge_kernel(const __grid_constant__ MergeParams p) {
    __shared__ float factor[kMaxPieces];
    __shared__ float other[128];
    const int row = blockIdx.x;
    const int node = row % p.nodes, head = (row / p.nodes) % p.q_heads, b = row / p.nodes / p.q_heads;
    grid_dependency_wait();
    if (p.node_count && node >= p.node_count[b]) return;
    RowPieces r;
    if (p.part.span) r = row_pieces(p.part, p.kv.kv_heads, p.q_heads, b, head, p.kv.length(b));
    else r = {static_cast<size_t>(row) * p.part.splits, 1, split_pieces(p, b)};
    if (p.part.span && r.count == 1) return;   // written by the attention kernel itself
    // the first eight pieces of each half are fetched before their factors are known
    const int half = threadIdx.x >> 7;
    float early[8];
    {
        const int d = threadIdx.x & 127;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            early[i] = half + 2 * i < r.count && d < p.dim_v ? p.part.o[(r.first + static_cast<size_t>(half + 2 * i) * r.step) * p.part.o_step + d] : 0.0F;
    }
    if (threadIdx.x < 32) row_statistics(p.part, r, factor);
    __syncthreads();
    T* dst = static_cast<T*>(p.out) + (p.token_major ? (static_cast<size_t>(b) * p.nodes + node) * p.q_heads + head
                                                     : static_cast<size_t>(row)) * p.dim_v;
    for (int d0 = 0; d0 < p.dim_v; d0 += 128) {
        const int d = d0 + (threadIdx.x & 127);
        float a = 0.0F;
        if (d0 == 0)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (half + 2 * i < r.count && factor[half + 2 * i] != 0.0F) a = fmaf(factor[half + 2 * i], early[i], a);
        if (d < p.dim_v)
#pragma unroll 8
            for (int i = half + (d0 == 0 ? 16 : 0); i < r.count; i += 2) {
                const float f = factor[i];
                if (f != 0.0F) a = fmaf(f, p.part.o[(r.first + static_cast<size_t>(i) * r.step) * p.part.o_step + d], a);
            }
        if (half) other[threadIdx.x & 127] = a;
        __syncthreads();
        if (!half && d < p.dim_v) dst[d] = from_float<T>(a + other[threadIdx.x]);
        __syncthreads();
    }
}

// The same with one warp per output row, for many rows.
template <class T>
__global__ void __launch_bounds__(256) merge_rows_kernel(const __grid_constant__ MergeParams p, int rows) {
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= rows) return;
    const int node = row % p.nodes, head = (row / p.nodes) % p.q_heads, b = row / p.nodes / p.q_heads;
    grid_dependency_wait();
    if (p.node_count && node >= p.node_count[b]) return;
    RowPieces r;
    if (p.part.span) r = row_pieces(p.part, p.kv.kv_heads, p.q_heads, b, head, p.kv.length(b));
    else r = {static_cast<size_t>(row) * p.part.splits, 1, split_pieces(p, b)};
    if (p.part.span && r.count == 1) return;   // written by the attention kernel itself
    T* dst = static_cast<T*>(p.out) + (p.token_major ? (static_cast<size_t>(b) * p.nodes + node) * p.q_heads + head
                                                     : static_cast<size_t>(row)) * p.dim_v;
    // up to kAtOnce pieces of the first 64 elements are fetched while the maximum is found
    constexpr int kAtOnce = 8;
    float early[kAtOnce][2];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
            early[i][j] = i < r.count && lane + 32 * j < p.dim_v ? p.part.o[(r.first + static_cast<size_t>(i) * r.step) * p.part.o_step + lane + 32 * j] : 0.0F;
    const float2 stats = row_statistics(p.part, r, nullptr);
    const auto factor = [&](int i) -> float {
        const float m = p.part.ml[(r.first + static_cast<size_t>(i) * r.step) * p.part.ml_step];
        return m == -INFINITY ? 0.0F : exp2_fast(m - stats.x);
    };
    float a[8] = {};
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
        if (i >= r.count) continue;
        const float f = factor(i);
        if (f == 0.0F) continue;
        a[0] = fmaf(early[i][0], f, a[0]);
        a[1] = fmaf(early[i][1], f, a[1]);
    }
#pragma unroll 4
    for (int i = p.dim_v > 64 ? 0 : kAtOnce; i < r.count; ++i) {
        const float f = factor(i);
        const float* o = p.part.o + (r.first + static_cast<size_t>(i) * r.step) * p.part.o_step;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 32 * j < p.dim_v && (j >= 2 || i >= kAtOnce)) a[j] = f == 0.0F ? a[j] : fmaf(o[lane + 32 * j], f, a[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (lane + 32 * j < p.dim_v) dst[lane + 32 * j] = from_float<T>(a[j] * stats.y);
}

}  // namespace

sfb_status check_cache(const void* k_pool, const void* v_pool, const int* table, int batch, int kv_heads, int dim, int dim_v,
                       int block_tokens, int max_blocks, int num_blocks, int dtype, const char* what) {
    const std::string name(what);
    SFB_REQUIRE(k_pool && v_pool && table, name + ": null tensor");
    SFB_REQUIRE(batch > 0 && kv_heads > 0 && dim > 0 && dim_v > 0 && block_tokens > 0 && max_blocks > 0 && num_blocks > 0,
                name + ": invalid cache shape");
    SFB_REQUIRE(dtype == SFB_F32 || dtype == SFB_BF16, name + ": unknown dtype");
    if (dim > 256 || dim_v > 256) return fail(SFB_UNSUPPORTED, name + ": head dimension > 256");
    if (batch > 65535 || kv_heads > 4096) return fail(SFB_UNSUPPORTED, name + ": more than 65535 sequences or 4096 K/V heads");
    if (static_cast<int64_t>(max_blocks) * block_tokens > (int64_t{1} << 29))   // (a warp adds up 32 sequences' units in 32 bits)
        return fail(SFB_UNSUPPORTED, name + ": more than 2^29 positions in a block table");
    return SFB_OK;
}

PagedView make_view(const void* k_pool, const void* v_pool, const int* table, const int* lens, int kv_heads, int dim, int dim_v,
                    int block_tokens, int max_blocks, int num_blocks, int max_context) {
    PagedView kv{};
    kv.k_pool = k_pool; kv.v_pool = v_pool; kv.table = table; kv.lens = lens;
    kv.kv_heads = kv_heads; kv.dim = dim; kv.dim_v = dim_v; kv.block_tokens = block_tokens;
    kv.block_shift = shift_of(block_tokens);
    kv.max_blocks = max_blocks; kv.num_blocks = num_blocks;
    const int covered = max_blocks * block_tokens;
    kv.limit = max_context < covered ? max_context : covered;
    kv.status = device_status_word();
    return kv;
}

// The tensor-core kernel takes bf16, head_dim = head_dim_value = 128 or 64 and blocks of a multiple of 16 tokens; its
// CTAs, two per SM, take equal ranges of all work.  The other one cuts every row into splits of whole blocks: as long as
// two CTAs per SM allow (the ramp of a split is paid once), but at most 512 positions, which evens out ragged contexts (2048:
// 195 instead of 157 us for 64 float32 sequences to 4096 tokens, 307 instead of 252 for eight of 8192), and at least 64.
StepPlan step_plan(int dtype, int dim, int dim_v, int batch, int q_heads, int kv_heads, int tokens, int block_tokens, int num_blocks,
                   int wanted, bool wide) {
    StepPlan plan{};
    const int blocks = tokens > 0 ? ceil_div(tokens, block_tokens) : 1;
    const int64_t slots = 2LL * sm_count(), heads = static_cast<int64_t>(batch) * kv_heads;
    plan.mma = wide && dtype == SFB_BF16 && (dim == 128 || dim == 64) && dim_v == dim && block_tokens % 16 == 0 &&
               static_cast<int64_t>(num_blocks) * kv_heads * block_tokens < (int64_t{1} << 30);
    if (plan.mma) {
        plan.pairs = heads * ceil_div(q_heads / kv_heads, kPieceHeads);
        const int64_t units = plan.pairs * blocks * (block_tokens / 16);
        int64_t ctas = wanted > 0 && plan.pairs * wanted < slots ? plan.pairs * wanted : slots;
        if (ctas > kMaxPieces) ctas = kMaxPieces;
        plan.ctas = static_cast<int>(units < ctas ? units : ctas);
        plan.bytes = round_up16(sizeof(float) * (2 + dim_v) * kPieceHeads * static_cast<size_t>(plan.ctas + plan.pairs)) +
                     sizeof(int2) * static_cast<size_t>(plan.pairs);
        return plan;
    }
    int splits = wanted;
    if (splits <= 0) {
        splits = static_cast<int>(slots / heads < tokens / 64 ? slots / heads : tokens / 64);
        if (splits < ceil_div(tokens, 512)) splits = ceil_div(tokens, 512);
    }
    if (splits > 128) splits = 128;
    if (splits > blocks) splits = blocks;
    if (splits < 1) splits = 1;
    plan.chunk_blocks = ceil_div(blocks, splits);
    plan.splits = ceil_div(blocks, plan.chunk_blocks);
    plan.bytes = sizeof(float) * static_cast<size_t>(batch) * q_heads * plan.splits * (dim_v + 2);
    return plan;
}

Partials step_partials(const StepPlan& plan, int batch, int q_heads, int dim_v, void* workspace) {
    float* ws = static_cast<float*>(workspace);
    if (!plan.mma) return {ws, ws + 2, nullptr, plan.splits, dim_v + 2, dim_v + 2};
    const size_t pieces = static_cast<size_t>(plan.ctas + plan.pairs) * kPieceHeads;
    char* span = reinterpret_cast<char*>(ws) + round_up16(sizeof(float) * (2 + dim_v) * pieces);
    return {ws + pieces * dim_v, ws, reinterpret_cast<int2*>(span), 0, 2, dim_v};
}

sfb_status step_attention(const StepParams& p, const StepPlan& plan, int dtype, cudaStream_t stream) {
    if (plan.mma) return step_mma(p, plan, stream);
    return dtype == SFB_F32 ? step_typed<float>(p, stream) : step_typed<bf16>(p, stream);
}

sfb_status merge_partials(const MergeParams& p, int dtype, cudaStream_t stream) {
    // a CTA per row while that leaves at most four per SM (all pieces in flight at once), else a warp per row
    const int64_t rows = static_cast<int64_t>(p.batch) * p.q_heads * p.nodes;
    if (rows > 4LL * sm_count()) {
        const dim3 grid(static_cast<unsigned>(ceil_div64(rows, 8)));
        if (dtype == SFB_F32) SFB_CUDA(launch_dependent(merge_rows_kernel<float>, grid, dim3(256), 0, stream, p, static_cast<int>(rows)));
        else SFB_CUDA(launch_dependent(merge_rows_kernel<bf16>, grid, dim3(256), 0, stream, p, static_cast<int>(rows)));
        return check_launch("attention_merge");
    }
    const dim3 grid(static_cast<unsigned>(rows));
    if (dtype == SFB_F32) SFB_CUDA(launch_dependent(merge_kernel<float>, grid, dim3(256), 0, stream, p));
    else SFB_CUDA(launch_dependent(merge_kernel<bf16>, grid, dim3(256), 0, stream, p));
    return check_launch("attention_merge");
}

}  // namespace sfb
