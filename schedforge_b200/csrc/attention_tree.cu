// Attention of a tree of drafted tokens over a paged cache: the entry point, the split rule and the CUDA-core kernel (types,
// head dimensions and alignments that the tensor-core kernels do not take).
//
// The query rows of one (sequence, K/V head) are the group's heads times the nodes, contiguous in memory.  The keys are
// the committed positions followed by the drafted nodes; a row sees all of the first and its ancestors of the second,
// kept as one bit per (node, node).  A CTA takes 64 rows and a range of keys (split) in tiles of 64 keys.  Scores and
// products are register-blocked outer products out of shared memory: a thread has 8 rows (4 where the value dimension
// is above 128) and 4 keys, so a four-element step costs 12 wide shared-memory reads for 128 multiply-adds, and the
// fp32 pipe is the bound, not the reads.  A row belongs to 16 lanes of one warp, which exchange its maximum by shuffles.
#include "attention_tree.cuh"

namespace sfb {
namespace {

constexpr int BM = 64, BN = 64;
constexpr int kPStride = BN + 4;

template <int NV> struct TreeTile {
    static constexpr int kRows = NV <= 2 ? 8 : 4;             // query rows of a thread
    static constexpr int kThreads = BM / kRows * 16;
};

__host__ __device__ inline int padded(int dim) { return ((dim + 3) & ~3) + 4; }  // floats per Q / K row in shared memory

size_t tree_smem(int dim, int nv, int nodes) {
    return sizeof(float) * (static_cast<size_t>(BM + BN) * padded(dim) + static_cast<size_t>(BN) * nv * 64 + static_cast<size_t>(BM) * kPStride) +
           4 * sizeof(void*) * BN + sizeof(uint32_t) * 9 * nodes;
}

template <class T>
__device__ __forceinline__ float4 load4(const T* p, int left, bool vec) {
    if (vec) {
        if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float4*>(p);
        else {
            const uint2 f = *reinterpret_cast<const uint2*>(p);
            return make_float4(__uint_as_float(f.x << 16), __uint_as_float(f.x & 0xffff0000u), __uint_as_float(f.y << 16),
                               __uint_as_float(f.y & 0xffff0000u));
        }
    }
    return make_float4(to_float(p[0]), left > 1 ? to_float(p[1]) : 0.0F, left > 2 ? to_float(p[2]) : 0.0F, left > 3 ? to_float(p[3]) : 0.0F);
}

// 64 rows of dim elements into [64][stride] floats, zero where row(r) is nullptr and behind the row's end.  ASYNC
// (float32, 16-byte aligned rows, factor 1): by cp.async, to be waited for.
template <int THREADS, class T, bool ASYNC, class Row>
__device__ __forceinline__ void load_tile(float* dst, int stride, int dim, int width, bool vec, float factor, Row row) {
    const int pieces = width / 4;
    if constexpr (ASYNC && sizeof(T) == 4) {
        if (vec) {
#pragma unroll 8
            for (int i = threadIdx.x; i < 64 * pieces; i += THREADS) {
                const int r = i / pieces, d = (i - r * pieces) * 4;
                const T* src = row(r);
                const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(dst + r * stride + d));
                if (src && d < dim) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(src + d) : "memory");
                else *reinterpret_cast<float4*>(dst + r * stride + d) = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
            }
            return;
        }
    }
#pragma unroll 8
    for (int i = threadIdx.x; i < 64 * pieces; i += THREADS) {
        const int r = i / pieces, d = (i - r * pieces) * 4;
        const T* src = row(r);
        float4 v = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
        if (src && d < dim) v = load4(src + d, dim - d, vec);
        *reinterpret_cast<float4*>(dst + r * stride + d) = make_float4(v.x * factor, v.y * factor, v.z * factor, v.w * factor);
    }
}

template <class T, int NV>
__global__ void __launch_bounds__(TreeTile<NV>::kThreads)
tree_simt_kernel(const __grid_constant__ TreeParams p) {
    constexpr int kThreads = TreeTile<NV>::kThreads, R = TreeTile<NV>::kRows;
    extern __shared__ float4 tree_smem_raw[];
    const PagedView& kv = p.kv;
    const int stride = padded(kv.dim);
    float* qs = reinterpret_cast<float*>(tree_smem_raw);   // [BM][stride]
    float* ks = qs + BM * stride;                          // [BN][stride]
    float* vs = ks + BN * stride;                          // [BN][NV * 64]
    float* ps = vs + BN * NV * 64;                         // [BM][kPStride]
    const T** k_rows = reinterpret_cast<const T**>(ps + BM * kPStride);   // [2][BN] rows of this and the next tile, nullptr: masked
    const T** v_rows = k_rows + 2 * BN;
    uint32_t* seen = reinterpret_cast<uint32_t*>(v_rows + 2 * BN);        // [nodes][8]
    int* parent = reinterpret_cast<int*>(seen + 8 * p.nodes);
    const int group = p.q_heads / kv.kv_heads, rows_all = group * p.nodes;
    const int row_tiles = (rows_all + BM - 1) / BM;
    const int tile = blockIdx.x % row_tiles, split = blockIdx.x / row_tiles;
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    grid_dependency_wait();
    const int ctx = kv.length(b);
    const int count = tree_node_count(p, b);
    const int keys = ctx + count;
    const int k0 = min(keys, split * p.chunk), k1 = split == p.splits - 1 ? keys : min(keys, k0 + p.chunk);
    const int row0 = tile * BM;
    if (k0 >= k1) return;     // (an empty split leaves no piece)
    if (k1 > ctx) tree_ancestors(p, b, count, parent, seen);
    const T* q = static_cast<const T*>(p.q) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * rows_all * kv.dim;
    load_tile<kThreads, T, false>(qs, stride, kv.dim, (kv.dim + 3) & ~3, p.vec, p.scale_log2,
                           [&](int r) { return row0 + r < rows_all ? q + static_cast<size_t>(row0 + r) * kv.dim : nullptr; });
    float o[R][NV * 4], m[R], l[R];
    int node[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0F;
        node[i] = (row0 + ty * R + i) % p.nodes;
#pragma unroll
        for (int j = 0; j < NV * 4; ++j) o[i][j] = 0.0F;
    }
    const T* draft_k = static_cast<const T*>(p.draft_k) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.nodes * kv.dim;
    const T* draft_v = static_cast<const T*>(p.draft_v) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.nodes * kv.dim_v;
    // committed rows come from the pool, drafted ones from their own tensors
    const auto find_rows = [&](int t0, int buffer) {
        if (threadIdx.x >= BN) return;
        const int key = t0 + threadIdx.x;
        const T *kr = nullptr, *vr = nullptr;
        if (key < min(k1, ctx)) {
            const int64_t at = kv.row(b, kvh, key);
            if (at >= 0) {
                kr = static_cast<const T*>(kv.k_pool) + at * kv.dim;
                vr = static_cast<const T*>(kv.v_pool) + at * kv.dim_v;
            }
        } else if (key < k1) {
            kr = draft_k + static_cast<size_t>(key - ctx) * kv.dim;
            vr = draft_v + static_cast<size_t>(key - ctx) * kv.dim_v;
        }
        k_rows[buffer * BN + threadIdx.x] = kr;
        v_rows[buffer * BN + threadIdx.x] = vr;
    };
    // K of the next tile is fetched under the softmax and the P.V of this one, V under the scores of the next
    const auto fetch_k = [&](int buffer) {
        load_tile<kThreads, T, true>(ks, stride, kv.dim, (kv.dim + 3) & ~3, p.vec, 1.0F, [&](int r) { return k_rows[buffer * BN + r]; });
    };
    const auto fetch_v = [&](int buffer) {
        load_tile<kThreads, T, true>(vs, NV * 64, kv.dim_v, NV * 64, p.vec, 1.0F, [&](int r) { return v_rows[buffer * BN + r]; });
    };
    const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    const auto wait_but_one = [] { asm volatile("cp.async.wait_group 1;" ::: "memory"); };
    {
        find_rows(k0, 0);
        __syncthreads();
        fetch_k(0);
        commit();
        fetch_v(0);
        commit();
    }
    int buffer = 0;
    for (int t0 = k0; t0 < k1; t0 += BN, buffer ^= 1) {
        const bool more = t0 + BN < k1;
        if (more) find_rows(t0 + BN, buffer ^ 1);
        wait_but_one();      // K
        __syncthreads();
        float s[R][4] = {};
#pragma unroll 2
        for (int d = 0; d < kv.dim; d += 4) {
            float4 ka[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) ka[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * stride + d);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const float4 qa = *reinterpret_cast<const float4*>(qs + (ty * R + i) * stride + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = fmaf(qa.x, ka[j].x, s[i][j]);
                    s[i][j] = fmaf(qa.y, ka[j].y, s[i][j]);
                    s[i][j] = fmaf(qa.z, ka[j].z, s[i][j]);
                    s[i][j] = fmaf(qa.w, ka[j].w, s[i][j]);
                }
            }
        }
        if (t0 + BN > ctx || t0 + BN > k1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = t0 + tx + 16 * j;
#pragma unroll
                for (int i = 0; i < R; ++i)
                    if (key >= k1 || (key >= ctx && !(seen[node[i] * 8 + ((key - ctx) >> 5)] >> ((key - ctx) & 31) & 1u))) s[i][j] = -INFINITY;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (!k_rows[buffer * BN + tx + 16 * j])
#pragma unroll
                for (int i = 0; i < R; ++i) s[i][j] = -INFINITY;
        __syncthreads();
        if (more) fetch_k(buffer ^ 1);
        commit();
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float top = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            top = fmaxf(top, m[i]);
            const float alpha = top == -INFINITY ? 1.0F : exp2f(m[i] - top);
            m[i] = top;
            l[i] *= alpha;
#pragma unroll
            for (int j = 0; j < NV * 4; ++j) o[i][j] *= alpha;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float e = s[i][j] == -INFINITY ? 0.0F : exp2f(s[i][j] - top);
                l[i] += e;   // this lane's share of the row sum
                ps[(ty * R + i) * kPStride + tx + 16 * j] = e;
            }
        }
        wait_but_one();      // V
        __syncthreads();
#pragma unroll 2
        for (int k = 0; k < BN; k += 4) {
            float4 e[R];
#pragma unroll
            for (int i = 0; i < R; ++i) e[i] = *reinterpret_cast<const float4*>(ps + (ty * R + i) * kPStride + k);
#pragma unroll
            for (int c = 0; c < NV; ++c)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float4 v = *reinterpret_cast<const float4*>(vs + (k + u) * NV * 64 + c * 64 + tx * 4);
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        const float w = u == 0 ? e[i].x : u == 1 ? e[i].y : u == 2 ? e[i].z : e[i].w;
                        o[i][c * 4] = fmaf(w, v.x, o[i][c * 4]);
                        o[i][c * 4 + 1] = fmaf(w, v.y, o[i][c * 4 + 1]);
                        o[i][c * 4 + 2] = fmaf(w, v.z, o[i][c * 4 + 2]);
                        o[i][c * 4 + 3] = fmaf(w, v.w, o[i][c * 4 + 3]);
                    }
                }
        }
        __syncthreads();
        if (more) fetch_v(buffer ^ 1);
        commit();
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int w = 1; w < 16; w <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
        const int r = row0 + ty * R + i;
        if (r >= rows_all || node[i] >= count) continue;
        const size_t row = (static_cast<size_t>(b) * kv.kv_heads + kvh) * rows_all + r;
        if (p.splits == 1) {
            const float inv = l[i] == 0.0F ? 0.0F : 1.0F / l[i];
            T* dst = static_cast<T*>(p.out) + tree_out_row(p, b, kvh * group + r / p.nodes, node[i]) * kv.dim_v;
#pragma unroll
            for (int c = 0; c < NV; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c * 64 + tx * 4 + j < kv.dim_v) dst[c * 64 + tx * 4 + j] = from_float<T>(o[i][c * 4 + j] * inv);
        } else {
            float* rec = p.partials + (row * p.splits + split) * (kv.dim_v + 2);
            if (tx == 0) { rec[0] = m[i]; rec[1] = l[i]; }
#pragma unroll
            for (int c = 0; c < NV; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c * 64 + tx * 4 + j < kv.dim_v) rec[2 + c * 64 + tx * 4 + j] = o[i][c * 4 + j];
        }
    }
}

template <class T, int NV>
sfb_status launch_tree(const TreeParams& p, cudaStream_t stream) {
    const size_t smem = tree_smem(p.kv.dim, NV, p.nodes);
    // (the same limit for every shape, since another thread may be launching the kernel)
    static const int most = static_cast<int>(tree_smem(256, NV, SFB_MAX_TREE_NODES));
    SFB_CUDA(cudaFuncSetAttribute(tree_simt_kernel<T, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    const int rows = p.q_heads / p.kv.kv_heads * p.nodes;
    const dim3 grid(ceil_div(rows, BM) * p.splits, p.kv.kv_heads, p.batch);
    SFB_CUDA(launch_dependent(tree_simt_kernel<T, NV>, grid, dim3(TreeTile<NV>::kThreads), smem, stream, p));
    return check_launch("attention_tree");
}

template <class T>
sfb_status tree_simt(const TreeParams& p, cudaStream_t stream) {
    switch (ceil_div(p.kv.dim_v, 64)) {
        case 1: return launch_tree<T, 1>(p, stream);
        case 2: return launch_tree<T, 2>(p, stream);
        case 3: return launch_tree<T, 3>(p, stream);
        default: return launch_tree<T, 4>(p, stream);
    }
}

struct TreeLayout {
    int splits, chunk;
    size_t total;
};

// Splits of the key axis: tiles of 64 keys, about four CTAs per SM, at least one tile each (at least two: 24 us instead of
// 19 for one float32 sequence of 1500 tokens, 39 instead of 26 on the CUDA cores).  Two CTAs per SM, what the float32 kernel
// holds at once, are better without raggedness (54 -> 47 us at 16 such sequences) and worse with it (36 -> 43).
TreeLayout tree_layout(const sfb_tree_args& a) {
    TreeLayout l{};
    const int covered = a.max_blocks * a.block_tokens;
    const int limit = (a.max_context < covered ? a.max_context : covered) + a.nodes;
    const int64_t base = static_cast<int64_t>(a.batch) * a.kv_heads * ceil_div(a.q_heads / a.kv_heads * a.nodes, tree_tf32_shape(a) ? 128 : BM);
    int splits = a.splits;
    if (splits <= 0) {
        const int64_t wanted = (4LL * sm_count() + base - 1) / base;
        const int most = ceil_div(limit, BN);
        splits = static_cast<int>(wanted < most ? wanted : most);
    }
    if (splits > 128) splits = 128;
    if (splits < 1) splits = 1;
    l.chunk = ceil_div(ceil_div(limit, splits), BN) * BN;
    l.splits = ceil_div(limit, l.chunk);
    l.total = l.splits == 1 ? 0 : sizeof(float) * static_cast<size_t>(a.batch) * a.q_heads * a.nodes * l.splits * (a.head_dim_value + 2);
    return l;
}

sfb_status check_tree(const sfb_tree_args* a) {
    SFB_REQUIRE(a, "tree attention: null arguments");
    SFB_TRY(check_cache(a->k_pool, a->v_pool, a->block_table, a->batch, a->kv_heads, a->head_dim, a->head_dim_value,
                        a->block_tokens, a->max_blocks, a->num_blocks, a->dtype, "tree attention"));
    SFB_REQUIRE(a->q_heads > 0 && a->q_heads % a->kv_heads == 0, "invalid grouped-query attention configuration");
    SFB_REQUIRE(a->nodes > 0, "tree attention: no nodes");
    SFB_REQUIRE(a->max_context >= 0, "tree attention: negative max_context");
    if (a->nodes > SFB_MAX_TREE_NODES) return fail(SFB_UNSUPPORTED, "tree attention: more than 256 nodes");
    if (static_cast<int64_t>(a->batch) * a->q_heads * a->nodes > (1 << 28)) return fail(SFB_UNSUPPORTED, "tree attention: more than 2^28 query rows");
    return SFB_OK;
}

}  // namespace
}  // namespace sfb

using namespace sfb;

extern "C" {

size_t sfb_attention_tree_workspace(const sfb_tree_args* a) {
    if (check_tree(a) != SFB_OK) return 0;
    const size_t simt = tree_layout(*a).total;
    const size_t tensor = tree_tcgen05_shape(*a) ? tree_tcgen05_workspace(*a) : 0;   // (the addresses may not be set yet)
    return tensor > simt ? tensor : simt;
}

sfb_status sfb_k_attention_tree_paged(const sfb_tree_args* a, sfb_stream stream) {
    SFB_TRY(check_tree(a));
    SFB_REQUIRE(a->q && a->context_len && a->draft_k && a->draft_v && a->parents && a->out, "tree attention: null tensor");
    const TreeLayout l = tree_layout(*a);
    const bool tensor = tree_tcgen05_supported(*a);
    SFB_REQUIRE((l.total == 0 && !tensor) || (a->workspace && aligned16(a->workspace)), "tree attention: the workspace is missing or not 16-byte aligned");
    cudaStream_t s = as_stream(stream);
    TreeParams p{};
    p.kv = make_view(a->k_pool, a->v_pool, a->block_table, a->context_len, a->kv_heads, a->head_dim, a->head_dim_value,
                     a->block_tokens, a->max_blocks, a->num_blocks, a->max_context);
    p.q = a->q; p.draft_k = a->draft_k; p.draft_v = a->draft_v; p.parents = a->parents; p.node_count = a->node_count;
    p.out = a->out; p.partials = static_cast<float*>(a->workspace);
    p.batch = a->batch; p.q_heads = a->q_heads; p.nodes = a->nodes; p.token_major = a->token_major;
    p.splits = l.splits; p.chunk = l.chunk;
    p.scale_log2 = (a->scale > 0.0F ? a->scale : 1.0F / sqrtf(static_cast<float>(a->head_dim))) * 1.4426950408889634F;
    p.vec = a->head_dim % 4 == 0 && a->head_dim_value % 4 == 0 && aligned16(a->q) && aligned16(a->k_pool) && aligned16(a->v_pool) && aligned16(a->draft_k) &&
            aligned16(a->draft_v);
    if (tensor) return tree_tcgen05(*a, p, s);
    if (p.vec && aligned16(a->out) && tree_tf32_shape(*a)) SFB_TRY(tree_tf32(p, s));
    else SFB_TRY(a->dtype == SFB_F32 ? tree_simt<float>(p, s) : tree_simt<bf16>(p, s));
    if (l.splits == 1) return SFB_OK;
    const Partials part{p.partials, p.partials + 2, nullptr, l.splits, a->head_dim_value + 2, a->head_dim_value + 2};
    return merge_partials({part, p.kv, a->out, a->node_count, a->batch, a->q_heads, a->nodes, a->head_dim_value, a->token_major, l.chunk}, a->dtype, s);
}

}  // extern "C"
