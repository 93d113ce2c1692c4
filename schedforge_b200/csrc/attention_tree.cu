// Attention of a tree of drafted tokens over a paged cache: the entry point, the split rule and the CUDA-core kernel
// (float32, and bf16 with head dimensions the tensor-core kernel does not take).
//
// The query rows of one (sequence, K/V head) are the group's heads times the nodes, contiguous in memory.  The keys are
// the committed positions followed by the drafted nodes; a row sees all of the first and its ancestors of the second,
// kept as one bit per (node, node).  A CTA takes 64 rows and a range of keys (split) in tiles of 64 keys: scores and
// products as register-blocked 4x4 outer products out of shared memory, online softmax per row, partial results of the
// splits merged afterwards.
#include "attention_tree.cuh"

namespace sfb {
namespace {

constexpr int BM = 64, BN = 64, kThreads = 256;
constexpr int kPStride = BN + 4;

__host__ __device__ inline int padded(int dim) { return ((dim + 3) & ~3) + 4; }  // floats per Q / K row in shared memory

size_t tree_smem(int dim, int nv) {
    return sizeof(float) * (static_cast<size_t>(BM + BN) * padded(dim) + static_cast<size_t>(BN) * nv * 64 + static_cast<size_t>(BM) * kPStride) +
           sizeof(uint32_t) * 8 * SFB_MAX_TREE_NODES + sizeof(int) * SFB_MAX_TREE_NODES;
}

// Loads `rows` rows of dim elements into [64][stride] floats, zero beyond; row(r) gives the element offset or -1.
template <class T, class Row>
__device__ __forceinline__ void load_tile(float* dst, int stride, const T* src, int dim, bool vec, float factor, Row row) {
    const int width = (dim + 3) & ~3;
    for (int i = threadIdx.x; i < 64 * (width / 4); i += kThreads) {
        const int r = i / (width / 4), d = (i % (width / 4)) * 4;
        const int64_t at = row(r);
        float v[4] = {0.0F, 0.0F, 0.0F, 0.0F};
        if (at >= 0) {
            const T* p = src + at * dim + d;
            if (vec) {
                if constexpr (sizeof(T) == 4) {
                    const float4 f = *reinterpret_cast<const float4*>(p);
                    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
                } else {
                    const uint2 f = *reinterpret_cast<const uint2*>(p);
                    v[0] = __uint_as_float(f.x << 16); v[1] = __uint_as_float(f.x & 0xffff0000u);
                    v[2] = __uint_as_float(f.y << 16); v[3] = __uint_as_float(f.y & 0xffff0000u);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (d + j < dim) v[j] = to_float(p[j]);
            }
        }
        *reinterpret_cast<float4*>(dst + r * stride + d) = make_float4(v[0] * factor, v[1] * factor, v[2] * factor, v[3] * factor);
    }
}

template <class T, int NV>
__global__ void __launch_bounds__(kThreads)
tree_simt_kernel(const __grid_constant__ TreeParams p) {
    extern __shared__ float4 tree_smem_raw[];
    const PagedView& kv = p.kv;
    const int stride = padded(kv.dim);
    float* qs = reinterpret_cast<float*>(tree_smem_raw);   // [BM][stride]
    float* ks = qs + BM * stride;                          // [BN][stride]
    float* vs = ks + BN * stride;                          // [BN][NV * 64]
    float* ps = vs + BN * NV * 64;                         // [BM][kPStride]
    uint32_t* seen = reinterpret_cast<uint32_t*>(ps + BM * kPStride);  // [nodes][8]
    int* parent = reinterpret_cast<int*>(seen + 8 * SFB_MAX_TREE_NODES);
    const int group = p.q_heads / kv.kv_heads, rows_all = group * p.nodes;
    const int row_tiles = (rows_all + BM - 1) / BM;
    const int tile = blockIdx.x % row_tiles, split = blockIdx.x / row_tiles;
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    grid_dependents_may_launch();
    grid_dependency_wait();
    const int ctx = kv.length(b);
    const int count = tree_node_count(p, b);
    const int keys = ctx + count;
    const int k0 = min(keys, split * p.chunk), k1 = split == p.splits - 1 ? keys : min(keys, k0 + p.chunk);
    const int row0 = tile * BM;
    const bool has_draft = k1 > ctx;
    if (has_draft) tree_ancestors(p, b, count, parent, seen);
    const T* q = static_cast<const T*>(p.q) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * rows_all * kv.dim;
    load_tile(qs, stride, q, kv.dim, p.vec, p.scale_log2, [&](int r) -> int64_t { return row0 + r < rows_all ? row0 + r : -1; });

    float o[4][NV * 4], m[4], l[4];
    int node[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0F;
        node[i] = (row0 + ty * 4 + i) % p.nodes;
#pragma unroll
        for (int j = 0; j < NV * 4; ++j) o[i][j] = 0.0F;
    }
    const T* draft_k = static_cast<const T*>(p.draft_k) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.nodes * kv.dim;
    const T* draft_v = static_cast<const T*>(p.draft_v) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.nodes * kv.dim_v;
    for (int t0 = k0; t0 < k1; t0 += BN) {
        __syncthreads();
        // committed rows come from the pool, drafted ones from their own tensors; a tile may hold both
        const int from_pool = min(max(ctx - t0, 0), BN), live = min(BN, k1 - t0);
        const auto pool_row = [&](int r) -> int64_t { return r < min(from_pool, live) ? kv.row(b, kvh, t0 + r) : -1; };
        if (from_pool > 0) {
            load_tile(ks, stride, static_cast<const T*>(kv.k_pool), kv.dim, p.vec, 1.0F, pool_row);
            load_tile(vs, NV * 64, static_cast<const T*>(kv.v_pool), kv.dim_v, p.vec, 1.0F, pool_row);
        }
        if (from_pool < live) {
            if (from_pool > 0) __syncthreads();
            const auto draft_row = [&](int r) -> int64_t { return r >= from_pool && r < live ? t0 + r - ctx : -2; };
            // (-2 in a mixed tile: the row was loaded above and must stay)
            const auto mixed = [&](float* dst, int st, const T* src, int dim) {
                const int width = (dim + 3) & ~3;
                for (int i = threadIdx.x; i < 64 * (width / 4); i += kThreads) {
                    const int r = i / (width / 4), d = (i % (width / 4)) * 4;
                    const int64_t at = draft_row(r);
                    if (at == -2 && r < from_pool) continue;
                    float v[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = at >= 0 && d + j < dim ? to_float(src[at * dim + d + j]) : 0.0F;
                    *reinterpret_cast<float4*>(dst + r * st + d) = make_float4(v[0], v[1], v[2], v[3]);
                }
            };
            mixed(ks, stride, draft_k, kv.dim);
            mixed(vs, NV * 64, draft_v, kv.dim_v);
        }
        __syncthreads();
        float s[4][4] = {};
        for (int d = 0; d < kv.dim; d += 4) {
            float4 qa[4], ka[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) qa[i] = *reinterpret_cast<const float4*>(qs + (ty * 4 + i) * stride + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) ka[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * stride + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = fmaf(qa[i].x, ka[j].x, s[i][j]);
                    s[i][j] = fmaf(qa[i].y, ka[j].y, s[i][j]);
                    s[i][j] = fmaf(qa[i].z, ka[j].z, s[i][j]);
                    s[i][j] = fmaf(qa[i].w, ka[j].w, s[i][j]);
                }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int key = t0 + tx + 16 * j;
            const bool inside = key < k1;
            const bool draft = key >= ctx;
            const bool there = inside && (draft || kv.row(b, kvh, key) >= 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool visible = there && (!draft || (seen[node[i] * 8 + ((key - ctx) >> 5)] >> ((key - ctx) & 31) & 1u));
                if (!visible) s[i][j] = -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
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
                ps[(ty * 4 + i) * kPStride + tx + 16 * j] = e;
            }
        }
        __syncthreads();
        for (int k = 0; k < live; ++k) {
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = ps[(ty * 4 + i) * kPStride + k];
#pragma unroll
            for (int c = 0; c < NV; ++c) {
                const float4 v = *reinterpret_cast<const float4*>(vs + k * NV * 64 + c * 64 + tx * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[i][c * 4] = fmaf(e[i], v.x, o[i][c * 4]);
                    o[i][c * 4 + 1] = fmaf(e[i], v.y, o[i][c * 4 + 1]);
                    o[i][c * 4 + 2] = fmaf(e[i], v.z, o[i][c * 4 + 2]);
                    o[i][c * 4 + 3] = fmaf(e[i], v.w, o[i][c * 4 + 3]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int w = 1; w < 16; w <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
        const int r = row0 + ty * 4 + i;
        if (r >= rows_all || node[i] >= count) continue;
        const size_t row = (static_cast<size_t>(b) * kv.kv_heads + kvh) * rows_all + r;
        if (p.splits == 1) {
            const float inv = l[i] > 0.0F ? 1.0F / l[i] : (l[i] == 0.0F ? 0.0F : l[i]);
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
    const size_t smem = tree_smem(p.kv.dim, NV);
    SFB_CUDA(cudaFuncSetAttribute(tree_simt_kernel<T, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    const int rows = p.q_heads / p.kv.kv_heads * p.nodes;
    const dim3 grid(ceil_div(rows, BM) * p.splits, p.kv.kv_heads, p.batch);
    SFB_CUDA(launch_dependent(tree_simt_kernel<T, NV>, grid, dim3(kThreads), smem, stream, p));
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

// Splits of the key axis: tiles of 64 keys, as many splits as fill the GPU about twice, no split below 256 keys.
TreeLayout tree_layout(const sfb_tree_args& a) {
    TreeLayout l{};
    const int covered = a.max_blocks * a.block_tokens;
    const int limit = (a.max_context < covered ? a.max_context : covered) + a.nodes;
    const int64_t base = static_cast<int64_t>(a.batch) * a.kv_heads * ceil_div(a.q_heads / a.kv_heads * a.nodes, BM);
    int splits = a.splits;
    if (splits <= 0) {
        const int64_t wanted = (2LL * sm_count() + base - 1) / base;
        const int most = ceil_div(limit, 256);
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
    if (static_cast<int64_t>(a->q_heads) * a->nodes > (1 << 24)) return fail(SFB_UNSUPPORTED, "tree attention: more than 2^24 query rows per sequence");
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
    p.vec = a->head_dim % 4 == 0 && a->head_dim_value % 4 == 0 && aligned16(a->q) && aligned16(a->k_pool) && aligned16(a->v_pool);
    if (tensor) return tree_tcgen05(*a, p, s);
    SFB_TRY(a->dtype == SFB_F32 ? tree_simt<float>(p, s) : tree_simt<bf16>(p, s));
    if (l.splits == 1) return SFB_OK;
    const Partials part{p.partials, p.partials + 2, nullptr, l.splits, a->head_dim_value + 2, a->head_dim_value + 2};
    return merge_partials({part, p.kv, a->out, a->node_count, a->batch, a->q_heads, a->nodes, a->head_dim_value, a->token_major}, a->dtype, s);
}

}  // extern "C"
