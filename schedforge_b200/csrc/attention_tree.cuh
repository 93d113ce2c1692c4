// Parameters and the ancestor table shared by the tree-attention kernels.
#pragma once

#include "cache_ops.cuh"

namespace sfb {

struct TreeParams {
    PagedView kv;
    const void *q, *draft_k, *draft_v;
    const int *parents, *node_count;
    void* out;
    float* partials;
    int batch, q_heads, nodes, token_major, splits, chunk, vec;
    float scale_log2;
};

// float32, head dimensions that are multiples of 8 up to 128 (attention_tree_tf32.cu); the same layout of splits as the
// CUDA-core kernel, with row tiles of 128.
bool tree_tf32_shape(const sfb_tree_args& a);
sfb_status tree_tf32(const TreeParams& p, cudaStream_t stream);

// bf16, head_dim = head_dim_value = 128 or 64 (attention_tree_tcgen05.cu).
bool tree_tcgen05_shape(const sfb_tree_args& a);        // types and sizes
bool tree_tcgen05_supported(const sfb_tree_args& a);    // and addresses
size_t tree_tcgen05_workspace(const sfb_tree_args& a);
sfb_status tree_tcgen05(const sfb_tree_args& a, const TreeParams& t, cudaStream_t stream);

#ifdef __CUDACC__
__device__ __forceinline__ int tree_node_count(const TreeParams& p, int b) {
    if (!p.node_count) return p.nodes;
    int n = p.node_count[b];
    if (n < 0 || n > p.nodes) {
        n = n < 0 ? 0 : p.nodes;
        if (threadIdx.x == 0) atomicOr(p.kv.status, kCodeDecodeBounds);
    }
    return n;
}

// Context length and node count of a sequence, both loads in flight together.
__device__ __forceinline__ void tree_sizes(const TreeParams& p, int b, int& ctx, int& count, bool report) {
    const int length = p.kv.lens[b], nodes = p.node_count ? p.node_count[b] : p.nodes;
    ctx = min(max(length, 0), p.kv.limit);
    count = min(max(nodes, 0), p.nodes);
    if (report && (ctx != length || count != nodes)) atomicOr(p.kv.status, kCodeDecodeBounds);
}

__device__ __forceinline__ size_t tree_out_row(const TreeParams& p, int b, int head, int node) {
    return p.token_major ? (static_cast<size_t>(b) * p.nodes + node) * p.q_heads + head
                         : (static_cast<size_t>(b) * p.q_heads + head) * p.nodes + node;
}

// seen[8 * i + w]: bit j % 32 of word j / 32 says that node i sees node j (itself and its ancestors).  Parents are
// smaller than their children, so every walk ends.  All threads of the CTA call it; seen is ready after their next
// __syncthreads().
__device__ __forceinline__ void tree_ancestors(const TreeParams& p, int b, int count, int* parent, uint32_t* seen) {
    for (int i = threadIdx.x; i < p.nodes; i += blockDim.x) {
        int up = i < count ? p.parents[static_cast<size_t>(b) * p.nodes + i] : -1;
        if (up < -1 || up >= i) {
            up = -1;
            atomicOr(p.kv.status, kCodeDecodeBounds);
        }
        parent[i] = up;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.nodes; i += blockDim.x) {
        uint32_t words[8] = {};
        for (int j = i < count ? i : -1; j >= 0; j = parent[j]) {
#pragma unroll
            for (int w = 0; w < 8; ++w)
                if (w == j >> 5) words[w] |= 1u << (j & 31);
        }
#pragma unroll
        for (int w = 0; w < 8; ++w) seen[8 * i + w] = words[w];
    }
}
#endif

}  // namespace sfb
