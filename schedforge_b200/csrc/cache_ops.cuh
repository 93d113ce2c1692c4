// Shared pieces of the serving operators over the paged cache: guarded cache access, the split bookkeeping of the
// decode kernels and the merge of their partial results.
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
    __device__ __forceinline__ int64_t row(int b, int head, int position) const {
        const int block = block_of(position);
        const int page = table[static_cast<size_t>(b) * max_blocks + block];
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

// ---- one query token per sequence --------------------------------------------------------------------------------
// Attention of the query heads of one K/V head over the blocks of a list (selected != nullptr) or over the whole
// context.  Split s of a (sequence, K/V head) covers list entries [s * chunk_blocks, (s + 1) * chunk_blocks) and leaves
// (maximum, sum, numerator) in partials; maxima and logits are in base-2 units.  logits != nullptr: the scaled logit of
// every position is kept there.
struct StepParams {
    PagedView kv;
    const void* q;
    void* out;
    float* partials;
    float* logits;          // [batch, q_heads, logit_stride]
    const int* selected;    // [batch, kv_heads, budget]
    int64_t logit_stride;
    int budget;
    int batch, q_heads, splits, chunk_blocks;
    float scale_log2;
};

bool step_mma_supported(const StepParams& p, int dtype);   // attention_step_mma.cu
sfb_status step_mma(const StepParams& p, cudaStream_t stream);
sfb_status step_attention(const StepParams& p, int dtype, cudaStream_t stream);
int step_splits(int batch, int kv_heads, int tokens, int block_tokens, int wanted, int* chunk_blocks);

// ---- merge of split partials ---------------------------------------------------------------------------------------
// Rows are (b, q_head, node); nodes == 1 and node_count == nullptr for single-token decode.
struct MergeParams {
    const float* partials;  // [rows][splits][dim_v + 2]
    void* out;
    const int* node_count;
    int batch, q_heads, nodes, dim_v, splits, token_major;
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
#endif

}  // namespace sfb
