// Tree attention in float32 on the warp-level tensor path (head dimensions up to 128, multiples of 8, 16-byte aligned).
//
// A float32 value is split into two TF32 parts, x = hi + lo with hi the upper 11 bits of the significand and lo the
// next 11, and a product is hi hi + hi lo + lo hi, accumulated in 32 bits: what is dropped is 2^-22 of each term, a quarter of the
// rounding of a float32 sum of sixteen.  Three m16n8k8 products replace 32 multiply-adds a lane, so the instruction
// count falls to a fifth of the CUDA-core form (attention_tree.cu), which had no issue slots left to cover its
// loads (16 sequences of up to 1500 tokens, 27 nodes, 64-dimensional heads: 68 us there).
// A CTA takes 128 query rows of one (sequence, K/V head) and a split of the keys in tiles of 64.  A warp owns 32 rows (16
// where a head dimension is above 64); P goes through its own part of shared memory, so that both products are rolled loops:
// fully unrolled they spent a third of the time waiting for instructions.  K of the next tile is fetched (cp.async) under the softmax and P.V of this one, V under the scores of the next.
#include "attention_tree.cuh"

namespace sfb {
namespace {

constexpr int BN = 64, BM = 128;

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// hi is x rounded to 11 bits, so that of the 12 bits and the sign of lo the instruction, which reads the upper 19 bits
// of a register, drops one at most.
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}

// acc(t, n) += the products of four column tiles n and all row tiles t over `steps` steps of eight, operands from
// a(step, t, hi, lo) and b(step, n, hi, lo).  The instruction truncates its sums, so the large products run at most DEPTH
// steps in an accumulator of their own before a rounded addition takes them over, and the small ones, which have 11 bits to
// spare, meet them at the end.  (All three products in one accumulator running on over the tiles: 2.6e-6 off at logits of ten.)
// Products of one accumulator are at least 4 * M instructions apart, since each waits for the one before.
template <int M, int DEPTH, class Acc, class A, class B>
__device__ __forceinline__ void multiply(Acc acc, int steps, A a, B b) {
    float small[M][4][4];
#pragma unroll
    for (int t = 0; t < M; ++t)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) small[t][n][i] = 0.0F;
#pragma unroll 1
    for (int step0 = 0; step0 < steps; step0 += DEPTH) {
        float big[M][4][4];
#pragma unroll
        for (int t = 0; t < M; ++t)
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) big[t][n][i] = 0.0F;
#pragma unroll
        for (int u = 0; u < DEPTH; ++u) {
            const int step = step0 + u;
            if (step >= steps) continue;
            uint32_t ah[M][4], al[M][4], bh[4][2], bl[4][2];
#pragma unroll
            for (int t = 0; t < M; ++t) a(step, t, ah[t], al[t]);
#pragma unroll
            for (int n = 0; n < 4; ++n) b(step, n, bh[n], bl[n]);
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int t = 0; t < M; ++t) mma_tf32(small[t][n], al[t], bh[n][0], bh[n][1]);
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int t = 0; t < M; ++t) mma_tf32(big[t][n], ah[t], bh[n][0], bh[n][1]);
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int t = 0; t < M; ++t) mma_tf32(small[t][n], ah[t], bl[n][0], bl[n][1]);
        }
#pragma unroll
        for (int t = 0; t < M; ++t)
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc(t, n)[i] += big[t][n][i];
    }
#pragma unroll
    for (int t = 0; t < M; ++t)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc(t, n)[i] += small[t][n][i];
}

__host__ __device__ inline int k_stride(int dim) { return dim + 4; }                      // an odd multiple of 4: rows on different banks
__host__ __device__ inline int v_stride(int dim_v) { return (dim_v + 31) / 32 * 32 + 8; }  // 8 mod 32: four rows on different banks
constexpr int kPStride = BN + 4;

size_t smem_bytes(int dim, int dim_v, int nodes) {
    return sizeof(float) * (static_cast<size_t>(BM + BN) * k_stride(dim) + static_cast<size_t>(BN) * v_stride(dim_v) + static_cast<size_t>(BM) * kPStride) +
           4 * sizeof(void*) * BN + sizeof(uint32_t) * 9 * nodes;
}

template <int WIDE>   // 8: both head dimensions up to 64, 16: up to 128
struct Tile {
    static constexpr int kM = WIDE == 8 ? 2 : 1;         // 16-row tiles of a warp
    static constexpr int kWarps = BM / 16 / kM, kThreads = kWarps * 32;
};

template <int WIDE>
__global__ void __launch_bounds__(Tile<WIDE>::kThreads)
tree_tf32_kernel(const __grid_constant__ TreeParams p) {
    constexpr int M = Tile<WIDE>::kM, kThreads = Tile<WIDE>::kThreads, kNT = BN / 8;
    extern __shared__ float4 tree_smem_raw[];
    __shared__ int missing[2];   // the tile has keys without a block
    const PagedView& kv = p.kv;
    const int sk = k_stride(kv.dim), sv = v_stride(kv.dim_v);
    float* qs = reinterpret_cast<float*>(tree_smem_raw);   // [BM][sk]
    float* ks = qs + BM * sk;                              // [BN][sk]
    float* vs = ks + BN * sk;                              // [BN][sv]
    float* ps = vs + BN * sv;                              // [BM][kPStride]
    const float** k_rows = reinterpret_cast<const float**>(ps + BM * kPStride);   // [2][BN] rows of this and the next tile, nullptr: masked
    const float** v_rows = k_rows + 2 * BN;
    uint32_t* seen = reinterpret_cast<uint32_t*>(v_rows + 2 * BN);          // [nodes][8]
    int* parent = reinterpret_cast<int*>(seen + 8 * p.nodes);
    const int group = p.q_heads / kv.kv_heads, rows_all = group * p.nodes;
    const int row_tiles = (rows_all + BM - 1) / BM;
    const int tile = blockIdx.x % row_tiles, split_id = blockIdx.x / row_tiles;
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r4 = lane >> 2, quad = lane & 3;
    grid_dependency_wait();
    const int ctx = kv.length(b);
    const int count = tree_node_count(p, b);
    const int keys = ctx + count;
    const int k0 = min(keys, split_id * p.chunk), k1 = split_id == p.splits - 1 ? keys : min(keys, k0 + p.chunk);
    const int row0 = tile * BM, warp_row = row0 + warp * 16 * M;
    if (k1 > ctx) tree_ancestors(p, b, count, parent, seen);
    const float* q = static_cast<const float*>(p.q) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * rows_all * kv.dim;
    const float* draft_k = static_cast<const float*>(p.draft_k) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.nodes * kv.dim;
    const float* draft_v = static_cast<const float*>(p.draft_v) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.nodes * kv.dim_v;
    const auto find_rows = [&](int t0, int buffer) {
        for (int i = threadIdx.x; i < BN; i += kThreads) {
            const int key = t0 + i;
            const float *kr = nullptr, *vr = nullptr;
            if (key < min(k1, ctx)) {
                const int64_t at = kv.row(b, kvh, key);
                if (at < 0) missing[buffer] = 1;
                else {
                    kr = static_cast<const float*>(kv.k_pool) + at * kv.dim;
                    vr = static_cast<const float*>(kv.v_pool) + at * kv.dim_v;
                }
            } else if (key < k1) {
                kr = draft_k + static_cast<size_t>(key - ctx) * kv.dim;
                vr = draft_v + static_cast<size_t>(key - ctx) * kv.dim_v;
            }
            k_rows[buffer * BN + i] = kr;
            v_rows[buffer * BN + i] = vr;
        }
    };
    const auto fetch = [&](float* dst, int stride, int dim, const float** rows) {
        const int pieces = dim / 4;
#pragma unroll 8
        for (int i = threadIdx.x; i < BN * pieces; i += kThreads) {
            const int r = i / pieces, d = (i - r * pieces) * 4;
            const float* src = rows[r];
            if (src) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst + r * stride + d))), "l"(src + d) : "memory");
            else *reinterpret_cast<float4*>(dst + r * stride + d) = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
        }
    };
    const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    const auto wait_but_one = [] { asm volatile("cp.async.wait_group 1;" ::: "memory"); };
    if (threadIdx.x < 2) missing[threadIdx.x] = 0;
    __syncthreads();
    if (k0 < k1) {
        find_rows(k0, 0);
        __syncthreads();
        fetch(ks, sk, kv.dim, k_rows);
        commit();
        fetch(vs, sv, kv.dim_v, v_rows);
        commit();
        const int pieces = kv.dim / 4;
#pragma unroll 8
        for (int i = threadIdx.x; i < BM * pieces; i += kThreads) {
            const int r = i / pieces, d = (i - r * pieces) * 4;
            float4 v = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
            if (row0 + r < rows_all) v = *reinterpret_cast<const float4*>(q + static_cast<size_t>(row0 + r) * kv.dim + d);
            *reinterpret_cast<float4*>(qs + r * sk + d) = make_float4(v.x * p.scale_log2, v.y * p.scale_log2, v.z * p.scale_log2, v.w * p.scale_log2);
        }
    }
    // row i of this lane: warp_row + 16 * (i / 2) + 8 * (i % 2) + r4
    float o[M][WIDE][4], m[2 * M], l[2 * M];
    int node[2 * M];
#pragma unroll
    for (int i = 0; i < 2 * M; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0F;
        node[i] = (warp_row + 16 * (i >> 1) + 8 * (i & 1) + r4) % p.nodes;
    }
#pragma unroll
    for (int t = 0; t < M; ++t)
#pragma unroll
        for (int n = 0; n < WIDE; ++n) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.0F;
    const bool busy = warp_row < rows_all;   // the warp has rows
    float* my_p = ps + warp * 16 * M * kPStride;
    const int nv = kv.dim_v / 8;
    int buffer = 0;
    for (int t0 = k0; t0 < k1; t0 += BN, buffer ^= 1) {
        const bool more = t0 + BN < k1;
        if (more) find_rows(t0 + BN, buffer ^ 1);
        wait_but_one();      // K
        __syncthreads();
        float s[M][kNT][4];
        if (busy) {
#pragma unroll
            for (int t = 0; t < M; ++t)
#pragma unroll
                for (int n = 0; n < kNT; ++n) s[t][n][0] = s[t][n][1] = s[t][n][2] = s[t][n][3] = 0.0F;
#pragma unroll
            for (int n0 = 0; n0 < kNT; n0 += 4)
                multiply<M, 1>([&](int t, int n) -> float (&)[4] { return s[t][n0 + n]; }, kv.dim / 8,
                    [&](int step, int t, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
                        const float* qa = qs + (warp * 16 * M + 16 * t + r4) * sk + 8 * step + quad;
                        split(qa[0], hi[0], lo[0]);
                        split(qa[8 * sk], hi[1], lo[1]);
                        split(qa[4], hi[2], lo[2]);
                        split(qa[8 * sk + 4], hi[3], lo[3]);
                    },
                    [&](int step, int n, uint32_t (&hi)[2], uint32_t (&lo)[2]) {
                        const float* ka = ks + (8 * (n0 + n) + r4) * sk + 8 * step + quad;
                        split(ka[0], hi[0], lo[0]);
                        split(ka[4], hi[1], lo[1]);
                    });
            if (t0 + BN > ctx || t0 + BN > k1) {
#pragma unroll
                for (int n = 0; n < kNT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = t0 + 8 * n + 2 * quad + e;
#pragma unroll
                        for (int i = 0; i < 2 * M; ++i)
                            if (key >= k1 || (key >= ctx && !(seen[node[i] * 8 + ((key - ctx) >> 5)] >> ((key - ctx) & 31) & 1u)))
                                s[i >> 1][n][2 * (i & 1) + e] = -INFINITY;
                    }
            }
            if (missing[buffer]) {
#pragma unroll
                for (int n = 0; n < kNT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (!k_rows[buffer * BN + 8 * n + 2 * quad + e])
#pragma unroll
                            for (int i = 0; i < 2 * M; ++i) s[i >> 1][n][2 * (i & 1) + e] = -INFINITY;
            }
        }
        __syncthreads();
        if (more) fetch(ks, sk, kv.dim, k_rows + (buffer ^ 1) * BN);
        commit();
        if (busy) {
#pragma unroll
            for (int i = 0; i < 2 * M; ++i) {
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < kNT; ++n) top = fmaxf(top, fmaxf(s[i >> 1][n][2 * (i & 1)], s[i >> 1][n][2 * (i & 1) + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                top = fmaxf(top, m[i]);
                const float base = top == -INFINITY ? 0.0F : top;     // (2^-inf = 0 for masked keys)
                const float alpha = exp2_fast(m[i] - base);
                m[i] = top;
                l[i] *= alpha;
#pragma unroll
                for (int n = 0; n < WIDE; ++n) { o[i >> 1][n][2 * (i & 1)] *= alpha; o[i >> 1][n][2 * (i & 1) + 1] *= alpha; }
#pragma unroll
                for (int n = 0; n < kNT; ++n) {
                    float2 e;
                    e.x = exp2_fast(s[i >> 1][n][2 * (i & 1)] - base);
                    e.y = exp2_fast(s[i >> 1][n][2 * (i & 1) + 1] - base);
                    l[i] += e.x + e.y;   // this lane's share of the row sum
                    *reinterpret_cast<float2*>(my_p + (16 * (i >> 1) + 8 * (i & 1) + r4) * kPStride + 8 * n + 2 * quad) = e;
                }
            }
        }
        wait_but_one();      // V
        __syncthreads();
        if (busy) {
#pragma unroll
            for (int n0 = 0; n0 < WIDE; n0 += 4) {
                if (n0 >= nv) continue;      // (columns of V's rows past dim_v feed outputs that are not stored)
                multiply<M, 2>([&](int t, int n) -> float (&)[4] { return o[t][n0 + n]; }, BN / 8,
                    [&](int step, int t, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
                        const float* pa = my_p + (16 * t + r4) * kPStride + 8 * step + quad;
                        split(pa[0], hi[0], lo[0]);
                        split(pa[8 * kPStride], hi[1], lo[1]);
                        split(pa[4], hi[2], lo[2]);
                        split(pa[8 * kPStride + 4], hi[3], lo[3]);
                    },
                    [&](int step, int n, uint32_t (&hi)[2], uint32_t (&lo)[2]) {
                        const float* va = vs + (8 * step + quad) * sv + (n0 + n < nv ? 8 * (n0 + n) : 0) + r4;
                        split(va[0], hi[0], lo[0]);
                        split(va[4 * sv], hi[1], lo[1]);
                    });
            }
        }
        __syncthreads();
        if (more) fetch(vs, sv, kv.dim_v, v_rows + (buffer ^ 1) * BN);
        commit();
    }
#pragma unroll
    for (int i = 0; i < 2 * M; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const int r = warp_row + 16 * (i >> 1) + 8 * (i & 1) + r4;
        if (r >= rows_all || node[i] >= count) continue;
        const size_t row = (static_cast<size_t>(b) * kv.kv_heads + kvh) * rows_all + r;
        float* dst;
        float inv = 1.0F;
        if (p.splits == 1) {
            inv = l[i] == 0.0F ? 0.0F : 1.0F / l[i];
            dst = static_cast<float*>(p.out) + tree_out_row(p, b, kvh * group + r / p.nodes, node[i]) * kv.dim_v;
        } else {
            float* rec = p.partials + (row * p.splits + split_id) * (kv.dim_v + 2);
            if (quad == 0) { rec[0] = m[i]; rec[1] = l[i]; }
            dst = rec + 2;
        }
#pragma unroll
        for (int n = 0; n < WIDE; ++n)
            if (n < nv)
                *reinterpret_cast<float2*>(dst + 8 * n + 2 * quad) = make_float2(o[i >> 1][n][2 * (i & 1)] * inv, o[i >> 1][n][2 * (i & 1) + 1] * inv);
    }
}

template <int WIDE>
sfb_status launch(const TreeParams& p, cudaStream_t stream) {
    const size_t smem = smem_bytes(p.kv.dim, p.kv.dim_v, p.nodes);
    SFB_CUDA(cudaFuncSetAttribute(tree_tf32_kernel<WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    const int rows = p.q_heads / p.kv.kv_heads * p.nodes;
    const dim3 grid(ceil_div(rows, BM) * p.splits, p.kv.kv_heads, p.batch);
    SFB_CUDA(launch_dependent(tree_tf32_kernel<WIDE>, grid, dim3(Tile<WIDE>::kThreads), smem, stream, p));
    return check_launch("attention_tree_tf32");
}

}  // namespace

bool tree_tf32_shape(const sfb_tree_args& a) {
    return a.dtype == SFB_F32 && a.head_dim % 8 == 0 && a.head_dim_value % 8 == 0 && a.head_dim <= 128 && a.head_dim_value <= 128;
}

sfb_status tree_tf32(const TreeParams& p, cudaStream_t stream) {
    return p.kv.dim <= 64 && p.kv.dim_v <= 64 ? launch<8>(p, stream) : launch<16>(p, stream);
}

}  // namespace sfb
