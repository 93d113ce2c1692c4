// Tree attention in float32 on the warp-level tensor path (head dimensions up to 128, multiples of 8, 16-byte aligned).
//
// A float32 value is split into two TF32 parts, x = hi + lo with hi the upper 11 bits of the significand and lo the
// next 11, and a product is hi hi + hi lo + lo hi, accumulated in 32 bits: what is dropped is 2^-22 of each term, a quarter of the
// rounding of a float32 sum of sixteen.  Three m16n8k8 products replace 32 multiply-adds a lane, so the instruction
// count falls to a fifth of the CUDA-core form (attention_tree.cu), which had no issue slots left to cover its
// loads (16 sequences of up to 1500 tokens, 27 nodes, 64-dimensional heads: 68 us there).
// A CTA takes 128 query rows of one (sequence, K/V head) and a split of the keys in tiles of 64.  A warp owns 32 rows (16
// where a head dimension is above 64); P goes through its own part of shared memory, so that both products are rolled
// loops: fully unrolled they spent a third of the time waiting for instructions.  K of the next tile is fetched (cp.async)
// under the softmax and P.V of this one, V under the scores of the next.
// That case takes 36 us with the joining: 2.4 us of bytes, 10 us of TF32 products (8 cycles each a scheduler), the rest
// latencies that two warps a scheduler (255 registers, 108 KB a CTA) cover in part.  Sixteen rows a warp and twice the
// warps: 41 against 40 us, eight column tiles at a time then: 43.
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

// acc(t, n) += the products of N column tiles n and M row tiles t over `steps` steps of eight, operands from
// a(step, t, hi, lo) and b(step, n, hi, lo).  The instruction truncates its sums, so an accumulator starts from zero every
// DEPTH steps, takes the small products first, while truncation costs nothing, then the large ones, and a rounded addition
// takes it over.  (All three products in one accumulator running on over the tiles: 2.6e-6 off at logits of ten.)
// Four column tiles at a time, so that the products of one accumulator, each of which waits for the one before, are 4 * M
// instructions apart.
template <int M, int N, int DEPTH, class Acc, class A, class B>
__device__ __forceinline__ void multiply(Acc acc, int steps, A a, B b) {
#pragma unroll 1
    for (int step0 = 0; step0 < steps; step0 += DEPTH) {
        uint32_t ah[DEPTH][M][4], al[DEPTH][M][4];
#pragma unroll
        for (int u = 0; u < DEPTH; ++u)
#pragma unroll
            for (int t = 0; t < M; ++t) a(step0 + u, t, ah[u][t], al[u][t]);
#pragma unroll
        for (int n0 = 0; n0 < N; n0 += 4) {
            float sum[M][4][4];
            uint32_t bh[DEPTH][4][2], bl[DEPTH][4][2];
#pragma unroll
            for (int t = 0; t < M; ++t)
#pragma unroll
                for (int n = 0; n < 4; ++n) sum[t][n][0] = sum[t][n][1] = sum[t][n][2] = sum[t][n][3] = 0.0F;
#pragma unroll
            for (int u = 0; u < DEPTH; ++u)
#pragma unroll
                for (int n = 0; n < 4; ++n) b(step0 + u, n0 + n, bh[u][n], bl[u][n]);
#pragma unroll
            for (int u = 0; u < DEPTH; ++u) {
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int t = 0; t < M; ++t) mma_tf32(sum[t][n], al[u][t], bh[u][n][0], bh[u][n][1]);
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int t = 0; t < M; ++t) mma_tf32(sum[t][n], ah[u][t], bl[u][n][0], bl[u][n][1]);
            }
#pragma unroll
            for (int u = 0; u < DEPTH; ++u)
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int t = 0; t < M; ++t) mma_tf32(sum[t][n], ah[u][t], bh[u][n][0], bh[u][n][1]);
#pragma unroll
            for (int t = 0; t < M; ++t)
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc(t, n0 + n)[i] += sum[t][n][i];
        }
    }
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
    constexpr int kPieces = 2 * WIDE;      // lanes that copy a row, 16 bytes each
    constexpr int kRowsAtOnce = kThreads / kPieces;
    extern __shared__ float4 tree_smem_raw[];
    __shared__ int missing[2];   // the tile has keys without a block
    __shared__ int row_of[BM];   // head in the group * 256 + node of every row, -1: none
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
    // the rows of live nodes only, closely packed: a tree of half its nodes costs half the products
    const int row0 = tile * BM, warp_row = warp * 16 * M, rows_live = group * count;
    if (row0 >= rows_live || k0 >= k1) return;     // (an empty split leaves no piece)
    for (int i = threadIdx.x; i < BM; i += kThreads) {
        const int r = row0 + i;
        row_of[i] = r < rows_live ? (r / count) * 256 + r % count : -1;
    }
    if (k1 > ctx) tree_ancestors(p, b, count, parent, seen);
    const float* q = static_cast<const float*>(p.q) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * rows_all * kv.dim;
    const float* draft_k = static_cast<const float*>(p.draft_k) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.nodes * kv.dim;
    const float* draft_v = static_cast<const float*>(p.draft_v) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.nodes * kv.dim_v;
    const auto find = [&](int t0) {   // the block of key t0 + thread, read long before it is needed
        const int key = t0 + static_cast<int>(threadIdx.x);
        return threadIdx.x < BN && key < min(k1, ctx) ? kv.page(b, key) : -1;
    };
    const auto note = [&](int t0, int page, int buffer) {
        if (threadIdx.x < BN) {
            const int i = threadIdx.x, key = t0 + i;
            const float *kr = nullptr, *vr = nullptr;
            if (key < min(k1, ctx)) {
                const int64_t at = kv.row_in(page, kvh, key);
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
        const int d = 4 * (threadIdx.x % kPieces);
        if (d >= dim) return;
        const float* from[BN / kRowsAtOnce];   // (read together: the copies between them are barriers to the compiler)
#pragma unroll
        for (int i = 0; i < BN / kRowsAtOnce; ++i) from[i] = rows[threadIdx.x / kPieces + i * kRowsAtOnce];
#pragma unroll
        for (int i = 0; i < BN / kRowsAtOnce; ++i) {
            const int r = threadIdx.x / kPieces + i * kRowsAtOnce;
            const float* src = from[i];
            if (src) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst + r * stride + d))), "l"(src + d) : "memory");
            else *reinterpret_cast<float4*>(dst + r * stride + d) = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
        }
    };
    const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    const auto wait_but_one = [] { asm volatile("cp.async.wait_group 1;" ::: "memory"); };
    if (threadIdx.x < 2) missing[threadIdx.x] = 0;
    __syncthreads();
    {
        note(k0, find(k0), 0);
        __syncthreads();
        fetch(ks, sk, kv.dim, k_rows);
        commit();
        fetch(vs, sv, kv.dim_v, v_rows);
        commit();
        const int d = 4 * (threadIdx.x % kPieces);
        float4 v[BM / kRowsAtOnce];
#pragma unroll
        for (int i = 0; i < BM / kRowsAtOnce; ++i) {
            const int at = row_of[threadIdx.x / kPieces + i * kRowsAtOnce];
            v[i] = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
            if (at >= 0 && d < kv.dim) v[i] = *reinterpret_cast<const float4*>(q + static_cast<size_t>((at >> 8) * p.nodes + (at & 255)) * kv.dim + d);
        }
        if (d < kv.dim)
#pragma unroll
            for (int i = 0; i < BM / kRowsAtOnce; ++i)
                *reinterpret_cast<float4*>(qs + (threadIdx.x / kPieces + i * kRowsAtOnce) * sk + d) =
                    make_float4(v[i].x * p.scale_log2, v[i].y * p.scale_log2, v[i].z * p.scale_log2, v[i].w * p.scale_log2);
    }
    // row i of this lane: warp_row + 16 * (i / 2) + 8 * (i % 2) + r4
    float o[M][WIDE][4], m[2 * M], l[2 * M];
    int node[2 * M];
#pragma unroll
    for (int i = 0; i < 2 * M; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0F;
        node[i] = max(row_of[warp_row + 16 * (i >> 1) + 8 * (i & 1) + r4], 0) & 255;
    }
#pragma unroll
    for (int t = 0; t < M; ++t)
#pragma unroll
        for (int n = 0; n < WIDE; ++n) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.0F;
    const bool busy = row0 + warp_row < rows_live;   // the warp has rows
    float* my_p = ps + warp * 16 * M * kPStride;
    const int nv = kv.dim_v / 8;
    int buffer = 0;
    for (int t0 = k0; t0 < k1; t0 += BN, buffer ^= 1) {
        const bool more = t0 + BN < k1;
        const int next = more ? find(t0 + BN) : -1;
        wait_but_one();      // K
        __syncthreads();
        float s[M][kNT][4];
        if (busy) {
#pragma unroll
            for (int t = 0; t < M; ++t)
#pragma unroll
                for (int n = 0; n < kNT; ++n) s[t][n][0] = s[t][n][1] = s[t][n][2] = s[t][n][3] = 0.0F;
            multiply<M, kNT, 1>([&](int t, int n) -> float (&)[4] { return s[t][n]; }, kv.dim / 8,
                [&](int step, int t, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
                    const float* qa = qs + (warp * 16 * M + 16 * t + r4) * sk + 8 * step + quad;
                    split(qa[0], hi[0], lo[0]);
                    split(qa[8 * sk], hi[1], lo[1]);
                    split(qa[4], hi[2], lo[2]);
                    split(qa[8 * sk + 4], hi[3], lo[3]);
                },
                [&](int step, int n, uint32_t (&hi)[2], uint32_t (&lo)[2]) {
                    const float* ka = ks + (8 * n + r4) * sk + 8 * step + quad;
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
        if (more) note(t0 + BN, next, buffer ^ 1);
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
            multiply<M, WIDE, 2>([&](int t, int n) -> float (&)[4] { return o[t][n]; }, BN / 8,
                [&](int step, int t, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
                    const float* pa = my_p + (16 * t + r4) * kPStride + 8 * step + quad;
                    split(pa[0], hi[0], lo[0]);
                    split(pa[8 * kPStride], hi[1], lo[1]);
                    split(pa[4], hi[2], lo[2]);
                    split(pa[8 * kPStride + 4], hi[3], lo[3]);
                },
                [&](int step, int n, uint32_t (&hi)[2], uint32_t (&lo)[2]) {   // (columns past dim_v feed outputs that are not stored)
                    const float* va = vs + (8 * step + quad) * sv + (n < nv ? 8 * n : 0) + r4;
                    split(va[0], hi[0], lo[0]);
                    split(va[4 * sv], hi[1], lo[1]);
                });
        }
        __syncthreads();
        if (more) fetch(vs, sv, kv.dim_v, v_rows + (buffer ^ 1) * BN);
        commit();
    }
#pragma unroll
    for (int i = 0; i < 2 * M; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const int at = row_of[warp_row + 16 * (i >> 1) + 8 * (i & 1) + r4];
        if (at < 0) continue;
        const int head = kvh * group + (at >> 8);
        const size_t row = (static_cast<size_t>(b) * p.q_heads + head) * p.nodes + node[i];
        float* dst;
        float inv = 1.0F;
        if (p.splits == 1) {
            inv = l[i] == 0.0F ? 0.0F : 1.0F / l[i];
            dst = static_cast<float*>(p.out) + tree_out_row(p, b, head, node[i]) * kv.dim_v;
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
    // (the same limit for every shape, since another thread may be launching the kernel)
    static const int most = static_cast<int>(smem_bytes(8 * WIDE, 8 * WIDE, SFB_MAX_TREE_NODES));
    SFB_CUDA(cudaFuncSetAttribute(tree_tf32_kernel<WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
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
