// Single-token attention over a paged cache on the warp-level tensor path: bf16, head_dim = head_dim_value = 128 or
// 64, blocks of a multiple of 16 tokens, whole context or a list of blocks, with or without keeping the logits.
//
// HBM-bound: every K and V byte of a (sequence, K/V head) is read once and shared by up to eight query heads.  One CTA of
// four warps takes a split.  The unit is 16 tokens of one block: TMA brings its K and V rows as 16-row, 128-byte
// boxes (128-byte swizzle), four units per stage, so that ~96 KB per CTA and two CTAs per SM are in flight whatever
// the warps do.  A warp takes one unit per stage: scores by m16n8k16 products (the heads are rows 0-7, rows 8-15 are
// zero), base-2 online softmax with a lazily moved maximum, P as the A operand of P.V.  tcgen05 would need 128 rows for
// at most eight heads; the arithmetic here is far below the byte stream either way.
// Tokens of a unit past the context may hold anything: their scores are masked, and their V rows are zeroed in shared
// memory first (0 * NaN).  Waits are bounded.
#include "cache_ops.cuh"
#include "mma_sync.cuh"
#include "ptx_sm100.cuh"

namespace sfb {
namespace {

constexpr int U = 16;               // tokens per unit
constexpr int kUnits = 4;           // per stage, one per warp
constexpr int kThreads = 128;
constexpr int kHeads = 8;
constexpr int kMaxUnits = 4096;     // per split (their rows and positions are listed in shared memory)
constexpr uint32_t kCodeStep = 0x40;

template <int D>
struct Shape {
    static constexpr int kHalves = D / 64;
    static constexpr int kUnitBytes = U * D * 2;
    static constexpr int kStageBytes = 2 * kUnits * kUnitBytes;     // K units, then V units
    static constexpr int kStages = D == 128 ? 3 : 6;
};

// 16-byte chunk `chunk` (of D / 8) of token row `row` inside a swizzled unit.
__device__ __forceinline__ uint32_t unit_chunk(uint32_t unit, int row, int chunk) {
    return unit + (chunk >> 3) * (U * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

template <int D>
__global__ void __launch_bounds__(kThreads, 2)
step_mma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ StepParams p, int pool_rows) {
    using Sh = Shape<D>;
    constexpr int kStages = Sh::kStages, kUnitBytes = Sh::kUnitBytes, kStageBytes = Sh::kStageBytes;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes);
    uint64_t* empty_bar = full_bar + kStages;
    volatile uint32_t* abort_flag = reinterpret_cast<uint32_t*>(empty_bar + kStages);
    int2* units = reinterpret_cast<int2*>(empty_bar + kStages + 1);   // pool row and position; row pool_rows: no block
    const PagedView& kv = p.kv;
    const int group = p.q_heads / kv.kv_heads, chunks = (group + kHeads - 1) / kHeads;
    const int split = blockIdx.x, b = blockIdx.z;
    const int kvh = blockIdx.y / chunks, head0 = kvh * group + (blockIdx.y % chunks) * kHeads;
    const int heads = min(kHeads, (kvh + 1) * group - head0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, quad = lane & 3;
    const int record = D + 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 4);
        }
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async();
        ptx::prefetch_tensormap(&map_k);
        ptx::prefetch_tensormap(&map_v);
    }
    grid_dependents_may_launch();
    grid_dependency_wait();
    const int ctx = kv.length(b);
    const int blocks = ctx > 0 ? kv.block_of(ctx - 1) + 1 : 0;
    const int* list = p.selected ? p.selected + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.budget : nullptr;
    const int entries = list ? min(p.budget, blocks) : blocks;
    const int e0 = min(entries, split * p.chunk_blocks), e1 = min(entries, e0 + p.chunk_blocks);
    const int per_block = kv.block_tokens / U;
    const int n_units = (e1 - e0) * per_block;
    const size_t row0 = static_cast<size_t>(b) * p.q_heads + head0;
    if (n_units == 0) {
        if (p.splits == 1 && !p.logits) {
            for (int i = threadIdx.x; i < heads * D; i += kThreads) static_cast<bf16*>(p.out)[row0 * D + i] = __float2bfloat16_rn(0.0F);
        } else {
            for (int i = threadIdx.x; i < heads * record; i += kThreads)
                p.partials[((row0 + i / record) * p.splits + split) * record + i % record] = i % record == 0 ? -INFINITY : 0.0F;
        }
        return;
    }
    for (int i = threadIdx.x; i < n_units; i += kThreads) {
        const int e = i / per_block, inner = (i - e * per_block) * U;
        const int logical = list ? list[e0 + e] : e0 + e;
        int at = pool_rows, position = ctx;   // (an entry of -1 is not followed)
        if (logical >= 0) {
            position = logical * kv.block_tokens + inner;
            if (position < ctx) {
                const int page = kv.table[static_cast<size_t>(b) * kv.max_blocks + logical];
                if (page >= 0 && page < kv.num_blocks) at = (page * kv.kv_heads + kvh) * kv.block_tokens + inner;
                else atomicOr(kv.status, kCodeDecodeBounds);
            }
        }
        units[i] = make_int2(at, position);
    }
    // Q as A fragments, 16 elements of the head dimension per slice; rows past the heads are zero
    uint32_t qa[D / 16][4];
    {
        const bf16* q = static_cast<const bf16*>(p.q) + (row0 + row) * D;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            qa[s][0] = row < heads ? *reinterpret_cast<const uint32_t*>(q + 16 * s + quad * 2) : 0u;
            qa[s][2] = row < heads ? *reinterpret_cast<const uint32_t*>(q + 16 * s + 8 + quad * 2) : 0u;
            qa[s][1] = qa[s][3] = 0u;
        }
    }
    __syncthreads();
    const int n_stages = (n_units + kUnits - 1) / kUnits;
    const auto issue_stage = [&](int it) -> bool {   // thread 0 only
        const int s = it % kStages;
        if (!ptx::mbar_wait(ptx::smem_u32(&empty_bar[s]), ((it / kStages) & 1) ^ 1, abort_flag, kv.status, kCodeStep | 1)) return false;
        const int n = min(kUnits, n_units - it * kUnits);
        const uint32_t bar = ptx::smem_u32(&full_bar[s]);
        ptx::mbar_expect_tx(bar, static_cast<uint32_t>(n) * 2 * kUnitBytes);
        const uint32_t stage = ptx::smem_u32(smem + s * kStageBytes);
        for (int w = 0; w < n; ++w) {
            const int at = units[it * kUnits + w].x;
            const uint32_t kd = stage + w * kUnitBytes, vd = stage + (kUnits + w) * kUnitBytes;
#pragma unroll
            for (int h = 0; h < Sh::kHalves; ++h) {
                ptx::tma_load_2d(kd + h * U * 128, &map_k, bar, 64 * h, at);
                ptx::tma_load_2d(vd + h * U * 128, &map_v, bar, 64 * h, at);
            }
        }
        return true;
    };
    if (threadIdx.x == 0)
        for (int it = 0; it < min(kStages, n_stages); ++it) issue_stage(it);

    float o[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0F;
    float m_used = -INFINITY, l_part = 0.0F;   // l_part: this lane's share of the row sum
    float* logits = p.logits ? p.logits + (row0 + row) * p.logit_stride : nullptr;
    for (int it = 0; it < n_stages; ++it) {
        const int s = it % kStages;
        if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&full_bar[s]), (it / kStages) & 1, abort_flag, kv.status, kCodeStep | 2))) break;
        const int local = it * kUnits + warp;
        if (local < n_units) {
            const int2 unit = units[local];
            const int live = unit.x == pool_rows ? 0 : min(U, ctx - unit.y);
            const uint32_t kunit = ptx::smem_u32(smem + s * kStageBytes + warp * kUnitBytes);
            const uint32_t vunit = kunit + kUnits * kUnitBytes;
            if (live < U) {
                uint8_t* v = smem + s * kStageBytes + (kUnits + warp) * kUnitBytes;
                for (int i = lane; i < (U - live) * 8 * Sh::kHalves; i += 32) {
                    const int piece = i & 7, half = (i >> 3) % Sh::kHalves, dead = live + (i >> 3) / Sh::kHalves;
                    *reinterpret_cast<uint4*>(v + half * U * 128 + dead * 128 + piece * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                ptx::fence_proxy_async();   // (the stage is refilled by TMA)
                __syncwarp();
            }
            float sc[2][4], x[4];
            float tile_max = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.0F;
#pragma unroll
                for (int sp = 0; sp < D / 32; ++sp) {
                    uint32_t kb[4];
                    ldmatrix_x4(unit_chunk(kunit, 8 * t + (lane & 7), 4 * sp + (lane >> 3)), kb);
                    mma_bf16(sc[t], qa[2 * sp], kb[0], kb[1]);
                    mma_bf16(sc[t], qa[2 * sp + 1], kb[2], kb[3]);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int token = 8 * t + 2 * quad + e;
                    x[2 * t + e] = token < live ? sc[t][e] * p.scale_log2 : -INFINITY;
                    tile_max = fmaxf(tile_max, x[2 * t + e]);
                }
                if (logits && row < heads) {
                    const int position = unit.y + 8 * t + 2 * quad;
                    if (position + 1 < ctx) *reinterpret_cast<float2*>(logits + position) = make_float2(x[2 * t], x[2 * t + 1]);
                    else if (position < ctx) logits[position] = x[2 * t];
                }
            }
            tile_max = fmaxf(tile_max, __shfl_xor_sync(0xffffffffu, tile_max, 1));
            tile_max = fmaxf(tile_max, __shfl_xor_sync(0xffffffffu, tile_max, 2));
            if (tile_max > m_used + 8.0F) {  // lazily moved maximum (also the first unit: m_used = -inf)
                const float alpha = exp2_fast(m_used - tile_max);
                l_part *= alpha;
#pragma unroll
                for (int j = 0; j < D / 8; ++j) { o[j][0] *= alpha; o[j][1] *= alpha; }
                m_used = tile_max;
            }
            uint32_t pa[4];
            {
                float pr[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    pr[i] = x[i] == -INFINITY ? 0.0F : exp2_fast(x[i] - m_used);
                    l_part += pr[i];
                }
                pa[0] = pack_bf16(pr[0], pr[1]);   // the weights are rounded to bf16 for the product, the sum is not
                pa[2] = pack_bf16(pr[2], pr[3]);
                pa[1] = pa[3] = 0u;
            }
#pragma unroll
            for (int jp = 0; jp < D / 16; ++jp) {
                uint32_t vb[4];
                ldmatrix_x4_trans(unit_chunk(vunit, ((lane >> 3) & 1) * 8 + (lane & 7), 2 * jp + (lane >> 4)), vb);
                mma_bf16(o[2 * jp], pa, vb[0], vb[1]);
                mma_bf16(o[2 * jp + 1], pa, vb[2], vb[3]);
            }
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&empty_bar[s]));
        if (threadIdx.x == 0 && it + kStages < n_stages) issue_stage(it + kStages);   // (a wait that gives up sets the abort flag)
    }
    __syncthreads();
    if (*abort_flag)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);  // let copies in flight land before the CTA exits

    l_part += __shfl_xor_sync(0xffffffffu, l_part, 1);
    l_part += __shfl_xor_sync(0xffffffffu, l_part, 2);
    // the four warps meet in shared memory (the stages are free now)
    float* wm = reinterpret_cast<float*>(smem);   // [4][kHeads]
    float* wl = wm + 4 * kHeads;                  // [4][kHeads]
    float* wo = wl + 4 * kHeads;                  // [4][kHeads][D]
    if (quad == 0) { wm[warp * kHeads + row] = m_used; wl[warp * kHeads + row] = l_part; }
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<float2*>(wo + (warp * kHeads + row) * D + 8 * j + 2 * quad) = make_float2(o[j][0], o[j][1]);
    __syncthreads();
    for (int i = threadIdx.x; i < heads * D; i += kThreads) {
        const int h = i / D, d = i % D;
        const float top = fmaxf(fmaxf(wm[h], wm[kHeads + h]), fmaxf(wm[2 * kHeads + h], wm[3 * kHeads + h]));
        float sum = 0.0F, a = 0.0F;
        if (top != -INFINITY) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = wm[w * kHeads + h] == -INFINITY ? 0.0F : exp2_fast(wm[w * kHeads + h] - top);
                sum += wl[w * kHeads + h] * f;
                a += wo[(w * kHeads + h) * D + d] * f;
            }
        }
        if (p.splits == 1 && !p.logits) {
            static_cast<bf16*>(p.out)[(row0 + h) * D + d] = __float2bfloat16_rn(sum == 0.0F ? 0.0F : a / sum);
        } else {
            float* rec = p.partials + ((row0 + h) * p.splits + split) * record;
            if (d == 0) { rec[0] = top; rec[1] = sum; }
            rec[2 + d] = a;
        }
    }
}

template <int D>
sfb_status launch_mma(const StepParams& p, cudaStream_t stream) {
    const PagedView& kv = p.kv;
    CUtensorMap mk, mv;
    const int pool_rows = kv.num_blocks * kv.kv_heads * kv.block_tokens;
    if (!encode_tensor_map_bf16_2d(&mk, kv.k_pool, pool_rows, D, U, 64) || !encode_tensor_map_bf16_2d(&mv, kv.v_pool, pool_rows, D, U, 64))
        return SFB_CUDA_ERROR;
    const int units = p.chunk_blocks * (kv.block_tokens / U);
    const size_t smem = static_cast<size_t>(Shape<D>::kStages) * Shape<D>::kStageBytes + 16 * Shape<D>::kStages + 8 +
                        sizeof(int2) * units + 1024;
    SFB_CUDA(cudaFuncSetAttribute(step_mma_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    const dim3 grid(p.splits, kv.kv_heads * ceil_div(p.q_heads / kv.kv_heads, kHeads), p.batch);
    SFB_CUDA(launch_dependent(step_mma_kernel<D>, grid, dim3(kThreads), smem, stream, mk, mv, p, pool_rows));
    return check_launch("attention_step_mma");
}

}  // namespace

bool step_mma_supported(const StepParams& p, int dtype) {
    const PagedView& kv = p.kv;
    return dtype == SFB_BF16 && (kv.dim == 128 || kv.dim == 64) && kv.dim_v == kv.dim && kv.block_tokens % U == 0 &&
           static_cast<int64_t>(p.chunk_blocks) * (kv.block_tokens / U) <= kMaxUnits &&
           static_cast<int64_t>(kv.num_blocks) * kv.kv_heads * kv.block_tokens < (int64_t{1} << 30) && aligned16(kv.k_pool) &&
           aligned16(kv.v_pool) && (reinterpret_cast<uintptr_t>(p.q) & 3) == 0;
}

sfb_status step_mma(const StepParams& p, cudaStream_t stream) {
    return p.kv.dim == 128 ? launch_mma<128>(p, stream) : launch_mma<64>(p, stream);
}

}  // namespace sfb
