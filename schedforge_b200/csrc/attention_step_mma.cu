// Single-token attention over a paged cache on the warp-level tensor path: bf16, head_dim = head_dim_value = 128 or
// 64, blocks of a multiple of 16 tokens, whole context or a list of blocks, with or without keeping the logits.
//
// HBM-bound: every K and V byte of a (sequence, K/V head) is read once and shared by up to eight query heads.  The unit
// is 16 tokens of one block.  The units of all (sequence, K/V head, eight heads) pairs are laid end to end and every CTA
// takes one equal range: two CTAs per SM, one round, no tail however ragged the contexts are (batch 64, contexts of 512 to
// 8192 tokens: splits of 2048 tokens ran at 0.78 of the copy bandwidth, 2.6 rounds of which the last is not full).
// A copy warp brings a unit's K and V rows as 16-row, 128-byte boxes by TMA (128-byte swizzle), four units per stage,
// ~96 KB per CTA in flight, and runs on into the next pair while the others still work on the last.  Each of the four
// other warps takes one unit per stage: scores by m16n8k16 products (the heads are rows 0-7, rows 8-15 are zero), base-2
// online softmax with a lazily moved maximum, P as the A operand of P.V.  tcgen05 would need 128 rows for at most eight
// heads; the arithmetic here is far below the byte stream either way.
// Tokens of a unit past the context may hold anything: their scores are masked, and their V rows are zeroed in shared
// memory first (0 * NaN).  Waits are bounded.
#include "cache_ops.cuh"
#include "mma_sync.cuh"
#include "ptx_sm100.cuh"

namespace sfb {
namespace {

constexpr int U = 16;               // tokens per unit
constexpr int kUnits = 4;           // per stage, one per warp
constexpr int kThreads = 160;        // four warps that compute, one that copies
constexpr int kHeads = kPieceHeads;
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

// Position of a warp in the CTA's range of units.
struct Walk {
    int b, sub, x, ctx, units, left;

    __device__ __forceinline__ static int units_of(const StepParams& p, int ctx) {
        if (ctx == 0) return 0;
        if (!p.selected) return (ctx + U - 1) / U;
        return min(p.budget, p.kv.block_of(ctx - 1) + 1) * (p.kv.block_tokens / U);
    }
    __device__ __forceinline__ void read(const StepParams& p) {
        ctx = p.kv.length(b);
        units = units_of(p, ctx);
    }
    __device__ __forceinline__ int take() const { return min(left, units - x); }
    __device__ __forceinline__ void advance(const StepParams& p, int subs, int n) {
        left -= n;
        x += n;
        if (x < units || left <= 0) return;
        x = 0;
        if (++sub < subs) return;
        sub = 0;
        do {
            if (++b >= p.batch) { left = 0; return; }
            read(p);
        } while (units == 0);
    }
};

template <int D>
__global__ void __launch_bounds__(kThreads, 2)
step_mma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ StepParams p, int pool_rows) {
    using Sh = Shape<D>;
    constexpr int kStages = Sh::kStages, kUnitBytes = Sh::kUnitBytes, kStageBytes = Sh::kStageBytes;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* merge_o = reinterpret_cast<float*>(smem + kStages * kStageBytes);      // [3][kHeads][D], of warps 1 to 3
    float2* merge_ml = reinterpret_cast<float2*>(merge_o + 3 * kHeads * D);       // [3][kHeads]
    int2* meta = reinterpret_cast<int2*>(merge_ml + 3 * kHeads);                  // [kStages][kUnits] pool row, position
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(meta + kStages * kUnits);
    uint64_t* empty_bar = full_bar + kStages;
    uint64_t* merge_bar = empty_bar + kStages;    // [2]: the warps' results are there / have been read
    int* start = reinterpret_cast<int*>(merge_bar + 2);
    volatile uint32_t* abort_flag = reinterpret_cast<uint32_t*>(start + 6);
    const PagedView& kv = p.kv;
    const int group = p.q_heads / kv.kv_heads, chunks = (group + kHeads - 1) / kHeads, subs = kv.kv_heads * chunks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(ptx::smem_u32(&full_bar[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&empty_bar[s]), 4);
        }
        ptx::mbar_init(ptx::smem_u32(&merge_bar[0]), 3);
        ptx::mbar_init(ptx::smem_u32(&merge_bar[1]), 1);
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async();
        ptx::prefetch_tensormap(&map_k);
        ptx::prefetch_tensormap(&map_v);
    }
    grid_dependency_wait();
    if (warp == 4) even_range(p.batch, subs, kUnits, [&](int b) { return Walk::units_of(p, kv.length(b)); }, start);
    __syncthreads();
    Walk w{};
    w.left = start[3];
    if (w.left > 0) {
        w.b = start[0]; w.sub = start[1]; w.x = start[2];
        w.read(p);
    }
    if (warp == 4) {
        // ---------------------------------------------------------------- copies
        // lane = (unit of the stage, K or V, half): each lane issues one box
        const int per_block = kv.block_tokens / U, block_units = per_block;
        const int unit = lane / (2 * Sh::kHalves), which = lane / Sh::kHalves & 1, half = lane % Sh::kHalves;
        uint32_t n_stage = 0;
        bool ok = true;
        while (ok && w.left > 0) {
            const int n = w.take(), kvh = w.sub / chunks;
            const int* list = p.selected ? p.selected + (static_cast<size_t>(w.b) * kv.kv_heads + kvh) * p.budget : nullptr;
            const int* table = kv.table + static_cast<size_t>(w.b) * kv.max_blocks;
            const auto locate = [&](int i) -> int2 {   // pool row and position of unit i of the pair
                if (unit >= kUnits || i >= w.x + n) return make_int2(-1, 0);
                const int e = i / block_units, inner = (i - e * block_units) * U;
                const int logical = list ? list[e] : e;
                if (logical < 0) return make_int2(pool_rows, w.ctx);          // (an entry of -1 is not followed)
                const int position = logical * kv.block_tokens + inner;
                if (position >= w.ctx) return make_int2(pool_rows, w.ctx);    // behind the context: nothing live
                const int page = table[logical];
                if (page >= 0 && page < kv.num_blocks) return make_int2((page * kv.kv_heads + kvh) * kv.block_tokens + inner, position);
                if (which == 0 && half == 0) atomicOr(kv.status, kCodeDecodeBounds);
                return make_int2(pool_rows, position);                         // outside the tensor map: reads zeros
            };
            int2 next = locate(w.x + unit);
            for (int i0 = w.x; i0 < w.x + n; i0 += kUnits, ++n_stage) {
                const int2 mine = next;
                next = locate(i0 + kUnits + unit);        // in flight while this stage waits
                const int s = n_stage % kStages;
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&empty_bar[s]), ((n_stage / kStages) & 1) ^ 1, abort_flag, kv.status, kCodeStep | 1));
                if (!ok) break;
                const uint32_t bar = ptx::smem_u32(&full_bar[s]);
                if (mine.x >= 0 && which == 0 && half == 0) meta[s * kUnits + unit] = mine;
                __syncwarp();
                if (lane == 0) ptx::mbar_expect_tx(bar, static_cast<uint32_t>(min(kUnits, w.x + n - i0)) * 2 * kUnitBytes);
                __syncwarp();
                if (mine.x >= 0)
                    ptx::tma_load_2d(ptx::smem_u32(smem + s * kStageBytes + (which * kUnits + unit) * kUnitBytes + half * U * 128), which ? &map_v : &map_k,
                                     bar, 64 * half, mine.x);
            }
            w.advance(p, subs, n);
        }
    } else {
        // ---------------------------------------------------------------- arithmetic
        const int row = lane >> 2, quad = lane & 3;
        uint32_t n_stage = 0, n_piece = 0;
        bool ok = true;
        while (ok && w.left > 0) {
            const int n = w.take(), kvh = w.sub / chunks, head0 = kvh * group + (w.sub % chunks) * kHeads;
            const int heads = min(kHeads, (kvh + 1) * group - head0);
            const size_t row0 = static_cast<size_t>(w.b) * p.q_heads + head0;
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
            float o[D / 8][4];
#pragma unroll
            for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0F;
            float m_used = -INFINITY, l_part = 0.0F;   // l_part: this lane's share of the row sum
            float* logits = p.logits ? p.logits + (row0 + row) * p.logit_stride : nullptr;
            for (int i0 = 0; i0 < n; i0 += kUnits, ++n_stage) {
                const int s = n_stage % kStages;
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&full_bar[s]), (n_stage / kStages) & 1, abort_flag, kv.status, kCodeStep | 2));
                if (!ok) break;
                if (i0 + warp < n) {
                    const int2 unit = meta[s * kUnits + warp];
                    const int live = unit.x == pool_rows ? 0 : min(U, w.ctx - unit.y);
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
                            if (position + 1 < w.ctx) *reinterpret_cast<float2*>(logits + position) = make_float2(x[2 * t], x[2 * t + 1]);
                            else if (position < w.ctx) logits[position] = x[2 * t];
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
            }
            if (!ok) break;
            l_part += __shfl_xor_sync(0xffffffffu, l_part, 1);
            l_part += __shfl_xor_sync(0xffffffffu, l_part, 2);
            // warps 1 to 3 leave their results in shared memory, warp 0 joins them with its own
            const auto wait = [&](int i, uint32_t parity) -> bool {
                return __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&merge_bar[i]), parity, abort_flag, kv.status, kCodeStep | 4));
            };
            if (warp > 0) {
                ok = wait(1, (n_piece & 1) ^ 1);
                if (!ok) break;
                if (quad == 0) merge_ml[(warp - 1) * kHeads + row] = make_float2(m_used, l_part);
#pragma unroll
                for (int j = 0; j < D / 8; ++j)
                    *reinterpret_cast<float2*>(merge_o + ((warp - 1) * kHeads + row) * D + 8 * j + 2 * quad) = make_float2(o[j][0], o[j][1]);
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&merge_bar[0]));
            } else {
                ok = wait(0, n_piece & 1);
                if (!ok) break;
                float2 ml[3];
                float top = m_used, f[3];
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    ml[i] = merge_ml[i * kHeads + row];
                    top = fmaxf(top, ml[i].x);
                }
                const float f0 = m_used == -INFINITY ? 0.0F : exp2_fast(m_used - top);
                float sum = l_part * f0;
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    f[i] = ml[i].x == -INFINITY ? 0.0F : exp2_fast(ml[i].x - top);
                    sum += ml[i].y * f[i];
                }
                const bool direct = w.x == 0 && n == w.units && !p.logits;
                const float inv = direct ? (sum == 0.0F ? 0.0F : 1.0F / sum) : 1.0F;
                const size_t pair = static_cast<size_t>(w.b) * subs + w.sub;
                const size_t index = (blockIdx.x + pair) * kHeads + row;
                float* part = p.part.o + index * D;
                bf16* dst = static_cast<bf16*>(p.out) + (row0 + row) * D;
                if (row < heads) {
                    if (!direct && quad == 0) *reinterpret_cast<float2*>(p.part.ml + index * 2) = make_float2(top, sum);
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) {
                        float a = o[j][0] * f0, c = o[j][1] * f0;
#pragma unroll
                        for (int i = 0; i < 3; ++i) {
                            const float2 v = *reinterpret_cast<const float2*>(merge_o + (i * kHeads + row) * D + 8 * j + 2 * quad);
                            a = fmaf(v.x, f[i], a);
                            c = fmaf(v.y, f[i], c);
                        }
                        if (direct) *reinterpret_cast<__nv_bfloat162*>(dst + 8 * j + 2 * quad) = __floats2bfloat162_rn(a * inv, c * inv);
                        else *reinterpret_cast<float2*>(part + 8 * j + 2 * quad) = make_float2(a, c);
                    }
                }
                if (lane == 0 && w.x == 0) {   // the owner of the pair's first unit; all ranges but the last have one length
                    const int per = start[4], beyond = w.units - n;
                    p.part.span[pair] = make_int2(blockIdx.x, blockIdx.x + (beyond + per - 1) / per);
                }
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&merge_bar[1]));
            }
            ++n_piece;
            w.advance(p, subs, n);
        }
    }
    __syncthreads();
    if (*abort_flag)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);  // let copies in flight land before the CTA exits
}

template <int D>
sfb_status launch_mma(const StepParams& p, const StepPlan& plan, cudaStream_t stream) {
    const PagedView& kv = p.kv;
    CUtensorMap mk, mv;
    const int pool_rows = kv.num_blocks * kv.kv_heads * kv.block_tokens;
    if (!encode_tensor_map_bf16_2d(&mk, kv.k_pool, pool_rows, D, U, 64) || !encode_tensor_map_bf16_2d(&mv, kv.v_pool, pool_rows, D, U, 64))
        return SFB_CUDA_ERROR;
    constexpr int smem = Shape<D>::kStages * Shape<D>::kStageBytes + 3 * kHeads * (D * 4 + 8) + Shape<D>::kStages * (kUnits * 8 + 16) + 64 + 1024;
    static_assert(2 * (smem + 1024) <= 228 * 1024, "two CTAs per SM");
    SFB_CUDA(cudaFuncSetAttribute(step_mma_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    SFB_CUDA(launch_dependent(step_mma_kernel<D>, dim3(plan.ctas), dim3(kThreads), smem, stream, mk, mv, p, pool_rows));
    return check_launch("attention_step_mma");
}

}  // namespace

sfb_status step_mma(const StepParams& p, const StepPlan& plan, cudaStream_t stream) {
    return p.kv.dim == 128 ? launch_mma<128>(p, plan, stream) : launch_mma<64>(p, plan, stream);
}

}  // namespace sfb
