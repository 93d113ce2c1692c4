// Tree attention on the 5th-generation tensor cores (bf16, head_dim = head_dim_value = 128 or 64, blocks of a multiple
// of eight tokens).
//
// The query rows of one (sequence, K/V head) - the group's heads times the nodes - are the M dimension: 128 rows fill
// an MMA tile however few are live, which costs nothing while the K/V bytes bound the time (a 128-key tile of K and V
// is 64 KB, 1.45 us of one SM's share of the HBM rate; its two products take 0.55 us of the tensor pipe).
// Keys are walked in tiles of 128: the committed positions (gathered from the pool by TMA, one box per run of
// tokens inside a block), then the drafted nodes (their own tensors; a row's ancestors as bits).
//
// Work is cut evenly: the tiles of all (sequence, K/V head, row group) pairs are laid end to end and every CTA takes
// one equal range, so ragged contexts leave no SM idle.  A pair that lies in one CTA writes its output
// directly; the pieces of a pair that was cut are kept as (maximum, sum, numerator) and joined by a second kernel.
//
// 384 threads, roles as in the prefill kernel: two softmax groups of 128 threads (thread = row = tensor-memory lane),
// two copy warps (Q and K, V), one MMA warp; S and P share tensor memory columns, P is the A operand of P.V.
//   ROWS = 256: the two groups own two 128-row tiles and meet every key tile;
//   ROWS = 128: both own the same rows and take alternate key tiles, each with its own running maximum and
//               accumulator; the first group joins them at the end of a piece, out of tensor memory.
// A slot's scores of the next tile are issued behind its P.V of this one, since P lies over them.  Taken in two steps of 64 keys
// (two S/P areas a slot), one step's products run under the softmax of the other, at the price of N = 64 products, which read
// Q from shared memory twice as often: 69 -> 61 us for 8 sequences of 8192 tokens, one node, 128 elements a head.  It does not
// pay with two row tiles, where the other tile's products fill the time already (113 -> 123 us with 256 rows), nor at 64
// elements a head, where the products are half as long (44 -> 50 us).
// Positions past the context in a loaded block may hold anything: their scores are masked and their V rows are zeroed
// in shared memory before the product (0 * NaN).  Warps without a live row skip the arithmetic.  Waits are bounded.
#include "attention_tree.cuh"
#include "ptx_sm100.cuh"

namespace sfb {
namespace {

constexpr int KT = 128;
constexpr int kThreads = 384;
constexpr int kHalfBytes = KT * 64 * 2;
constexpr uint32_t kTmemCols = 512;   // S_th (P_th over its first half) at t * 128 + h * 64, O_t at 256 + t * D
constexpr uint32_t kOCol = 256;
constexpr uint32_t kCodeTree = 0x80;
constexpr float kRescaleThreshold = 8.0F;  // log2 units
constexpr int kBadRing = 16;

template <int D, int ROWS>
struct Shape {
    static constexpr int kHalves = D / 64;
    static constexpr int kQTiles = ROWS / 128;
    // A tile of keys is taken in one step or in two: see the head of the file.
    static constexpr int kSteps = ROWS == 128 && D == 128 ? 2 : 1, kKeys = KT / kSteps;
    static constexpr int kQBytes = kHalves * kHalfBytes;   // one 128-row tile
    static constexpr int kTileBytes = kHalves * kHalfBytes;
    static constexpr int kStages = D == 64 ? 5 : (ROWS == 128 ? 3 : 2);
    static constexpr int kParentBytes = 2 * SFB_MAX_TREE_NODES;
    static constexpr int kSmemBytes = kQTiles * kQBytes + 2 * kStages * kTileBytes + kParentBytes + 128 * 8 + 512 + 1024;
};

struct TreeTcParams {
    TreeParams t;
    int rows_all, row_groups, box_rows;
    int64_t pairs;
    int pool_rows;
    float* part_o;          // [2 * grid][ROWS][D], by piece_of
    float2* part_ml;        // [2 * grid][ROWS]
    int2* pair_span;        // [pairs]: first and last CTA
};

// Place of a cut pair's piece: a CTA has at most one pair that began before it and one that begins in it and goes on.
__device__ __forceinline__ int64_t piece_of(int cta, bool begins) { return 2 * static_cast<int64_t>(cta) + (begins ? 1 : 0); }

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Two float32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\nfma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ int tiles_of(int ctx, int count) {
    return count > 0 ? (ctx + KT - 1) / KT + (count + KT - 1) / KT : 0;
}

// Position of a role in the CTA's range of tiles.
struct Walk {
    int b, sub, x, ctx, count, tiles;  // sub = kvh * row_groups + row group
    int64_t left;

    __device__ __forceinline__ void read(const TreeTcParams& p) {
        tree_sizes(p.t, b, ctx, count, false);
        tiles = tiles_of(ctx, count);
    }
    __device__ __forceinline__ int take() const { return static_cast<int>(left < tiles - x ? left : tiles - x); }
    __device__ __forceinline__ void advance(const TreeTcParams& p, int n) {
        left -= n;
        x += n;
        if (x < tiles || left <= 0) return;
        x = 0;
        if (++sub < p.t.kv.kv_heads * p.row_groups) return;
        sub = 0;
        do {
            if (++b >= p.t.batch) { left = 0; return; }
            read(p);
        } while (tiles == 0);
    }
};

template <int D, int ROWS>
__global__ void __launch_bounds__(kThreads, 1)
tree_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_dk,
                    const __grid_constant__ CUtensorMap map_dv, const __grid_constant__ TreeTcParams p) {
    using Sh = Shape<D, ROWS>;
    constexpr int kStages = Sh::kStages, kHalves = Sh::kHalves, kTileBytes = Sh::kTileBytes;
    constexpr bool kTwoTiles = ROWS == 256;
    constexpr int kSteps = Sh::kSteps, KH = Sh::kKeys;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_smem = smem;
    uint8_t* k_smem = q_smem + Sh::kQTiles * Sh::kQBytes;
    uint8_t* v_smem = k_smem + kStages * kTileBytes;
    uint8_t* parent_smem = v_smem + kStages * kTileBytes;                           // [2][256], 255 = no parent
    float2* ml_smem = reinterpret_cast<float2*>(parent_smem + Sh::kParentBytes);    // [128]
    uint64_t* bars = reinterpret_cast<uint64_t*>(ml_smem + 128);
    uint64_t* q_full = bars;
    uint64_t* q_empty = bars + 1;
    uint64_t* s_full = bars + 2;     // [2][2]: scores of slot t, step h; with two steps, h = 0 once more behind a piece's last tile
    uint64_t* p_full = bars + 6;     // [2][2]
    uint64_t* par_full = bars + 10;  // [2]
    uint64_t* ml_full = bars + 12;   // group 1's maxima and sums are in shared memory
    uint64_t* o_free = bars + 13;    // group 0 has read group 1's accumulator
    uint64_t* o_full = bars + 14;    // [2]
    uint64_t* k_full = bars + 16;
    uint64_t* k_empty = k_full + kStages;
    uint64_t* v_full = k_empty + kStages;
    uint64_t* v_empty = v_full + kStages;
    uint32_t* words = reinterpret_cast<uint32_t*>(v_empty + kStages);
    uint32_t* tmem_slot = words;
    volatile uint32_t* abort_flag = words + 1;
    int* start = reinterpret_cast<int*>(words + 2);   // even_range: b, sub, x, tiles in the range, tiles of a full range
    volatile uint32_t* bad = words + 8;               // [kBadRing], runs of eight keys without a block
    const TreeParams& t_ = p.t;
    const PagedView& kv = t_.kv;
    uint32_t* status = kv.status;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        ptx::mbar_init(ptx::smem_u32(q_full), 1);
        ptx::mbar_init(ptx::smem_u32(q_empty), 1);
        for (int t = 0; t < 2; ++t) {
            for (int h = 0; h < 2; ++h) {
                ptx::mbar_init(ptx::smem_u32(&s_full[2 * t + h]), 1);
                ptx::mbar_init(ptx::smem_u32(&p_full[2 * t + h]), 128);
            }
            ptx::mbar_init(ptx::smem_u32(&o_full[t]), 1);
            ptx::mbar_init(ptx::smem_u32(&par_full[t]), 128);
        }
        ptx::mbar_init(ptx::smem_u32(ml_full), 128);
        ptx::mbar_init(ptx::smem_u32(o_free), 128);
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(ptx::smem_u32(&k_full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&k_empty[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&v_full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&v_empty[s]), 1);
        }
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async();
        ptx::prefetch_tensormap(&map_q);
        ptx::prefetch_tensormap(&map_k);
        ptx::prefetch_tensormap(&map_v);
        ptx::prefetch_tensormap(&map_dk);
        ptx::prefetch_tensormap(&map_dv);
    }
    if (warp == 9) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_slot), kTmemCols);
        ptx::tmem_relinquish();
    }
    grid_dependency_wait();
    if (warp == 10) {
        even_range(t_.batch, static_cast<int64_t>(kv.kv_heads) * p.row_groups, 1,
                   [&](int b) {
                       int ctx, count;
                       tree_sizes(t_, b, ctx, count, blockIdx.x == 0);   // (the first CTA reports for all sequences)
                       return tiles_of(ctx, count);
                   }, start);
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    Walk w{};
    w.left = start[3];
    if (w.left > 0) {
        w.b = start[0]; w.sub = start[1]; w.x = start[2];
        w.read(p);
    }

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (warp == 8 || warp == 11) {
            // ------------------------------------------------------------ copies: warp 8 Q and K, warp 11 V
            const bool keys = warp == 8;
            uint64_t* empty = keys ? k_empty : v_empty;
            uint64_t* full = keys ? k_full : v_full;
            uint8_t* ring = keys ? k_smem : v_smem;
            const CUtensorMap* map_pool = keys ? &map_k : &map_v;
            const CUtensorMap* map_draft = keys ? &map_dk : &map_dv;
            const int boxes = KT / p.box_rows;
            const int box = lane / kHalves, half = lane % kHalves;
            const uint32_t box_bits = (p.box_rows == 128 ? 0xffffu : ((1u << (p.box_rows / 8)) - 1));
            uint32_t n_kv = 0, n_seg = 0;
            const auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
                return __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(bar), parity, abort_flag, status, kCodeTree | 1));
            };
            bool ok = true;
            while (ok && w.left > 0) {
                const int n = w.take();
                const int kvh = w.sub / p.row_groups, rg = w.sub % p.row_groups;
                const int n_ctx = (w.ctx + KT - 1) / KT;
                const int head = w.b * kv.kv_heads + kvh;
                const int* table = kv.table + static_cast<size_t>(w.b) * kv.max_blocks;
                const auto row_of = [&](int x) -> int {   // pool row of this lane's box in context tile x, -1: no block, -2: nothing to load
                    const int pos = x * KT + box * p.box_rows;
                    if (x >= n_ctx || box >= boxes || pos >= w.ctx) return -2;
                    const int block = kv.block_of(pos);
                    const int page = table[block];
                    return page < 0 || page >= kv.num_blocks ? -1
                                                             : (page * kv.kv_heads + kvh) * kv.block_tokens + (pos - block * kv.block_tokens);
                };
                int row = row_of(w.x);
                if (keys) {
                    ok = wait(q_empty, (n_seg & 1) ^ 1);
                    if (!ok) break;
                    if (lane == 0) {
                        const uint32_t bar = ptx::smem_u32(q_full);
                        ptx::mbar_expect_tx(bar, Sh::kQTiles * Sh::kQBytes);
                        const int q_row = head * p.rows_all + rg * ROWS;
                        for (int i = 0; i < Sh::kQTiles; ++i)
                            for (int h = 0; h < kHalves; ++h)
                                ptx::tma_load_2d(ptx::smem_u32(q_smem + i * Sh::kQBytes + h * kHalfBytes), &map_q, bar, 64 * h, q_row + 128 * i);
                    }
                    ++n_seg;
                }
                for (int x = w.x; x < w.x + n; ++x, ++n_kv) {
                    const int s = n_kv % kStages;
                    const int mine = row;
                    row = x + 1 < w.x + n ? row_of(x + 1) : -2;    // in flight while this tile waits for its stage
                    const bool draft = x >= n_ctx;
                    const uint32_t missing = __reduce_or_sync(0xffffffffu, mine == -1 ? box_bits << (box * (p.box_rows / 8)) : 0u);
                    const uint32_t loaded = __popc(__ballot_sync(0xffffffffu, mine > -2)) * (p.box_rows * 128);
                    if (missing && lane == 0) atomicOr(status, kCodeDecodeBounds);
                    ok = wait(&empty[s], ((n_kv / kStages) & 1) ^ 1);
                    if (!ok) break;
                    const uint32_t bar = ptx::smem_u32(&full[s]), stage = ptx::smem_u32(ring + s * kTileBytes);
                    if (lane == 0) {
                        if (keys) bad[n_kv % kBadRing] = missing;
                        ptx::mbar_expect_tx(bar, draft ? kTileBytes : loaded);
                    }
                    __syncwarp();
                    if (draft) {
                        if (lane < kHalves) ptx::tma_load_3d(stage + lane * kHalfBytes, map_draft, bar, 64 * lane, (x - n_ctx) * KT, head);
                    } else if (mine > -2) {   // (a row outside the tensor map reads zeros)
                        ptx::tma_load_2d(stage + half * kHalfBytes + box * p.box_rows * 128, map_pool, bar, 64 * half, mine == -1 ? p.pool_rows : mine);
                    }
                }
                w.advance(p, n);
            }
        } else if (warp == 9) {
            // ------------------------------------------------------------ MMA issue
            // (the whole warp walks along, so that the operands are uniform; one lane of it issues)
            constexpr uint32_t idesc_qk = ptx::umma_idesc_bf16(128, KH, 0, 0);
            constexpr uint32_t idesc_pv = ptx::umma_idesc_bf16(128, D, 0, 1);
            const uint64_t q_desc = ptx::umma_desc_k_sw128(ptx::smem_u32(q_smem)), k_desc = ptx::umma_desc_k_sw128(ptx::smem_u32(k_smem)),
                           v_desc = ptx::umma_desc_mn_sw128(ptx::smem_u32(v_smem), kHalfBytes, 1024);
            const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
            uint32_t n_kv = 0, n_seg = 0, p_parity = 0;   // tiles and pieces so far, parity of the uses of each P (bits)
            const auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
                return __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(bar), parity, abort_flag, status, kCodeTree | 2));
            };
            bool ok = true;
            while (ok && w.left > 0) {
                const int n = __shfl_sync(0xffffffffu, w.take(), 0);
                const int items = kTwoTiles ? 2 * n : n;
                ok = wait(q_full, n_seg & 1);
                if (!ok) break;
                // S_th = Q . K_jh^T for item i (tile j, slot t), step h
                const auto issue_qk = [&](int i, int t, int h) -> bool {
                    const uint32_t g = n_kv + (kTwoTiles ? i >> 1 : i), stage = g % kStages;
                    if (h == 0 && (!kTwoTiles || t == 0)) {   // (the others meet the tile that this one has waited for)
                        if (!wait(&k_full[stage], (g / kStages) & 1)) return false;
                        ptx::tc_fence_after();
                    }
                    // (a step along K only adds to the address field of the descriptors)
                    const uint64_t qa = q_desc + (kTwoTiles ? t : 0) * (Sh::kQBytes >> 4), ka = k_desc + stage * (kTileBytes >> 4) + h * (KH * 128 >> 4);
#pragma unroll
                    for (int half = 0; half < kHalves; ++half)
                        ptx::umma_bf16_x4_warp(tmem + t * KT + h * KH, qa + half * (kHalfBytes >> 4), ka + half * (kHalfBytes >> 4), idesc_qk, half != 0);
                    return true;
                };
                const auto after_qk = [&](int i, int t, int h) {
                    if (h < kSteps - 1) return;
                    if (!kTwoTiles || t == 1) ptx::umma_commit_warp(ptx::smem_u32(&k_empty[(n_kv + (kTwoTiles ? i >> 1 : i)) % kStages]));
                    if (i == items - 1) ptx::umma_commit_warp(ptx::smem_u32(q_empty));
                };
#pragma unroll
                for (int h = 0; h < kSteps; ++h)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (!ok || t >= items) continue;
                        ok = issue_qk(t, t, h);
                        ptx::umma_commit_warp(ptx::smem_u32(&s_full[2 * t + h]));
                        after_qk(t, t, h);
                    }
                for (int i0 = 0; ok && i0 < items; i0 += 2) {
#pragma unroll
                    for (int h = 0; h < kSteps; ++h)
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const int i = i0 + t, at = 2 * t + h;
                            if (!ok || i >= items) continue;
                            const uint32_t g = n_kv + (kTwoTiles ? i >> 1 : i), stage = g % kStages;
                            if (h == 0 && (!kTwoTiles || t == 0)) ok = wait(&v_full[stage], (g / kStages) & 1);
                            ok = ok && wait(&p_full[at], p_parity >> at & 1);
                            if (!ok) continue;
                            p_parity ^= 1u << at;
                            ptx::tc_fence_after();
                            // O_t += P_th . V_jh; then the scores of the slot's next tile (the tensor pipe runs in order: P_th is
                            // consumed before S_th is overwritten)
#pragma unroll
                            for (int k = 0; k < KH / 64; ++k)
                                ptx::umma_bf16_ts_x4_warp(tmem + kOCol + t * D, tmem + t * KT + h * KH + k * 32,
                                                          v_desc + stage * (kTileBytes >> 4) + (h * KH + k * 64) * (128 >> 4), idesc_pv, (i0 | h | k) != 0);
                            if (h == kSteps - 1 && (!kTwoTiles || t == 1) && i + 2 >= items) ptx::umma_commit_warp(ptx::smem_u32(&v_empty[stage]));
                            if (i + 2 < items) ok = issue_qk(i + 2, t, h);
                            if (i + 2 < items || h < kSteps - 1) ptx::umma_commit_warp(ptx::smem_u32(&s_full[at]));
                            else ptx::umma_commit_warp(ptx::smem_u32(&o_full[t]));
                            if (i + 2 < items) {
                                after_qk(i + 2, t, h);
                                if (h == kSteps - 1 && (!kTwoTiles || t == 1)) ptx::umma_commit_warp(ptx::smem_u32(&v_empty[stage]));
                            }
                        }
                }
                n_kv += n;
                ++n_seg;
                w.advance(p, n);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        // ---------------------------------------------------------------- softmax groups
        const int t = warp >> 2;
        const int quarter = warp & 3;
        const int r = quarter * 32 + lane;                       // tensor-memory lane
        const int tile_row = (kTwoTiles ? t * 128 : 0) + r;      // row inside the row group
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_addr = tmem_base + lane_base + t * KT;
        const uint32_t o_addr = tmem_base + lane_base + kOCol + t * D;
        uint8_t* parent = parent_smem + t * SFB_MAX_TREE_NODES;
        uint32_t n_kv = 0, n_first = 0, n_second = 0, n_out = 0, n_seg = 0, n_par = 0;   // n_first, n_second: uses of s_full
        bool ok = true;
        while (ok && w.left > 0) {
            const int n = w.take();
            const int kvh = w.sub / p.row_groups, rg = w.sub % p.row_groups;
            const int n_ctx = (w.ctx + KT - 1) / KT;
            const int row = rg * ROWS + tile_row;                // query row of the pair
            const int node = row % t_.nodes;
            const bool live_row = row < p.rows_all && node < w.count;
            const bool live_warp = __any_sync(0xffffffffu, live_row);
            float m_used = -INFINITY, row_sum = 0.0F;
            int used = 0;
            for (int j = kTwoTiles ? 0 : t; ok && j < n; j += kTwoTiles ? 1 : 2, ++used) {
                const int x = w.x + j;
                const uint32_t g = n_kv + j;
                const bool draft = x >= n_ctx;
                if (draft) {   // parents come in while the scores are computed
                    for (int i = r; i < w.count; i += 128) {
                        int up = t_.parents[static_cast<size_t>(w.b) * t_.nodes + i];
                        if (up < -1 || up >= i) {
                            up = -1;
                            atomicOr(status, kCodeDecodeBounds);
                        }
                        parent[i] = static_cast<uint8_t>(up);   // (-1 becomes 255; a parent is at most 254)
                    }
                    ptx::mbar_arrive(ptx::smem_u32(&par_full[t]));
                }
                ok = ptx::mbar_wait(ptx::smem_u32(&s_full[2 * t]), n_first & 1, abort_flag, status, kCodeTree | 4);
                if (!ok) break;
                ptx::tc_fence_after();
                const int key0 = draft ? (x - n_ctx) * KT : x * KT;
                const int live = min(KT, (draft ? w.count : w.ctx) - key0);
                uint32_t see[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
                bool masked = live < KT;
                if (draft) {
                    masked = true;
                    ok = ptx::mbar_wait(ptx::smem_u32(&par_full[t]), n_par & 1, abort_flag, status, kCodeTree | 4);
                    if (!ok) break;
                    ++n_par;
                    see[0] = see[1] = see[2] = see[3] = 0u;
                    for (int i = live_row ? node : -1; i >= 0;) {
                        const int at = i - key0;
                        if (at >= 0 && at < KT) {
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                if (at >> 5 == q) see[q] |= 1u << (at & 31);
                        }
                        const int up = parent[i];
                        i = up == 255 ? -1 : up;
                    }
                } else {
                    const uint32_t missing = bad[g % kBadRing];
                    if (live < KT || missing) {
                        masked = true;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int left = live - 32 * q;
                            uint32_t bits = left >= 32 ? 0xffffffffu : (left > 0 ? (1u << left) - 1 : 0u);
#pragma unroll
                            for (int u = 0; u < 4; ++u)
                                if (missing >> (4 * q + u) & 1u) bits &= ~(0xffu << (8 * u));
                            see[q] = bits;
                        }
                    }
                }
                if (live < KT) {
                    // rows of V past the live keys: whatever the block (or the stage) holds becomes zero
                    ok = ptx::mbar_wait(ptx::smem_u32(&v_full[g % kStages]), (g / kStages) & 1, abort_flag, status, kCodeTree | 4);
                    if (!ok) break;
                    uint8_t* v_tile = v_smem + (g % kStages) * kTileBytes;
                    for (int i = r; i < (KT - live) * 8 * kHalves; i += 128) {
                        const int piece = i & 7, half = (i >> 3) % kHalves, dead = live + (i >> 3) / kHalves;
                        *reinterpret_cast<uint4*>(v_tile + half * kHalfBytes + dead * 128 + piece * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    ptx::fence_proxy_async();
                }
#pragma unroll
                for (int h = 0; h < kSteps; ++h) {
                    if (h == 1) {
                        ok = ptx::mbar_wait(ptx::smem_u32(&s_full[2 * t + 1]), n_second & 1, abort_flag, status, kCodeTree | 4);
                        if (!ok) break;
                        ptx::tc_fence_after();
                    }
                    if (live_warp) {
                        uint32_t raw[KH / 32][32];
#pragma unroll
                        for (int c = 0; c < KH / 32; ++c) ptx::tmem_ld_32x32(s_addr + h * KH + c * 32, raw[c]);
                        ptx::tmem_ld_wait();
                        if (masked) {
#pragma unroll
                            for (int c = 0; c < KH / 32; ++c)
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                    if (!(see[h * (KH / 32) + c] >> i & 1u)) raw[c][i] = 0xff800000u;  // -inf, and 2^-inf = 0 below
                        }
                        float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
                        for (int c = 0; c < KH / 32; ++c)
#pragma unroll
                            for (int i = 0; i < 32; i += 8) {
                                const uint32_t* v = &raw[c][i];
                                mx0 = max3(mx0, __uint_as_float(v[0]), __uint_as_float(v[1]));
                                mx1 = max3(mx1, __uint_as_float(v[2]), __uint_as_float(v[3]));
                                mx2 = max3(mx2, __uint_as_float(v[4]), __uint_as_float(v[5]));
                                mx3 = max3(mx3, __uint_as_float(v[6]), __uint_as_float(v[7]));
                            }
                        const float step_max = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * t_.scale_log2;
                        // lazy running maximum: O_t is only touched when it outgrows the one in use by 2^8.  With one step to a
                        // tile every earlier product of the slot has finished when S_t is complete; with two the one of the step
                        // before may still run, and what is committed behind it is the other step's next scores.
                        const bool grow = step_max > m_used + kRescaleThreshold;
                        if ((used > 0 || h > 0) && __any_sync(0xffffffffu, grow)) {
                            if (kSteps == 2) {
                                ok = ptx::mbar_wait(ptx::smem_u32(&s_full[2 * t + 1 - h]), (h == 0 ? n_second : n_first + 1) & 1, abort_flag, status, kCodeTree | 4);
                                ok = __all_sync(0xffffffffu, ok);
                                if (!ok) break;
                                ptx::tc_fence_after();
                            }
                            const float alpha = grow ? exp2_fast(m_used - step_max) : 1.0F;
#pragma unroll 1
                            for (int c = 0; c < D / 32; ++c) {
                                uint32_t o[32];
                                ptx::tmem_ld_32x32(o_addr + c * 32, o);
                                ptx::tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                                ptx::tmem_st_32x32(o_addr + c * 32, o);
                            }
                            ptx::tmem_st_wait();
                            row_sum *= alpha;
                        }
                        if (grow) m_used = step_max;
                        const float neg_m = m_used == -INFINITY ? 0.0F : -m_used;
                        float2 s0 = make_float2(0.0F, 0.0F), s1 = s0;
                        const float2 scale = make_float2(t_.scale_log2, t_.scale_log2), shift = make_float2(neg_m, neg_m);
#pragma unroll
                        for (int c = 0; c < KH / 32; ++c) {
                            uint32_t packed[16];
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                float2 x = fma2(make_float2(__uint_as_float(raw[c][i]), __uint_as_float(raw[c][i + 1])), scale, shift);
                                float2 y = fma2(make_float2(__uint_as_float(raw[c][i + 2]), __uint_as_float(raw[c][i + 3])), scale, shift);
                                x = make_float2(exp2_fast(x.x), exp2_fast(x.y));
                                y = make_float2(exp2_fast(y.x), exp2_fast(y.y));
                                s0 = add2(s0, x);
                                s1 = add2(s1, y);
                                // the weights are rounded to bf16 for the product; the row sum keeps 32 bits
                                const __nv_bfloat162 lo = __floats2bfloat162_rn(x.x, x.y), hi = __floats2bfloat162_rn(y.x, y.y);
                                packed[i / 2] = *reinterpret_cast<const uint32_t*>(&lo);
                                packed[i / 2 + 1] = *reinterpret_cast<const uint32_t*>(&hi);
                            }
                            ptx::tmem_st_32x16(s_addr + h * KH + c * 16, packed);
                        }
                        ptx::tmem_st_wait();
                        row_sum += (s0.x + s0.y) + (s1.x + s1.y);
                    }
                    ptx::tc_fence_before();
                    ptx::mbar_arrive(ptx::smem_u32(&p_full[2 * t + h]));
                }
                if (!ok) break;
                ++n_first;
                ++n_second;
            }
            if (ok && used > 0) {
                ok = ptx::mbar_wait(ptx::smem_u32(&o_full[t]), n_out & 1, abort_flag, status, kCodeTree | 4);
                ++n_out;
                if (kSteps == 2) ++n_first;
                ptx::tc_fence_after();
            }
            if (!ok) break;
            // ---- the piece's result
            float f0 = 1.0F, f1 = 0.0F;     // factors of this group's and (ROWS == 128) the other group's accumulator
            if constexpr (!kTwoTiles) {
                if (t == 1) {
                    ml_smem[r] = make_float2(m_used, row_sum);
                    ptx::mbar_arrive(ptx::smem_u32(ml_full));
                    ok = ptx::mbar_wait(ptx::smem_u32(o_free), n_seg & 1, abort_flag, status, kCodeTree | 4);
                } else {
                    ok = ptx::mbar_wait(ptx::smem_u32(ml_full), n_seg & 1, abort_flag, status, kCodeTree | 4);
                    if (!ok) break;
                    ptx::tc_fence_after();
                    const float2 other = ml_smem[r];
                    const float top = fmaxf(m_used, other.x);
                    f0 = m_used == -INFINITY ? 0.0F : exp2_fast(m_used - top);
                    f1 = other.x == -INFINITY ? 0.0F : exp2_fast(other.x - top);
                    row_sum = row_sum * f0 + other.y * f1;
                    m_used = top;
                }
                if (!ok) break;
            }
            const bool whole = w.x == 0 && n == w.tiles;
            const int64_t pair = static_cast<int64_t>(w.b) * kv.kv_heads * p.row_groups + w.sub;
            if ((kTwoTiles || t == 0) && live_warp) {
                const float inv = whole ? (row_sum == 0.0F ? 0.0F : 1.0F / row_sum) : 1.0F;
                f0 *= inv;
                f1 *= inv;
                const bool second = !kTwoTiles && n > 1;
                const int64_t piece = piece_of(blockIdx.x, w.x == 0);
                bf16* dst = static_cast<bf16*>(t_.out) +
                            tree_out_row(t_, w.b, kvh * (t_.q_heads / kv.kv_heads) + row / t_.nodes, node) * D;
                float* part = p.part_o + (piece * ROWS + tile_row) * D;
                if (!whole && live_row) p.part_ml[piece * ROWS + tile_row] = make_float2(m_used, row_sum);
#pragma unroll 2
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32], o2[32];
                    ptx::tmem_ld_32x32(o_addr + c * 32, o);
                    if (second) ptx::tmem_ld_32x32(o_addr + D + c * 32, o2);
                    ptx::tmem_ld_wait();
                    float v[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        v[i] = __uint_as_float(o[i]) * f0;
                        if (second && f1 != 0.0F) v[i] = fmaf(__uint_as_float(o2[i]), f1, v[i]);
                    }
                    if (!live_row) continue;
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint4 packed;
                            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&packed);
#pragma unroll
                            for (int k = 0; k < 4; ++k) h[k] = __floats2bfloat162_rn(v[8 * i + 2 * k], v[8 * i + 2 * k + 1]);
                            reinterpret_cast<uint4*>(dst + c * 32)[i] = packed;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            reinterpret_cast<float4*>(part + c * 32)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                    }
                }
            }
            if (!kTwoTiles && t == 0) {
                ptx::tc_fence_before();
                ptx::mbar_arrive(ptx::smem_u32(o_free));
            }
            if (threadIdx.x == 0 && w.x == 0) {   // (one thread per pair: the owner of its first tile)
                // (all ranges but the last have one length: the last CTA of the pair follows from it)
                const int64_t per = start[4];
                const int64_t beyond = w.tiles - n;
                p.pair_span[pair] = make_int2(blockIdx.x, static_cast<int>(blockIdx.x + (beyond + per - 1) / per));
            }
            n_kv += n;
            ++n_seg;
            w.advance(p, n);
        }
    }

    __syncwarp();
    ptx::tc_fence_before();
    __syncthreads();
    if (*abort_flag)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);  // copies in flight land before the CTA leaves
    if (warp == 9) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem_base, kTmemCols);
    }
}

// Joins the pieces of pairs that were cut: one warp per query row, which reads up to kAtOnce pieces at the same time.  Eight
// where all CTAs are on the GPU at once (8 rows, 5 pieces: 11.1 us with the attention, 11.7 with four), else four, with five CTAs
// an SM instead of three (2048 CTAs of 2 to 4 pieces: 111.4 -> 109.1 us).
template <int D, int kAtOnce>
__global__ void __launch_bounds__(256, kAtOnce == 4 ? 5 : 1)
tree_join_kernel(const __grid_constant__ TreeTcParams p, int rows_cta) {
    constexpr int V = D / 32;
    const TreeParams& t = p.t;
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const int slices = rows_cta / 8;
    const int64_t pair = blockIdx.x / slices;
    const int tile_row = (blockIdx.x % slices) * 8 + (threadIdx.x >> 5);
    const int subs = t.kv.kv_heads * p.row_groups;
    const int b = static_cast<int>(pair / subs), sub = static_cast<int>(pair % subs);
    const int kvh = sub / p.row_groups, rg = sub % p.row_groups;
    const int row = rg * rows_cta + tile_row, node = row % t.nodes;
    if (row >= p.rows_all) return;
    const int2 span = p.pair_span[pair];      // (not written where the sequence has no nodes; then the count is 0)
    if (node >= tree_node_count(t, b)) return;
    if (span.x == span.y) return;   // written by the attention kernel itself
    const auto index = [&](int c) { return piece_of(c, c == span.x) * rows_cta + tile_row; };
    float2 ml[kAtOnce];
    float part[kAtOnce][V];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
        ml[i] = make_float2(-INFINITY, 0.0F);
        if (span.x + i > span.y) continue;
        ml[i] = p.part_ml[index(span.x + i)];
        const float* at = p.part_o + index(span.x + i) * D + lane * V;
#pragma unroll
        for (int k = 0; k < V; k += 2) {
            const float2 v = *reinterpret_cast<const float2*>(at + k);
            part[i][k] = v.x;
            part[i][k + 1] = v.y;
        }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) top = fmaxf(top, ml[i].x);
    for (int c = span.x + kAtOnce; c <= span.y; ++c) top = fmaxf(top, p.part_ml[index(c)].x);
    float sum = 0.0F, acc[V] = {};
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
        if (ml[i].x == -INFINITY) continue;
        const float f = exp2_fast(ml[i].x - top);
        sum = fmaf(ml[i].y, f, sum);
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = fmaf(part[i][k], f, acc[k]);
    }
    for (int c = span.x + kAtOnce; c <= span.y; ++c) {
        const float2 more = p.part_ml[index(c)];
        if (more.x == -INFINITY) continue;
        const float f = exp2_fast(more.x - top);
        sum = fmaf(more.y, f, sum);
        const float* at = p.part_o + index(c) * D + lane * V;
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = fmaf(at[k], f, acc[k]);
    }
    const float inv = sum == 0.0F ? 0.0F : 1.0F / sum;
    bf16* dst = static_cast<bf16*>(t.out) + tree_out_row(t, b, kvh * (t.q_heads / t.kv.kv_heads) + row / t.nodes, node) * D + lane * V;
#pragma unroll
    for (int i = 0; i < V; i += 2) *reinterpret_cast<__nv_bfloat162*>(dst + i) = __floats2bfloat162_rn(acc[i] * inv, acc[i + 1] * inv);
}

struct TcLayout {
    int rows_all, rows_cta, row_groups, grid;
    int64_t pairs;
    size_t ml, span, total;   // part_o first
};

TcLayout tc_layout(const sfb_tree_args& a) {
    TcLayout l{};
    l.rows_all = a.q_heads / a.kv_heads * a.nodes;
    l.rows_cta = l.rows_all <= 128 ? 128 : 256;
    l.row_groups = ceil_div(l.rows_all, l.rows_cta);
    l.pairs = static_cast<int64_t>(a.batch) * a.kv_heads * l.row_groups;
    const int covered = a.max_blocks * a.block_tokens;
    const int limit = a.max_context < covered ? a.max_context : covered;
    const int64_t most = l.pairs * (ceil_div(limit, KT) + ceil_div(a.nodes, KT));
    int ctas = sm_count();
    if (a.splits > 0 && l.pairs * a.splits < ctas) ctas = static_cast<int>(l.pairs * a.splits);
    l.grid = static_cast<int>(most < ctas ? most : ctas);
    const size_t pieces = 2 * static_cast<size_t>(l.grid);
    l.ml = sizeof(float) * pieces * l.rows_cta * a.head_dim;
    l.span = l.ml + sizeof(float2) * pieces * l.rows_cta;
    l.total = l.span + sizeof(int2) * static_cast<size_t>(l.pairs);
    return l;
}

template <int D, int ROWS>
sfb_status launch_tc(const sfb_tree_args& a, const TcLayout& l, TreeTcParams& p, cudaStream_t stream) {
    CUtensorMap mq, mk, mv, mdk, mdv;
    const uint64_t heads = static_cast<uint64_t>(a.batch) * a.kv_heads;
    if (!encode_tensor_map_bf16_2d(&mq, a.q, heads * l.rows_all, D, 128, 64) ||
        !encode_tensor_map_bf16_2d(&mk, a.k_pool, p.pool_rows, D, p.box_rows, 64) ||
        !encode_tensor_map_bf16_2d(&mv, a.v_pool, p.pool_rows, D, p.box_rows, 64) ||
        !encode_tensor_map_bf16_3d(&mdk, a.draft_k, D, a.nodes, heads, D, static_cast<uint64_t>(a.nodes) * D, 64, KT, 1) ||
        !encode_tensor_map_bf16_3d(&mdv, a.draft_v, D, a.nodes, heads, D, static_cast<uint64_t>(a.nodes) * D, 64, KT, 1))
        return SFB_CUDA_ERROR;
    constexpr int smem = Shape<D, ROWS>::kSmemBytes;
    static_assert(smem <= 227 * 1024, "shared memory of one SM");
    SFB_CUDA(cudaFuncSetAttribute(tree_tcgen05_kernel<D, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    SFB_CUDA(launch_dependent(tree_tcgen05_kernel<D, ROWS>, dim3(l.grid), dim3(kThreads), smem, stream, mq, mk, mv, mdk, mdv, p));
    SFB_TRY(check_launch("attention_tree_tcgen05"));
    const dim3 join(static_cast<unsigned>(l.pairs * (ROWS / 8)));
    if (join.x <= 3u * static_cast<unsigned>(sm_count())) SFB_CUDA(launch_dependent(tree_join_kernel<D, 8>, join, dim3(256), 0, stream, p, ROWS));
    else SFB_CUDA(launch_dependent(tree_join_kernel<D, 4>, join, dim3(256), 0, stream, p, ROWS));
    return check_launch("attention_tree_join");
}

}  // namespace

bool tree_tcgen05_shape(const sfb_tree_args& a) {
    const int64_t pool_rows = static_cast<int64_t>(a.num_blocks) * a.kv_heads * a.block_tokens;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.q_heads * a.nodes;
    return a.dtype == SFB_BF16 && (a.head_dim == 128 || a.head_dim == 64) && a.head_dim_value == a.head_dim &&
           a.block_tokens % 8 == 0 && pool_rows < (int64_t{1} << 30) && rows < (int64_t{1} << 26);
}

bool tree_tcgen05_supported(const sfb_tree_args& a) {
    return tree_tcgen05_shape(a) && aligned16(a.q) && aligned16(a.k_pool) && aligned16(a.v_pool) && aligned16(a.draft_k) &&
           aligned16(a.draft_v) && aligned16(a.out);
}

size_t tree_tcgen05_workspace(const sfb_tree_args& a) { return tc_layout(a).total; }

sfb_status tree_tcgen05(const sfb_tree_args& a, const TreeParams& t, cudaStream_t stream) {
    const TcLayout l = tc_layout(a);
    TreeTcParams p{};
    p.t = t;
    p.rows_all = l.rows_all; p.row_groups = l.row_groups; p.pairs = l.pairs;
    p.box_rows = 8;
    while (p.box_rows < 128 && a.block_tokens % (2 * p.box_rows) == 0) p.box_rows *= 2;
    p.pool_rows = a.num_blocks * a.kv_heads * a.block_tokens;
    char* ws = static_cast<char*>(a.workspace);
    p.part_o = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(ws + l.ml);
    p.pair_span = reinterpret_cast<int2*>(ws + l.span);
    if (a.head_dim == 128)
        return l.rows_cta == 128 ? launch_tc<128, 128>(a, l, p, stream) : launch_tc<128, 256>(a, l, p, stream);
    return l.rows_cta == 128 ? launch_tc<64, 128>(a, l, p, stream) : launch_tc<64, 256>(a, l, p, stream);
}

}  // namespace sfb
