// Accumulated attention weights, eviction by them, and the append of an accepted path.
//
// Weights: the decode kernel keeps every scaled logit (4 bytes per position and query head beside 4 * dim bytes of K and
// V); once the splits are merged, exp2(logit - maximum) / sum of each head is added to the running sums.
// Eviction: one CTA per (sequence, K/V head) finds the threshold of the kept weights and lists the kept rows that
// lie behind the new length and the freed slots before it.  There are equally many, and no slot is in both lists, so the
// rows can move in any order and with any parallelism.
#include <algorithm>

#include "cache_ops.cuh"
#include "select.cuh"

namespace sfb {
namespace {

// ---- weights ----------------------------------------------------------------------------------------------------

struct AddParams {
    PagedView kv;
    Partials part;
    const float *logits, *weights;
    float* weights_out;
    void* out;
    int* positions;
    const int* query_position;
    int64_t logit_stride;
    int q_heads, stride, wide;   // wide: rows of weights start on 16 bytes
};

constexpr int kAddThreads = 256;
constexpr int kAddHeads = 16;      // heads whose statistics are kept at once

// Grid (group + position chunks, K/V head, sequence).  The first `group` CTAs join the pieces of one query head each into
// its output; each of the others adds the weights of `chunk` positions (one, or a few times four a thread), whose first
// logits are fetched before the heads' maxima and sums have been worked out of the pieces.
template <class T>
__global__ void __launch_bounds__(kAddThreads)
add_weights_kernel(const __grid_constant__ AddParams p, int chunk) {
    __shared__ float factor[kMaxPieces];           // of every piece (output CTAs)
    __shared__ float half_sum[128];
    __shared__ float2 stats[kAddHeads];            // maximum, 1 / sum
    const PagedView& kv = p.kv;
    const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = p.q_heads / kv.kv_heads;
    grid_dependency_wait();
    const size_t row0 = static_cast<size_t>(b) * p.q_heads + kvh * group;
    const int ctx = kv.length(b);
    if (blockIdx.x < group) {
        const int g = blockIdx.x;
        const RowPieces r = row_pieces(p.part, kv.kv_heads, p.q_heads, b, kvh * group + g, ctx);
        if (warp == 0) row_statistics(p.part, r, factor);
        __syncthreads();
        T* dst = static_cast<T*>(p.out) + (row0 + g) * kv.dim_v;
        const int half = threadIdx.x >> 7;         // the halves of the CTA take alternate pieces
        for (int d0 = 0; d0 < kv.dim_v; d0 += 128) {
            const int d = d0 + (threadIdx.x & 127);
            float a = 0.0F;
            if (d < kv.dim_v)
#pragma unroll 8
                for (int i = half; i < r.count; i += 2) {
                    const float f = factor[i];
                    if (f != 0.0F) a = fmaf(p.part.o[(r.first + static_cast<size_t>(i) * r.step) * p.part.o_step + d], f, a);
                }
            if (half) half_sum[threadIdx.x & 127] = a;
            __syncthreads();
            if (!half && d < kv.dim_v) dst[d] = from_float<T>(a + half_sum[threadIdx.x]);
            __syncthreads();
        }
        return;
    }
    const int first = (blockIdx.x - group) * chunk, end = min(ctx, first + chunk);
    if (first >= ctx) return;
    const size_t wrow = (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.stride;
    const bool four = chunk > kAddThreads;                    // positions a thread takes, next to each other
    const int step = four ? 4 * kAddThreads : kAddThreads, t_first = first + (four ? 4 : 1) * static_cast<int>(threadIdx.x);
    const auto is_wide = [&](int t) { return four && p.wide && t + 4 <= end; };
    for (int g0 = 0; g0 < group; g0 += kAddHeads) {
        const int heads = min(kAddHeads, group - g0);
        // (later rounds of a group of more than kAddHeads heads add to what the first left)
        const float* before = g0 == 0 ? p.weights : p.weights_out;
        const float* logits = p.logits + (row0 + g0) * p.logit_stride;
        // the first four heads' logits and the old sums of the next positions are in flight under these ones' arithmetic
        float4 next[4], old_next = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
        const auto fetch = [&](int t) {
            if (!is_wide(t)) return;
            if (before) old_next = *reinterpret_cast<const float4*>(before + wrow + t);
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (g < heads) next[g] = *reinterpret_cast<const float4*>(logits + g * p.logit_stride + t);
        };
        fetch(t_first);
        __syncthreads();
        for (int g = warp; g < heads; g += kAddThreads / 32) {
            const float2 s = row_statistics(p.part, row_pieces(p.part, kv.kv_heads, p.q_heads, b, kvh * group + g0 + g, ctx), nullptr);
            if (lane == 0) stats[g] = s;
        }
        __syncthreads();
        for (int t = t_first; t < end; t += step) {
            if (is_wide(t)) {
                float4 x[4], sum = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
                const float4 old = old_next;
#pragma unroll
                for (int g = 0; g < 4; ++g) x[g] = next[g];
                fetch(t + step);
                const auto add = [&](const float4& v, int g) {
                    const float2 st = stats[g];
                    sum.x = fmaf(exp2_fast(v.x - st.x), st.y, sum.x);
                    sum.y = fmaf(exp2_fast(v.y - st.x), st.y, sum.y);
                    sum.z = fmaf(exp2_fast(v.z - st.x), st.y, sum.z);
                    sum.w = fmaf(exp2_fast(v.w - st.x), st.y, sum.w);
                };
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    if (g < heads) add(x[g], g);
#pragma unroll 4
                for (int g = 4; g < heads; ++g) add(*reinterpret_cast<const float4*>(logits + g * p.logit_stride + t), g);
                *reinterpret_cast<float4*>(p.weights_out + wrow + t) = make_float4(old.x + sum.x, old.y + sum.y, old.z + sum.z, old.w + sum.w);
            } else {
                for (int i = 0; i < (four ? 4 : 1) && t + i < end; ++i) {
                    float w = 0.0F;
#pragma unroll 4
                    for (int g = 0; g < heads; ++g) w = fmaf(exp2_fast(logits[g * p.logit_stride + t + i] - stats[g].x), stats[g].y, w);
                    p.weights_out[wrow + t + i] = (before ? before[wrow + t + i] : 0.0F) + w;
                }
            }
        }
    }
    if (p.positions && first <= ctx - 1 && ctx - 1 < end && threadIdx.x == 0) p.positions[wrow + ctx - 1] = p.query_position[b];
}

struct WeightsLayout {
    StepPlan step;
    int64_t logit_stride;
    size_t partials, total;
};

WeightsLayout weights_layout(const sfb_weights_args& a, bool wide) {
    WeightsLayout l{};
    const int covered = a.max_blocks * a.block_tokens;
    const int limit = a.max_context < covered ? a.max_context : covered;
    l.step = step_plan(a.dtype, a.head_dim, a.head_dim_value, a.batch, a.q_heads, a.kv_heads, limit, a.block_tokens, a.num_blocks,
                       a.splits, wide);
    l.logit_stride = (limit + 3) & ~3;
    l.partials = round_up16(l.step.bytes);
    l.total = l.partials + sizeof(float) * static_cast<size_t>(a.batch) * a.q_heads * l.logit_stride;
    return l;
}

sfb_status check_weights(const sfb_weights_args* a) {
    SFB_REQUIRE(a, "decode weights: null arguments");
    SFB_TRY(check_cache(a->k_pool, a->v_pool, a->block_table, a->batch, a->kv_heads, a->head_dim, a->head_dim_value,
                        a->block_tokens, a->max_blocks, a->num_blocks, a->dtype, "decode weights"));
    SFB_REQUIRE(a->q_heads > 0 && a->q_heads % a->kv_heads == 0, "invalid grouped-query attention configuration");
    SFB_REQUIRE(a->max_context > 0 && a->weight_stride >= a->max_context, "decode weights: weight_stride shorter than max_context");
    return SFB_OK;
}

// ---- eviction ------------------------------------------------------------------------------------------------------

struct EvictParams {
    PagedView kv;
    const float* weights;
    float* weights_out;
    const int* positions;
    int* positions_out;
    int* new_len;
    uint8_t* kept;         // [batch * kv_heads][max_context]
    int* moves;            // per (sequence, K/V head): old length, count, then max_moves destinations, then max_moves sources
    int max_moves, stride, budget, sink, recent, masked;   // masked: rows of at most kMaskItems slots
    int wide_items;        // longest stretch of a row shared by a cluster
};

constexpr int kEvictThreads = 1024;

// Lists the kept rows of a row that is too long for the bit mask, or has more safe positions than the budget holds: two walks in slot order,
// which rows are kept (ties go to the lower slot), then the ranks of freed slots and moved rows.
template <int THREADS, class Safe>
__device__ int evict_lists(const EvictParams& p, SelectShared& sh, const float* weights, const int* positions, float* weights_out,
                           int* positions_out, uint8_t* kept_bits, int* to, int* since, int n, int k, int room, const Threshold& t, Safe safe) {
    walk_ranks<THREADS>(sh.walk, n,
        [&](int i) {
            const bool s = safe(i);
            return (s ? 2 : 0) | (!s && room > 0 && t.cut != 0 && order_key(weights[i]) == t.low ? 1 : 0);
        },
        [&](int i, bool tie, bool s, int ties, int safes) {
            bool kept = s ? safes < k : (tie ? ties < t.cut : false);
            if (!s && !tie && room > 0) {
                const uint64_t v = order_key(weights[i]);
                kept = t.cut != 0 ? v > t.low : v >= t.low;
            }
            kept_bits[i] = kept;
        });
    __syncthreads();
    const uint64_t totals = walk_ranks<THREADS>(sh.walk, n,
        [&](int i) { return i < k ? (kept_bits[i] ? 0 : 1) : (kept_bits[i] ? 2 : 0); },
        [&](int i, bool hole, bool tail, int holes, int tails) {
            if (hole) { if (holes < p.max_moves) to[holes] = i; }
            else if (tail) { if (tails < p.max_moves) since[tails] = i; }
            else if (i < k) {
                weights_out[i] = weights[i];
                positions_out[i] = positions[i];
            }
        });
    return min(min(static_cast<int>(totals & 0xffffffffu), static_cast<int>(totals >> 32)), p.max_moves);
}

__global__ void __launch_bounds__(kEvictThreads)
evict_select_kernel(const __grid_constant__ EvictParams p) {
    __shared__ SelectShared sh;
    __shared__ int newest_of[32];
    const PagedView& kv = p.kv;
    const int b = blockIdx.y, kvh = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    const int n = kv.length(b), k = min(n, p.budget);
    const size_t row = static_cast<size_t>(b) * kv.kv_heads + kvh;
    const float* weights = p.weights + row * p.stride;
    const int* positions = p.positions + row * p.stride;
    float* weights_out = p.weights_out + row * p.stride;
    int* positions_out = p.positions_out + row * p.stride;
    int* to = p.moves + row * (2 + 2 * static_cast<size_t>(p.max_moves)) + 2;
    int* since = to + p.max_moves;
    uint8_t* kept_bits = p.kept + row * kv.limit;
    if (threadIdx.x == 0) to[-2] = n;
    if (k == n) {
        if (threadIdx.x == 0) to[-1] = 0;
        for (int i = threadIdx.x; i < n; i += kEvictThreads) {
            weights_out[i] = weights[i];
            positions_out[i] = positions[i];
        }
        return;
    }
    extern __shared__ uint32_t keys[];   // masked: positions, then the weights' keys (kForced for safe rows)
    int newest = -1;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += kEvictThreads) {
        const int at = positions[i];
        newest = max(newest, at);
        if (p.masked) keys[i] = static_cast<uint32_t>(at);
    }
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) newest_of[warp] = newest;
    __syncthreads();
    newest = __reduce_max_sync(0xffffffffu, newest_of[lane]);
    const int64_t recent_from = static_cast<int64_t>(newest) - p.recent;
    const int sink = p.sink;
    // rows kept by their position are counted first; the rest of the budget goes to the largest weights of the others
    const auto is_safe = [&](int at) { return at < sink || at > recent_from; };
    const auto safe = [&](int i) { return is_safe(positions[i]); };
    int n_safe = 0;
    if (p.masked) {
#pragma unroll 8
        for (int i = threadIdx.x; i < n; i += kEvictThreads) {   // (its own entries)
            const uint32_t key = static_cast<uint32_t>(order_key(weights[i]));
            const bool s = is_safe(static_cast<int>(keys[i]));
            keys[i] = s ? kForced : key;
            n_safe += s;
        }
    } else {
        for (int i = threadIdx.x; i < n; i += kEvictThreads) n_safe += safe(i);
    }
    n_safe = __reduce_add_sync(0xffffffffu, n_safe);
    __syncthreads();
    if (lane == 0) newest_of[warp] = n_safe;
    __syncthreads();
    n_safe = __reduce_add_sync(0xffffffffu, newest_of[lane]);
    const int room = k - n_safe;      // (positions that repeat can make more rows safe than the budget holds)
    int holes = 0;
    bool settled = false;
    if (p.masked && n_safe <= k) {
        if (room > 0) {
            settled = select_mask<kEvictThreads, true>(sh, keys, n, room, [](uint32_t&, uint32_t&) {}, [&](int j) -> uint64_t { return keys[sh.near[j]]; });
        } else {
            for (int i0 = warp * 32; i0 < n; i0 += kEvictThreads) {
                const unsigned word = __ballot_sync(0xffffffffu, i0 + lane < n && keys[i0 + lane] == kForced);
                if (lane == 0) sh.words[i0 >> 5] = word;
            }
            settled = true;
            __syncthreads();
        }
    }
    if (settled) {
        const unsigned totals = walk_bits<kEvictThreads>(sh.scan, (n + 31) / 32,
            [&](int w, unsigned& hole, unsigned& tail) {
                const int at = w * 32;
                const unsigned front = at + 32 <= k ? ~0u : (at >= k ? 0u : (1u << (k - at)) - 1);
                hole = ~sh.words[w] & front;
                tail = sh.words[w] & ~front;
            },
            [&](int i, int rank) { if (rank < p.max_moves) to[rank] = i; }, [&](int i, int rank) { if (rank < p.max_moves) since[rank] = i; });
        holes = min(min(static_cast<int>(totals & 0xffffu), static_cast<int>(totals >> 16)), p.max_moves);   // (both counts are equal)
#pragma unroll 4
        for (int i = threadIdx.x; i < k; i += kEvictThreads)
            if (sh.words[i >> 5] >> (i & 31) & 1u) {
                weights_out[i] = weights[i];
                positions_out[i] = positions[i];
            }
    } else {
        Threshold t{~0ull, 0};
        if (room > 0) t = select_threshold<kEvictThreads>(sh, n, room, [&](int i) -> uint64_t { return safe(i) ? 0 : order_key(weights[i]); });
        holes = evict_lists<kEvictThreads>(p, sh, weights, positions, weights_out, positions_out, kept_bits, to, since, n, k, room, t, safe);
    }
    __syncthreads();  // the lists, and every read of weights and positions that an aliased output may overwrite
    for (int j = threadIdx.x; j < holes; j += kEvictThreads) {
        weights_out[to[j]] = weights[since[j]];
        positions_out[to[j]] = positions[since[j]];
    }
    if (threadIdx.x == 0) to[-1] = holes;   // (slots behind the new length are cleared with the moves)
}

// The same with a cluster per row, for long rows: a CTA keeps the keys and positions of its stretch in shared memory.
constexpr int kWideThreads = 512, kWideFrom = 16384;

__global__ void __cluster_dims__(kWideCtas, 1, 1) __launch_bounds__(kWideThreads)
evict_select_wide_kernel(const __grid_constant__ EvictParams p) {
    __shared__ WideShared wide;
    __shared__ int newest_of[32];
    __shared__ int newest_here;
    auto cluster = cooperative_groups::this_cluster();
    const PagedView& kv = p.kv;
    const int b = blockIdx.y, kvh = blockIdx.x / kWideCtas, mine = cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    const int n = kv.length(b), k = min(n, p.budget);
    const size_t row = static_cast<size_t>(b) * kv.kv_heads + kvh;
    const float* weights = p.weights + row * p.stride;
    const int* positions = p.positions + row * p.stride;
    float* weights_out = p.weights_out + row * p.stride;
    int* positions_out = p.positions_out + row * p.stride;
    int* to = p.moves + row * (2 + 2 * static_cast<size_t>(p.max_moves)) + 2;
    int* since = to + p.max_moves;
    if (threadIdx.x == 0 && mine == 0) to[-2] = n;
    if (k == n) {
        if (threadIdx.x == 0 && mine == 0) to[-1] = 0;
        for (int i = mine * kWideThreads + threadIdx.x; i < n; i += kWideCtas * kWideThreads) {
            weights_out[i] = weights[i];
            positions_out[i] = positions[i];
        }
        return;
    }
    extern __shared__ __align__(16) uint32_t wide_keys[];
    uint32_t* keys = wide_keys;          // of the stretch: the weights' keys (kForced for safe rows), then the positions
    const int stretch = wide_stretch(n), base = min(n, mine * stretch), count = min(stretch, n - base);
    int* at = reinterpret_cast<int*>(keys + p.wide_items);
    int newest = -1;
#pragma unroll 4
    for (int i = threadIdx.x; i < count; i += kWideThreads) {   // (its own entries, here and below)
        at[i] = positions[base + i];
        keys[i] = static_cast<uint32_t>(order_key(weights[base + i]));
        newest = max(newest, at[i]);
    }
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) newest_of[warp] = newest;
    __syncthreads();
    if (warp == 0) {
        newest = __reduce_max_sync(0xffffffffu, lane < kWideThreads / 32 ? newest_of[lane] : -1);
        if (lane == 0) newest_here = newest;
    }
    cluster.sync();
    newest = __reduce_max_sync(0xffffffffu, *cluster.map_shared_rank(&newest_here, lane % kWideCtas));
    const int64_t recent_from = static_cast<int64_t>(newest) - p.recent;
    const int sink = p.sink;
    const auto is_safe = [&](int position) { return position < sink || position > recent_from; };
    int n_safe = 0;
    for (int i = threadIdx.x; i < count; i += kWideThreads)
        if (is_safe(at[i])) {
            keys[i] = kForced;
            ++n_safe;
        }
    n_safe = __reduce_add_sync(0xffffffffu, n_safe);
    __syncthreads();
    if (lane == 0) newest_of[warp] = n_safe;
    __syncthreads();
    n_safe = __reduce_add_sync(0xffffffffu, lane < kWideThreads / 32 ? newest_of[lane] : 0);
    const int room = k - static_cast<int>(offsets_before(cluster, wide, n_safe, 0).all_a);
    bool settled = false;
    if (room > 0) {
        settled = select_mask_wide<kWideThreads>(cluster, wide, keys, count, base, room,
                                                 [&](int j) -> uint64_t { return keys[wide.near[j] - base]; });
    } else if (room == 0) {
        for (int i0 = warp * 32; i0 < count; i0 += kWideThreads) {
            const unsigned word = __ballot_sync(0xffffffffu, i0 + lane < count && keys[i0 + lane] == kForced);
            if (lane == 0) wide.words[i0 >> 5] = word;
        }
        settled = true;
        __syncthreads();
    }
    if (!settled) {        // more safe positions than the budget holds (all CTAs of the cluster agree)
        cluster.sync();    // the others' shared memory is not read any more
        if (mine != 0) return;
        SelectShared& sh = *reinterpret_cast<SelectShared*>(wide_keys);   // (the keys are not needed any more)
        const auto safe = [&](int i) { return is_safe(positions[i]); };
        Threshold t{~0ull, 0};
        if (room > 0) t = select_threshold<kWideThreads>(sh, n, room, [&](int i) -> uint64_t { return safe(i) ? 0 : order_key(weights[i]); });
        const int holes = evict_lists<kWideThreads>(p, sh, weights, positions, weights_out, positions_out, p.kept + row * kv.limit, to, since, n, k, room, t, safe);
        __syncthreads();
        for (int j = threadIdx.x; j < holes; j += kWideThreads) {
            weights_out[to[j]] = weights[since[j]];
            positions_out[to[j]] = positions[since[j]];
        }
        if (threadIdx.x == 0) to[-1] = holes;
        return;
    }
    // freed slots before the new length and kept rows behind it
    const int words = (count + 31) / 32;
    const auto masks = [&](int w, unsigned& hole, unsigned& tail) {
        const int first = base + w * 32, left = count - w * 32;
        const unsigned live = left >= 32 ? ~0u : (1u << left) - 1;
        const unsigned front = (first + 32 <= k ? ~0u : (first >= k ? 0u : (1u << (k - first)) - 1)) & live;
        hole = ~wide.words[w] & front;
        tail = wide.words[w] & ~front & live;
    };
    unsigned n_hole = 0, n_tail = 0;
    for (int w = threadIdx.x; w < words; w += kWideThreads) {
        unsigned hole, tail;
        masks(w, hole, tail);
        n_hole += __popc(hole);
        n_tail += __popc(tail);
    }
    n_hole = __reduce_add_sync(0xffffffffu, n_hole);
    n_tail = __reduce_add_sync(0xffffffffu, n_tail);
    if (lane == 0) { wide.lo[warp] = n_hole; wide.hi[warp] = n_tail; }
    cluster.sync();        // (also: every CTA is done with the safe rows' counts)
    n_hole = __reduce_add_sync(0xffffffffu, lane < kWideThreads / 32 ? wide.lo[lane] : 0u);
    n_tail = __reduce_add_sync(0xffffffffu, lane < kWideThreads / 32 ? wide.hi[lane] : 0u);
    const WideOffsets before = offsets_before(cluster, wide, n_hole, n_tail);
    walk_bits<kWideThreads>(wide.scan, words, masks,
        [&](int i, int rank) { if (static_cast<int>(before.a) + rank < p.max_moves) to[before.a + rank] = base + i; },
        [&](int i, int rank) { if (static_cast<int>(before.b) + rank < p.max_moves) since[before.b + rank] = base + i; });
    for (int i = threadIdx.x; i < count; i += kWideThreads)
        if (base + i < k && (wide.words[i >> 5] >> (i & 31) & 1u)) {
            weights_out[base + i] = weights[base + i];
            positions_out[base + i] = at[i];
        }
    const int holes = min(min(static_cast<int>(before.all_a), static_cast<int>(before.all_b)), p.max_moves);
    if (threadIdx.x == 0 && mine == 0) to[-1] = holes;
    cluster.sync();        // the lists, and every read of weights and positions that an aliased output may overwrite
    for (int j = mine * kWideThreads + threadIdx.x; j < holes; j += kWideCtas * kWideThreads) {
        weights_out[to[j]] = weights[since[j]];
        positions_out[to[j]] = positions[since[j]];
    }
}

constexpr int kMoveRows = 4;

// A warp moves four rows at once (one after the other, each with its chain of list, table and row, moved 125 MB in 130 us); the entries behind the new length are cleared here, and new_len is written here, where
// nothing reads context_len (it may be the same array).
template <class V>
__global__ void __launch_bounds__(256)
evict_move_kernel(const __grid_constant__ EvictParams p, int k_units, int v_units) {
    const PagedView& kv = p.kv;
    const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    const int* to = p.moves + (static_cast<size_t>(b) * kv.kv_heads + kvh) * (2 + 2 * static_cast<size_t>(p.max_moves)) + 2;
    const int* since = to + p.max_moves;
    const int count = to[-1];
    V* keys = static_cast<V*>(const_cast<void*>(kv.k_pool));
    V* values = static_cast<V*>(const_cast<void*>(kv.v_pool));
    for (int j0 = (blockIdx.x * 8 + warp) * kMoveRows; j0 < count; j0 += gridDim.x * 8 * kMoveRows) {
        int64_t src = -1, dst = -1;
        if (lane < kMoveRows && j0 + lane < count) {
            src = kv.row(b, kvh, since[j0 + lane]);
            dst = kv.row(b, kvh, to[j0 + lane]);
            if (dst < 0) src = -1;
        }
        int64_t from[kMoveRows], into[kMoveRows];
#pragma unroll
        for (int r = 0; r < kMoveRows; ++r) {
            from[r] = __shfl_sync(0xffffffffu, src, r);
            into[r] = __shfl_sync(0xffffffffu, dst, r);
        }
        for (int i = lane; i < k_units + v_units; i += 32) {
            const bool key = i < k_units;
            V* pool = key ? keys : values;
            const int width = key ? k_units : v_units, at = key ? i : i - k_units;
            V unit[kMoveRows];
#pragma unroll
            for (int r = 0; r < kMoveRows; ++r)
                if (from[r] >= 0) unit[r] = pool[from[r] * width + at];
#pragma unroll
            for (int r = 0; r < kMoveRows; ++r)
                if (from[r] >= 0) pool[into[r] * width + at] = unit[r];
        }
    }
    const int n = to[-2], k = min(n, p.budget);
    const size_t row = (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.stride;
    for (int i = k + blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) {
        p.weights_out[row + i] = 0.0F;
        p.positions_out[row + i] = -1;
    }
    if (blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0) p.new_len[b] = k;
}

int evict_max_moves(const sfb_evict_args& a) {
    const int covered = a.max_blocks * a.block_tokens;
    const int limit = a.max_context < covered ? a.max_context : covered;
    const int beyond = limit - a.budget;
    return beyond <= 0 ? 0 : (beyond < a.budget ? beyond : a.budget);
}

size_t evict_moves_bytes(const sfb_evict_args& a) {
    return round_up16(sizeof(int) * static_cast<size_t>(a.batch) * a.kv_heads * (2 + 2 * static_cast<size_t>(evict_max_moves(a))));
}

sfb_status check_evict(const sfb_evict_args* a) {
    SFB_REQUIRE(a, "evict: null arguments");
    SFB_TRY(check_cache(a->k_pool, a->v_pool, a->block_table, a->batch, a->kv_heads, a->head_dim, a->head_dim_value,
                        a->block_tokens, a->max_blocks, a->num_blocks, a->dtype, "evict"));
    SFB_REQUIRE(a->max_context > 0 && a->weight_stride >= a->max_context, "evict: weight_stride shorter than max_context");
    SFB_REQUIRE(a->budget > 0 && a->sink_tokens >= 0 && a->recent_tokens >= 0 &&
                    static_cast<int64_t>(a->sink_tokens) + a->recent_tokens <= a->budget,
                "evict: the sink and recent tokens have to fit into the budget");
    return SFB_OK;
}

// ---- accepted path ---------------------------------------------------------------------------------------------------

struct AcceptParams {
    PagedView kv;
    const void *draft_k, *draft_v;
    const int *path, *path_len;
    int* new_len;
    int nodes, max_path;
};

// One warp per appended row.
template <class V>
__global__ void __launch_bounds__(256)
accept_kernel(const __grid_constant__ AcceptParams p, int k_units, int v_units) {
    const PagedView& kv = p.kv;
    const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    const int start = kv.lens[b];
    int count = p.path_len[b];
    if (count < 0 || count > p.max_path) {
        count = count < 0 ? 0 : p.max_path;
        if (threadIdx.x == 0) atomicOr(kv.status, kCodeDecodeBounds);
    }
    if (p.new_len && blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0) p.new_len[b] = start + count;
    const V* draft_k = static_cast<const V*>(p.draft_k) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.nodes * k_units;
    const V* draft_v = static_cast<const V*>(p.draft_v) + (static_cast<size_t>(b) * kv.kv_heads + kvh) * p.nodes * v_units;
    V* keys = static_cast<V*>(const_cast<void*>(kv.k_pool));
    V* values = static_cast<V*>(const_cast<void*>(kv.v_pool));
    for (int t = blockIdx.x * 8 + warp; t < count; t += gridDim.x * 8) {
        const int node = p.path[static_cast<size_t>(b) * p.max_path + t];
        const int64_t position = static_cast<int64_t>(start) + t;
        if (node < 0 || node >= p.nodes || position < 0 || position >= kv.limit) {
            atomicOr(kv.status, kCodeDecodeBounds);
            continue;
        }
        const int64_t dst = kv.row(b, kvh, static_cast<int>(position));
        if (dst < 0) continue;
        for (int i = lane; i < k_units; i += 32) keys[dst * k_units + i] = draft_k[static_cast<size_t>(node) * k_units + i];
        for (int i = lane; i < v_units; i += 32) values[dst * v_units + i] = draft_v[static_cast<size_t>(node) * v_units + i];
    }
}

// Rows are copied in units of 16 bytes where every row starts and ends on one, else in elements.
bool wide_rows(int dim, int dim_v, int dtype) {
    return dim * dtype_size(dtype) % 16 == 0 && dim_v * dtype_size(dtype) % 16 == 0;
}

}  // namespace
}  // namespace sfb

using namespace sfb;

extern "C" {

size_t sfb_attention_weights_workspace(const sfb_weights_args* a) {
    if (check_weights(a) != SFB_OK) return 0;
    return std::max(weights_layout(*a, true).total, weights_layout(*a, false).total);   // (the addresses may not be set yet)
}

sfb_status sfb_k_attention_decode_weights(const sfb_weights_args* a, sfb_stream stream) {
    SFB_TRY(check_weights(a));
    SFB_REQUIRE(a->q && a->context_len && a->out && a->weights_out && a->workspace, "decode weights: null tensor");
    SFB_REQUIRE(!a->positions || a->query_position, "decode weights: positions without query_position");
    SFB_REQUIRE(aligned16(a->workspace), "decode weights: the workspace has to be 16-byte aligned");
    const WeightsLayout l = weights_layout(*a, aligned16(a->k_pool) && aligned16(a->v_pool) && aligned16(a->q));
    cudaStream_t s = as_stream(stream);
    StepParams p{};
    p.kv = make_view(a->k_pool, a->v_pool, a->block_table, a->context_len, a->kv_heads, a->head_dim, a->head_dim_value,
                     a->block_tokens, a->max_blocks, a->num_blocks, a->max_context);
    p.q = a->q; p.out = a->out;
    p.part = step_partials(l.step, a->batch, a->q_heads, a->head_dim_value, a->workspace);
    p.logits = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + l.partials);
    p.logit_stride = l.logit_stride;
    p.batch = a->batch; p.q_heads = a->q_heads; p.chunk_blocks = l.step.chunk_blocks;
    p.scale_log2 = (a->scale > 0.0F ? a->scale : 1.0F / sqrtf(static_cast<float>(a->head_dim))) * 1.4426950408889634F;
    SFB_TRY(step_attention(p, l.step, a->dtype, s));
    const AddParams add{p.kv, p.part, p.logits, a->weights, a->weights_out, a->out, a->positions, a->query_position,
                        l.logit_stride, a->q_heads, a->weight_stride,
                        a->weight_stride % 4 == 0 && aligned16(a->weights) && aligned16(a->weights_out)};
    const int group = a->q_heads / a->kv_heads;
    // one position a thread as long as that leaves at most eight CTAs per SM, else four, and up to four times four one after the
    // other while four CTAs per SM remain (64 ragged sequences to 8192 tokens: 234 -> 230 us, attention included)
    const int64_t pairs = static_cast<int64_t>(a->kv_heads) * a->batch;
    int chunk = kAddThreads;
    if (pairs * ceil_div(p.kv.limit, chunk) > 8LL * sm_count()) {
        const int64_t times = pairs * ceil_div(p.kv.limit, 4 * kAddThreads) / (4LL * sm_count());
        chunk = 4 * kAddThreads * static_cast<int>(times < 1 ? 1 : times > 4 ? 4 : times);
    }
    const dim3 grid(group + ceil_div(p.kv.limit, chunk), a->kv_heads, a->batch);
    if (a->dtype == SFB_F32) SFB_CUDA(launch_dependent(add_weights_kernel<float>, grid, dim3(kAddThreads), 0, s, add, chunk));
    else SFB_CUDA(launch_dependent(add_weights_kernel<bf16>, grid, dim3(kAddThreads), 0, s, add, chunk));
    return check_launch("decode_weights_add");
}

size_t sfb_paged_kv_evict_workspace(const sfb_evict_args* a) {
    if (check_evict(a) != SFB_OK) return 0;
    return evict_moves_bytes(*a) + static_cast<size_t>(a->batch) * a->kv_heads * (a->max_context < a->max_blocks * a->block_tokens ? a->max_context : a->max_blocks * a->block_tokens);
}

sfb_status sfb_k_paged_kv_evict(const sfb_evict_args* a, sfb_stream stream) {
    SFB_TRY(check_evict(a));
    SFB_REQUIRE(a->context_len && a->weights && a->weights_out && a->positions && a->positions_out && a->new_len && a->workspace,
                "evict: null tensor");
    SFB_REQUIRE(aligned16(a->workspace), "evict: the workspace has to be 16-byte aligned");
    cudaStream_t s = as_stream(stream);
    EvictParams p{};
    p.kv = make_view(a->k_pool, a->v_pool, a->block_table, a->context_len, a->kv_heads, a->head_dim, a->head_dim_value,
                     a->block_tokens, a->max_blocks, a->num_blocks, a->max_context);
    p.weights = a->weights; p.weights_out = a->weights_out; p.positions = a->positions; p.positions_out = a->positions_out;
    p.new_len = a->new_len; p.moves = static_cast<int*>(a->workspace); p.max_moves = evict_max_moves(*a);
    p.kept = static_cast<uint8_t*>(a->workspace) + evict_moves_bytes(*a);
    p.stride = a->weight_stride; p.budget = a->budget; p.sink = a->sink_tokens; p.recent = a->recent_tokens;
    p.masked = p.kv.limit <= kMaskItems;
    // Long rows are shared by a cluster each: rows that one CTA's mask does not hold (65536 slots, 8 rows: 165 us by the walks
    // over 64-bit keys, 30 by a cluster; 131072: 332 and 40), and, while two CTAs an SM hold them all, rows of more than 16384
    // (32768 slots: 30 us by one CTA, 26 by a cluster; 24500: 28.5 and 24.9; 16384: 24.0 and 23.4; 6000: 17 and 21).
    const int64_t rows = static_cast<int64_t>(a->batch) * a->kv_heads;
    const bool wide_select = p.kv.limit <= kWideCtas * kWideItems &&
                             (!p.masked || (p.kv.limit > kWideFrom && rows * kWideCtas <= 2LL * sm_count()));
    const size_t key_bytes = p.masked ? sizeof(uint32_t) * static_cast<size_t>(p.kv.limit) : 0;
    SFB_CUDA(cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(uint32_t) * kMaskItems)));
    if (wide_select) {
        p.wide_items = wide_stretch(p.kv.limit);
        SFB_CUDA(cudaFuncSetAttribute(evict_select_wide_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * static_cast<int>(sizeof(uint32_t)) * kWideItems));
        SFB_CUDA(launch_dependent(evict_select_wide_kernel, dim3(a->kv_heads * kWideCtas, a->batch), dim3(kWideThreads),
                                  std::max(2 * sizeof(uint32_t) * static_cast<size_t>(p.wide_items), sizeof(SelectShared)), s, p));
    } else {
        SFB_CUDA(launch_dependent(evict_select_kernel, dim3(a->kv_heads, a->batch), dim3(kEvictThreads), key_bytes, s, p));
    }
    SFB_TRY(check_launch("evict_select"));
    // eight warps of four rows a CTA, about two rounds of eight CTAs an SM at most
    const int most = static_cast<int>(16LL * sm_count() / rows > 0 ? 16LL * sm_count() / rows : 1);
    const int wanted = ceil_div(p.max_moves, 8 * kMoveRows);
    const dim3 grid(wanted < 1 ? 1 : wanted < most ? wanted : most, a->kv_heads, a->batch);
    const bool wide = wide_rows(a->head_dim, a->head_dim_value, a->dtype) && aligned16(a->k_pool) && aligned16(a->v_pool);
    const int per = wide ? 16 / static_cast<int>(dtype_size(a->dtype)) : 1;
    const int ku = a->head_dim / per, vu = a->head_dim_value / per;
    if (wide) SFB_CUDA(launch_dependent(evict_move_kernel<uint4>, grid, dim3(256), 0, s, p, ku, vu));
    else if (a->dtype == SFB_F32) SFB_CUDA(launch_dependent(evict_move_kernel<uint32_t>, grid, dim3(256), 0, s, p, ku, vu));
    else SFB_CUDA(launch_dependent(evict_move_kernel<uint16_t>, grid, dim3(256), 0, s, p, ku, vu));
    return check_launch("evict_move");
}

sfb_status sfb_k_paged_kv_accept(const sfb_accept_args* a, sfb_stream stream) {
    SFB_REQUIRE(a && a->draft_k && a->draft_v && a->start_len && a->path && a->path_len, "accept: null tensor");
    SFB_TRY(check_cache(a->k_pool, a->v_pool, a->block_table, a->batch, a->kv_heads, a->head_dim, a->head_dim_value,
                        a->block_tokens, a->max_blocks, a->num_blocks, a->dtype, "accept"));
    SFB_REQUIRE(a->nodes > 0 && a->max_path > 0, "accept: no nodes or no path");
    SFB_REQUIRE(a->new_len != a->start_len, "accept: new_len must not be start_len");
    cudaStream_t s = as_stream(stream);
    AcceptParams p{};
    p.kv = make_view(a->k_pool, a->v_pool, a->block_table, a->start_len, a->kv_heads, a->head_dim, a->head_dim_value,
                     a->block_tokens, a->max_blocks, a->num_blocks, a->max_blocks * a->block_tokens);
    p.draft_k = a->draft_k; p.draft_v = a->draft_v; p.path = a->path; p.path_len = a->path_len; p.new_len = a->new_len;
    p.nodes = a->nodes; p.max_path = a->max_path;
    const dim3 grid(ceil_div(a->max_path, 8), a->kv_heads, a->batch);
    const bool wide = wide_rows(a->head_dim, a->head_dim_value, a->dtype) && aligned16(a->k_pool) && aligned16(a->v_pool) &&
                      aligned16(a->draft_k) && aligned16(a->draft_v);
    const int per = wide ? 16 / static_cast<int>(dtype_size(a->dtype)) : 1;
    const int ku = a->head_dim / per, vu = a->head_dim_value / per;
    if (wide) SFB_CUDA(launch_dependent(accept_kernel<uint4>, grid, dim3(256), 0, s, p, ku, vu));
    else if (a->dtype == SFB_F32) SFB_CUDA(launch_dependent(accept_kernel<uint32_t>, grid, dim3(256), 0, s, p, ku, vu));
    else SFB_CUDA(launch_dependent(accept_kernel<uint16_t>, grid, dim3(256), 0, s, p, ku, vu));
    return check_launch("paged_kv_accept");
}

}  // extern "C"
