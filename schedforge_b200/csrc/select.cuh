// Selection of the k largest of n keys by one CTA, ties to the lower index.
//
// Rows of up to kMaskItems keys of 32 bits (select_mask): the keys are counted in 2048 equal bins of their range, what
// lies above the bin of the k-th is kept, and the few keys inside it are ranked against one another; the result is one
// bit per key in shared memory.  A bin with too many keys is cut into bins again, until it holds few or equal ones.  Keys known to
// a tolerance of which too many are left, and longer rows, take keys of 64 bits that are narrowed bin by bin until
// the range holds one value (select_threshold: at most six passes).
// The order of the unsigned keys is the order wanted; a key of 0 does not take part.
#pragma once

#ifdef __CUDACC__
#include <cooperative_groups.h>
#endif

#include "common.cuh"

namespace sfb {

#ifdef __CUDACC__
constexpr int kSelectBins = 2048;

// Order-preserving integer images.  NaN gets 1, which ranks below every number; -0 counts as +0.
__device__ __forceinline__ uint64_t order_key(double v) {
    if (v != v) return 1;
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ uint64_t order_key(float v) {
    if (v != v) return 1;
    const uint32_t u = __float_as_uint(v + 0.0F);
    return (u >> 31) ? static_cast<uint32_t>(~u) : (u | 0x80000000u);
}

constexpr int kMaskItems = 40960;   // one bit each in shared memory
constexpr int kMaskWords = kMaskItems / 32;
constexpr int kNearItems = 512;     // keys ranked against one another

struct SelectShared {
    unsigned hist[kSelectBins];
    uint64_t lo[32], hi[32];
    unsigned scan[33];
    unsigned long long walk[32];
    uint64_t low, high;
    int rest, done;
    unsigned words[kMaskWords], ties[kMaskWords];
    int near[kNearItems];
    uint64_t near_key[kNearItems];
    int near_count, kept_count;
};

// What is kept: keys above `low`, and, where cut != 0, the first `cut` keys equal to it (in index order); where cut
// is 0, every key >= low.
struct Threshold {
    uint64_t low;
    int cut;
};

// All threads of the CTA call it; 1 <= k <= number of keys that are not 0.  key(i) is evaluated several times.
template <int THREADS, class Key>
__device__ Threshold select_threshold(SelectShared& sh, int n, int k, Key key) {
    constexpr int kWarps = THREADS / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t lo = ~0ull, hi = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const uint64_t v = key(i);
        lo = v != 0 && v < lo ? v : lo;
        hi = v > hi ? v : hi;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t a = __shfl_xor_sync(0xffffffffu, lo, o), b = __shfl_xor_sync(0xffffffffu, hi, o);
        lo = a < lo ? a : lo;
        hi = b > hi ? b : hi;
    }
    if (lane == 0) { sh.lo[warp] = lo; sh.hi[warp] = hi; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWarps; ++w) {
            lo = sh.lo[w] < lo ? sh.lo[w] : lo;
            hi = sh.hi[w] > hi ? sh.hi[w] : hi;
        }
        sh.low = lo; sh.high = hi; sh.rest = k; sh.done = 0;
    }
    // (six passes narrow any 64-bit range to one value; the bound only matters if keys change under the search)
    for (int pass = 0; pass < 8; ++pass) {
        for (int i = threadIdx.x; i < kSelectBins; i += THREADS) sh.hist[i] = 0;
        __syncthreads();
        const uint64_t low = sh.low, high = sh.high;
        const int bits = 64 - __clzll(static_cast<long long>(high - low));
        const int shift = bits > 11 ? bits - 11 : 0;
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const uint64_t v = key(i);
            if (v >= low && v <= high) atomicAdd(&sh.hist[static_cast<int>((v - low) >> shift)], 1u);
        }
        __syncthreads();
        // counts from the top: thread t owns bins [t * per, (t + 1) * per) counted downwards from the last bin
        constexpr int per = kSelectBins / THREADS > 0 ? kSelectBins / THREADS : 1;
        unsigned own = 0;
        if (static_cast<int>(threadIdx.x) * per < kSelectBins)
#pragma unroll
            for (int j = 0; j < per; ++j) own += sh.hist[kSelectBins - 1 - (threadIdx.x * per + j)];
        unsigned sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) sh.scan[warp] = sum;
        const int rest = sh.rest;
        __syncthreads();
        unsigned before = sum - own;
        for (int w = 0; w < warp; ++w) before += sh.scan[w];
        if (before < static_cast<unsigned>(rest) && before + own >= static_cast<unsigned>(rest)) {  // exactly one thread
            unsigned above = before;
            int bin = kSelectBins - 1 - threadIdx.x * per;
            while (above + sh.hist[bin] < static_cast<unsigned>(rest)) above += sh.hist[bin--];
            const uint64_t first = low + (static_cast<uint64_t>(bin) << shift);
            const uint64_t span = (1ull << shift) - 1;
            sh.rest = rest - static_cast<int>(above);
            sh.low = first;
            sh.high = high - first < span ? high : first + span;
            sh.done = shift == 0 || sh.hist[bin] == static_cast<unsigned>(sh.rest);
            if (sh.hist[bin] == static_cast<unsigned>(sh.rest)) sh.rest = 0;  // the whole bin is wanted
        }
        __syncthreads();
        if (sh.done) break;
    }
    const Threshold found{sh.low, sh.rest};
    __syncthreads();
    return found;
}

// words |= the first `room` set bits of ties, counting on from `before`.
template <int THREADS>
__device__ __forceinline__ void take_first(unsigned* scan, const unsigned* ties, unsigned* words, int count, int room, int before) {
    constexpr int kWarps = THREADS / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int w0 = 0; w0 < count; w0 += THREADS) {
        const int w = w0 + threadIdx.x;
        const unsigned bits = w < count ? ties[w] : 0u;
        const int own = __popc(bits);
        int incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) scan[warp] = incl;
        __syncthreads();
        const unsigned mine = lane < kWarps ? scan[lane] : 0u;
        const int take = room - (before + static_cast<int>(__reduce_add_sync(0xffffffffu, lane < warp ? mine : 0u)) + incl - own);
        before += static_cast<int>(__reduce_add_sync(0xffffffffu, mine));
        if (take > 0 && own > 0) {
            unsigned rest = bits;
            for (int i = 0; i < take && rest; ++i) rest &= rest - 1;
            words[w] |= bits & ~rest;
        }
        __syncthreads();
    }
}

constexpr uint32_t kForced = 0xffffffffu;   // a 32-bit key that is kept whatever the others are (no number's image)

// Bits of the kept keys in sh.words: the forced ones and the k largest of the others (n <= kMaskItems; 1 <= k <= number of
// other keys that are not 0).  keys: shared memory, complete after the callers' last barrier.  widen(low, high) may
// extend the range of keys that are ranked, and rank(j) gives the final key of near item j (index sh.near[j]; called by
// whole warps, all lanes of which return it): how keys known to a tolerance are ranked exactly where it matters.  EXACT: keys
// are final, so that a range of one value is settled by index (one with more than kNearItems keys always is).  Otherwise
// that many are not settled, and it returns false.  All threads call it.
template <int THREADS, bool EXACT, class Widen, class Rank>
__device__ bool select_mask(SelectShared& sh, const uint32_t* keys, int n, int k, Widen widen, Rank rank) {
    constexpr int kWarps = THREADS / 32, kPer = kSelectBins / THREADS;
    static_assert(kPer >= 1 && kWarps <= 32, "one or more bins a thread");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t low = ~0u, high = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const uint32_t v = keys[i];
        if (v != 0 && v != kForced) {
            low = min(low, v);
            high = max(high, v);
        }
    }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if (lane == 0) { sh.lo[warp] = low; sh.hi[warp] = high; }
#pragma unroll
    for (int j = 0; j < kPer; ++j) sh.hist[threadIdx.x * kPer + j] = 0;
    if (threadIdx.x == 0) sh.near_count = sh.kept_count = 0;
    __syncthreads();
    low = __reduce_min_sync(0xffffffffu, lane < kWarps ? static_cast<uint32_t>(sh.lo[lane]) : ~0u);
    high = __reduce_max_sync(0xffffffffu, lane < kWarps ? static_cast<uint32_t>(sh.hi[lane]) : 0u);
    int rest = k;
    for (int pass = 0; pass < 4; ++pass) {
        const int bits = 32 - __clz(high - low), shift = bits > 11 ? bits - 11 : 0;
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const uint32_t v = keys[i];
            if (v >= low && v <= high && v != kForced) atomicAdd(&sh.hist[(v - low) >> shift], 1u);
        }
        __syncthreads();
        // counts from the top: thread t owns kPer bins counted downwards from the last
        unsigned count[kPer], own = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) own += count[j] = sh.hist[kSelectBins - 1 - (threadIdx.x * kPer + j)];
        unsigned sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) sh.scan[warp] = sum;
        __syncthreads();
        unsigned above = __reduce_add_sync(0xffffffffu, lane < warp ? sh.scan[lane] : 0u) + sum - own;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (above < static_cast<unsigned>(rest) && above + count[j] >= static_cast<unsigned>(rest)) {   // one thread, one bin
                const uint32_t first = low + (static_cast<uint32_t>(kSelectBins - 1 - (threadIdx.x * kPer + j)) << shift);
                const uint32_t span = (1u << shift) - 1;
                sh.low = first;
                sh.high = high - first < span ? high : first + span;
                sh.rest = rest - static_cast<int>(above);
                sh.done = shift == 0 || count[j] <= kNearItems / 8;
            }
            above += count[j];
            sh.hist[kSelectBins - 1 - (threadIdx.x * kPer + j)] = 0;
        }
        __syncthreads();
        low = static_cast<uint32_t>(sh.low);
        high = static_cast<uint32_t>(sh.high);
        rest = sh.rest;
        if (sh.done) break;
        __syncthreads();
    }
    widen(low, high);
    int kept = 0;
    for (int i0 = warp * 32; i0 < n; i0 += THREADS) {
        const int i = i0 + lane;
        const uint32_t v = i < n ? keys[i] : 0;
        const unsigned word = __ballot_sync(0xffffffffu, v > high);
        kept += __popc(word & __ballot_sync(0xffffffffu, v != kForced));
        const bool is_near = v != 0 && v >= low && v <= high && v != kForced;
        const unsigned ties = __ballot_sync(0xffffffffu, is_near);
        if (lane == 0) {
            sh.words[i0 >> 5] = word;
            sh.ties[i0 >> 5] = ties;
        }
        if (is_near) {
            const int at = atomicAdd(&sh.near_count, 1);
            if (at < kNearItems) sh.near[at] = i;
        }
    }
    if (lane == 0 && kept) atomicAdd(&sh.kept_count, kept);
    __syncthreads();
    const int near = sh.near_count, room = k - sh.kept_count;
    if (EXACT && low == high) {
        take_first<THREADS>(sh.scan, sh.ties, sh.words, (n + 31) / 32, room, 0);
        return true;
    }
    if (near > kNearItems) return false;
    if (room >= near) {
        for (int j = threadIdx.x; j < near; j += THREADS) atomicOr(&sh.words[sh.near[j] >> 5], 1u << (sh.near[j] & 31));
    } else {
        for (int j = warp; j < near; j += kWarps) {
            const uint64_t v = rank(j);
            if (lane == 0) sh.near_key[j] = v;
        }
        __syncthreads();
        for (int j = threadIdx.x; j < near; j += THREADS) {
            const uint64_t v = sh.near_key[j];
            const int i = sh.near[j];
            int before = 0;
            for (int o = 0; o < near; ++o) {
                const uint64_t w = sh.near_key[o];
                before += w > v || (w == v && sh.near[o] < i);
            }
            if (before < room) atomicOr(&sh.words[i >> 5], 1u << (i & 31));
        }
    }
    __syncthreads();
    return true;
}

// ---- one row by a cluster ----------------------------------------------------------------------------------------
// select_mask for a row that the kWideCtas CTAs of a cluster share, each with a stretch of its entries: the counts of
// the bins, the range, the near keys and the totals are read out of the others' shared memory.  Rows of up to kWideCtas *
// kWideItems entries; the barriers of the cluster cost about 10 us in all, so it takes over where one CTA's walks cost more.
constexpr int kWideCtas = 8;
constexpr int kWideItems = 20480;     // longest stretch of a CTA

struct alignas(16) WideShared {
    unsigned hist[kSelectBins];
    unsigned scan[33];
    uint32_t lo[32], hi[32];
    uint32_t range[2];            // of this CTA's keys
    uint32_t low, high;
    int rest, done;
    int near_count, kept_count;   // of this CTA
    unsigned counts[2];           // for offsets_before
    int near[kNearItems], all[kNearItems];
    uint64_t near_key[kNearItems], all_key[kNearItems];
    unsigned words[kWideItems / 32], ties[kWideItems / 32];
};

// Stretch of CTA `rank`: a multiple of 32 entries, all but the last of the same length.
__host__ __device__ inline int wide_stretch(int n) { return ((n + kWideCtas - 1) / kWideCtas + 31) & ~31; }

// keys: this CTA's n entries, final, which are numbers base, base + 1, ... of the row.  Otherwise as select_mask; k counts over the
// whole row and is the same in all CTAs, and so is what is returned.
template <int THREADS, class Rank>
__device__ bool select_mask_wide(cooperative_groups::cluster_group& cluster, WideShared& sh, const uint32_t* keys, int n, int base, int k,
                                 Rank rank) {
    constexpr int kWarps = THREADS / 32, kPer = kSelectBins / THREADS;
    static_assert(kPer == 4, "four bins a thread: one 16-byte read of each CTA");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = cluster.block_rank();
    uint32_t low = ~0u, high = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const uint32_t v = keys[i];
        if (v != 0 && v != kForced) {
            low = min(low, v);
            high = max(high, v);
        }
    }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if (lane == 0) { sh.lo[warp] = low; sh.hi[warp] = high; }
    uint4* bins = reinterpret_cast<uint4*>(sh.hist);
    bins[threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
    if (threadIdx.x == 0) sh.near_count = sh.kept_count = 0;
    __syncthreads();
    if (warp == 0) {
        low = __reduce_min_sync(0xffffffffu, lane < kWarps ? sh.lo[lane] : ~0u);
        high = __reduce_max_sync(0xffffffffu, lane < kWarps ? sh.hi[lane] : 0u);
        if (lane == 0) { sh.range[0] = low; sh.range[1] = high; }
    }
    cluster.sync();
    {
        const uint32_t* other = cluster.map_shared_rank(sh.range, lane % kWideCtas);
        low = __reduce_min_sync(0xffffffffu, other[0]);
        high = __reduce_max_sync(0xffffffffu, other[1]);
    }
    int rest = k;
    for (int pass = 0; pass < 4; ++pass) {
        const int bits = 32 - __clz(high - low), shift = bits > 11 ? bits - 11 : 0;
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const uint32_t v = keys[i];
            if (v >= low && v <= high && v != kForced) atomicAdd(&sh.hist[(v - low) >> shift], 1u);
        }
        cluster.sync();
        // counts from the top: thread t owns four bins counted downwards from the last
        uint4 sum4 = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int c = 0; c < kWideCtas; ++c) {
            const uint4 v = cluster.map_shared_rank(bins, c)[THREADS - 1 - threadIdx.x];
            sum4.x += v.x; sum4.y += v.y; sum4.z += v.z; sum4.w += v.w;
        }
        const unsigned count[4] = {sum4.w, sum4.z, sum4.y, sum4.x};
        const unsigned own = count[0] + count[1] + count[2] + count[3];
        unsigned sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) sh.scan[warp] = sum;
        __syncthreads();
        unsigned above = __reduce_add_sync(0xffffffffu, lane < warp ? sh.scan[lane] : 0u) + sum - own;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (above < static_cast<unsigned>(rest) && above + count[j] >= static_cast<unsigned>(rest)) {   // one thread, one bin
                const uint32_t first = low + (static_cast<uint32_t>(kSelectBins - 1 - (threadIdx.x * kPer + j)) << shift);
                const uint32_t span = (1u << shift) - 1;
                sh.low = first;
                sh.high = high - first < span ? high : first + span;
                sh.rest = rest - static_cast<int>(above);
                sh.done = shift == 0 || count[j] <= kNearItems / 8;
            }
            above += count[j];
        }
        __syncthreads();
        low = sh.low;
        high = sh.high;
        rest = sh.rest;
        if (sh.done) break;     // (the same in all CTAs: they add up the same counts)
        cluster.sync();         // every CTA has read the bins
        bins[threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
    }
    int kept = 0;
    for (int i0 = warp * 32; i0 < n; i0 += THREADS) {
        const int i = i0 + lane;
        const uint32_t v = i < n ? keys[i] : 0;
        const unsigned word = __ballot_sync(0xffffffffu, v > high);
        kept += __popc(word & __ballot_sync(0xffffffffu, v != kForced));
        const bool is_near = v != 0 && v >= low && v <= high && v != kForced;
        const unsigned ties = __ballot_sync(0xffffffffu, is_near);
        if (lane == 0) {
            sh.words[i0 >> 5] = word;
            sh.ties[i0 >> 5] = ties;
        }
        if (is_near) {
            const int at = atomicAdd(&sh.near_count, 1);
            if (at < kNearItems) sh.near[at] = base + i;
        }
    }
    if (lane == 0 && kept) atomicAdd(&sh.kept_count, kept);
    cluster.sync();
    int all = 0, before = 0, room = k;     // near keys of the row, of the CTAs before this one
#pragma unroll
    for (int c = 0; c < kWideCtas; ++c) {
        const int near = *cluster.map_shared_rank(&sh.near_count, c);
        if (c < mine) before += near;
        all += near;
        room -= *cluster.map_shared_rank(&sh.kept_count, c);
    }
    const int near = sh.near_count;
    if (low == high) {
        take_first<THREADS>(sh.scan, sh.ties, sh.words, (n + 31) / 32, room, before);
        return true;
    }
    if (all > kNearItems) return false;
    if (room >= all) {
        for (int j = threadIdx.x; j < near; j += THREADS) atomicOr(&sh.words[(sh.near[j] - base) >> 5], 1u << ((sh.near[j] - base) & 31));
    } else {
        for (int j = warp; j < near; j += kWarps) {
            const uint64_t v = rank(j);
            if (lane < kWideCtas) {    // into every CTA's list
                cluster.map_shared_rank(sh.all, lane)[before + j] = sh.near[j];
                cluster.map_shared_rank(sh.all_key, lane)[before + j] = v;
            }
            if (lane == 0) sh.near_key[j] = v;
        }
        cluster.sync();
        for (int j = threadIdx.x; j < near; j += THREADS) {
            const uint64_t v = sh.near_key[j];
            const int i = sh.near[j];
            int ahead = 0;
            for (int o = 0; o < all; ++o) {
                const uint64_t w = sh.all_key[o];
                ahead += w > v || (w == v && sh.all[o] < i);
            }
            if (ahead < room) atomicOr(&sh.words[(i - base) >> 5], 1u << ((i - base) & 31));
        }
    }
    __syncthreads();
    return true;
}

// Sums of a and b (this CTA's counts, the same in all its threads) over the CTAs before this one, and over all.
struct WideOffsets {
    unsigned a, b, all_a, all_b;
};
__device__ __forceinline__ WideOffsets offsets_before(cooperative_groups::cluster_group& cluster, WideShared& sh, unsigned a, unsigned b) {
    if (threadIdx.x == 0) { sh.counts[0] = a; sh.counts[1] = b; }
    cluster.sync();
    WideOffsets o{0u, 0u, 0u, 0u};
    const unsigned mine = cluster.block_rank();
#pragma unroll
    for (unsigned c = 0; c < kWideCtas; ++c) {
        const unsigned* other = cluster.map_shared_rank(sh.counts, c);
        const unsigned x = other[0], y = other[1];
        if (c < mine) { o.a += x; o.b += y; }
        o.all_a += x;
        o.all_b += y;
    }
    return o;
}

// Walks the set bits of two masks of `words` words in ascending order: visit_a(index, rank), visit_b(index, rank).
// Returns the totals (a in the low, b in the high half; each below 2^16).
template <int THREADS, class Words, class VisitA, class VisitB>
__device__ __forceinline__ unsigned walk_bits(unsigned* scan, int words, Words get, VisitA visit_a, VisitB visit_b) {
    constexpr int kWarps = THREADS / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned before = 0;
    for (int w0 = 0; w0 < words; w0 += THREADS) {
        const int w = w0 + threadIdx.x;
        unsigned a = 0, b = 0;
        if (w < words) get(w, a, b);
        const unsigned own = static_cast<unsigned>(__popc(a)) | static_cast<unsigned>(__popc(b)) << 16;
        unsigned incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) scan[warp] = incl;
        __syncthreads();
        const unsigned mine = lane < kWarps ? scan[lane] : 0u;
        const unsigned at = before + __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0u) + incl - own;
        before += __reduce_add_sync(0xffffffffu, mine);
        int ra = static_cast<int>(at & 0xffffu), rb = static_cast<int>(at >> 16);
        for (; a; a &= a - 1) visit_a(w * 32 + __ffs(a) - 1, ra++);
        for (; b; b &= b - 1) visit_b(w * 32 + __ffs(b) - 1, rb++);
        __syncthreads();
    }
    return before;
}

// Walks [0, n) in index order with the flags a(i) and b(i), each warp a contiguous stretch: visit(i, a, b, ra, rb) is
// called for every i < n with the number of a and b flags before it.  flags(i) returns a | b << 1 and is evaluated
// twice.  Returns the totals (a in the low, b in the high half); all threads of the CTA call it.
template <int THREADS, class Flags, class Visit>
__device__ __forceinline__ uint64_t walk_ranks(unsigned long long* scan, int n, Flags flags, Visit visit) {
    constexpr int kWarps = THREADS / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int stretch = ((n + kWarps - 1) / kWarps + 31) & ~31;
    const int begin = min(n, warp * stretch), end = min(n, begin + stretch);
    unsigned ca = 0, cb = 0;
    for (int i0 = begin; i0 < end; i0 += 32) {
        const int f = i0 + lane < end ? flags(i0 + lane) : 0;
        ca += __popc(__ballot_sync(0xffffffffu, f & 1));
        cb += __popc(__ballot_sync(0xffffffffu, f & 2));
    }
    if (lane == 0) scan[warp] = static_cast<uint64_t>(cb) << 32 | ca;
    __syncthreads();
    uint64_t before = 0, total = 0;
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) {
        const uint64_t v = scan[w];
        if (w < warp) before += v;
        total += v;
    }
    __syncthreads();
    unsigned ra = static_cast<unsigned>(before), rb = static_cast<unsigned>(before >> 32);
    const unsigned below = (1u << lane) - 1;
    for (int i0 = begin; i0 < end; i0 += 32) {
        const int i = i0 + lane;
        const int f = i < end ? flags(i) : 0;
        const unsigned ma = __ballot_sync(0xffffffffu, f & 1), mb = __ballot_sync(0xffffffffu, f & 2);
        if (i < end) visit(i, (f & 1) != 0, (f & 2) != 0, static_cast<int>(ra + __popc(ma & below)), static_cast<int>(rb + __popc(mb & below)));
        ra += __popc(ma);
        rb += __popc(mb);
    }
    return total;
}
#endif

}  // namespace sfb
