// Selection of the k largest of n keys by one CTA, ties to the lower index.
//
// Keys are unsigned 64-bit words whose order is the order wanted; a key of 0 does not take part.  The k-th largest key is found by narrowing a
// range: the keys inside it are counted in 2048 equal bins, the bin that holds the k-th becomes the next range.  A
// range of 64 bits needs at most six passes; scores that differ in their leading bits need one or two, because a range
// whose keys are all wanted, or that has shrunk to one value, ends the search.
#pragma once

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

struct SelectShared {
    unsigned hist[kSelectBins];
    uint64_t lo[32], hi[32];
    unsigned scan[33];
    unsigned long long walk[32];
    uint64_t low, high;
    int rest, done;
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
