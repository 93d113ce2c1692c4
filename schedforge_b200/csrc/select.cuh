// Selection of the k largest of n keys by one CTA, ties to the lower index.
//
// Keys are unsigned 64-bit words whose order is the order wanted.  The k-th largest key is found by narrowing a
// range: the keys inside it are counted in 2048 equal bins, the bin that holds the k-th becomes the next range.  A
// range of 64 bits needs at most six passes; scores that differ in their leading bits need one or two, because a range
// whose keys are all wanted, or that has shrunk to one value, ends the search.
#pragma once

#include "common.cuh"

namespace sfb {

#ifdef __CUDACC__
constexpr int kSelectBins = 2048;

// Order-preserving integer images.  NaN gets 0, which ranks below everything; -0 counts as +0.
__device__ __forceinline__ uint64_t order_key(double v) {
    if (v != v) return 0;
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ uint64_t order_key(float v) {
    if (v != v) return 0;
    const uint32_t u = __float_as_uint(v + 0.0F);
    return (u >> 31) ? static_cast<uint32_t>(~u) : (u | 0x80000000u);
}

struct SelectShared {
    unsigned hist[kSelectBins];
    uint64_t lo[32], hi[32];
    unsigned scan[33];
    uint64_t low, high;
    int rest, done;
};

// What is kept: keys above `low`, and, where cut != 0, the first `cut` keys equal to it (in index order); where cut
// is 0, every key >= low.
struct Threshold {
    uint64_t low;
    int cut;
};

// All threads of the CTA call it; 1 <= k <= n.  key(i) is evaluated several times.
template <int THREADS, class Key>
__device__ Threshold select_threshold(SelectShared& sh, int n, int k, Key key) {
    constexpr int kWarps = THREADS / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t lo = ~0ull, hi = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const uint64_t v = key(i);
        lo = v < lo ? v : lo;
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
    if (k == n) {
        __syncthreads();
        return {sh.low, 0};
    }
    for (;;) {
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
            const uint64_t last = first + ((1ull << shift) - 1);
            sh.rest = rest - static_cast<int>(above);
            sh.low = first;
            sh.high = last < high ? last : high;
            sh.done = shift == 0 || sh.hist[bin] == static_cast<unsigned>(sh.rest);
            if (sh.hist[bin] == static_cast<unsigned>(sh.rest)) sh.rest = 0;  // the whole bin is wanted
        }
        __syncthreads();
        if (sh.done) return {sh.low, sh.rest};
    }
}

// Exclusive prefix sums over the CTA of two 0/1 flags per thread; totals in a_total, b_total.
template <int THREADS>
__device__ __forceinline__ void flag_ranks(unsigned* scan, bool a, bool b, int& a_rank, int& b_rank, int& a_total, int& b_total) {
    constexpr int kWarps = THREADS / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned ma = __ballot_sync(0xffffffffu, a), mb = __ballot_sync(0xffffffffu, b);
    if (lane == 0) scan[warp] = __popc(ma) | (__popc(mb) << 16);
    __syncthreads();
    unsigned before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const unsigned v = scan[w];
        if (w < warp) before += v;
        total += v;
    }
    const unsigned below = (1u << lane) - 1;
    a_rank = (before & 0xffff) + __popc(ma & below);
    b_rank = (before >> 16) + __popc(mb & below);
    a_total = total & 0xffff;
    b_total = total >> 16;
    __syncthreads();
}
#endif

}  // namespace sfb
