// Sums over the threads of a block that stop at a largest value, and bisection among what they leave.
#pragma once

#include "shv_device.hpp"

namespace shv {

constexpr uint32_t kFull = 1u << 30;  // sums stop here: no count of pages or rows that matters is as large

__device__ __forceinline__ uint32_t add_up_to(uint32_t a, uint32_t b) { return min(a + b, kFull); }

// N exclusive sums over a block of T threads, and the totals.
template <int T, int N>
__device__ __forceinline__ void block_scan(uint32_t (&v)[N], uint32_t (&total)[N], uint32_t (*waves)[T / 64]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t upto[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        upto[k] = v[k];
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t less = __shfl_up(upto[k], off, 64);
            if (lane >= off) upto[k] = add_up_to(upto[k], less);
        }
        if (lane == 63) waves[k][wave] = upto[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; k++) {
        uint32_t before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < T / 64; w++) {
            if (w == wave) before = all;
            all = add_up_to(all, waves[k][w]);
        }
        const uint32_t less = __shfl_up(upto[k], 1, 64);
        v[k] = lane == 0 ? before : add_up_to(before, less);
        total[k] = all;
    }
    __syncthreads();  // `waves` is free again
}

// The last of n ascending values that is not above x; the first is not.
__device__ __forceinline__ int last_not_above(const uint32_t *v, int n, uint32_t x) {
    int lo = 0;
    for (int hi = n; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

}  // namespace shv
