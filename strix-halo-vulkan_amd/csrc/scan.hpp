// Sums over the threads of a block that stop at a largest value, and bisection among what they leave.
#pragma once

#include "shv_device.hpp"

namespace shv {

constexpr uint32_t kFull = 1u << 30;  // sums stop here: no count of pages or rows that matters is as large

__device__ __forceinline__ uint32_t add_up_to(uint32_t a, uint32_t b) { return min(a + b, kFull); }

// Sum over a wave's lanes up to this one: four shifts within rows of 16 lanes, two carries between rows.  (By way of LDS six exchanges are a third of a microsecond.)
template <int CTRL, int ROW_MASK = 0xF>
__device__ __forceinline__ uint32_t shifted(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROW_MASK, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
    v = add_up_to(v, shifted<0x111>(v));
    v = add_up_to(v, shifted<0x112>(v));
    v = add_up_to(v, shifted<0x114>(v));
    v = add_up_to(v, shifted<0x118>(v));
    v = add_up_to(v, shifted<kDppBcast15, 0xA>(v));
    return add_up_to(v, shifted<kDppBcast31, 0xC>(v));
}

// N exclusive sums over a block of T threads, and the totals.
template <int T, int N>
__device__ __forceinline__ void block_scan(uint32_t (&v)[N], uint32_t (&total)[N], uint32_t (*waves)[T / 64]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t upto[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        upto[k] = wave_upto(v[k]);
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
        v[k] = add_up_to(before, shifted<0x138>(upto[k]));  // (the lane before's; of the first none)
        total[k] = all;
    }
    __syncthreads();  // `waves` is free again
}

// The same over the lanes of a wave.
template <int N>
__device__ __forceinline__ void wave_scan(uint32_t (&v)[N], uint32_t (&total)[N]) {
#pragma unroll
    for (int k = 0; k < N; k++) {
        const uint32_t upto = wave_upto(v[k]);
        total[k] = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(upto), 63));
        v[k] = shifted<0x138>(upto);
    }
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
