// Rows of heads as attention kernels prepare them: a lane a few dims, the norm and the rotation, cells and operands in binary16; and what lanes that share a
// query row of a matrix-core tile exchange.
#pragma once

#include "shv_device.hpp"

namespace shv {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void *lds_ptr_t;

// Sum over a wave, in every lane.
template <int CTRL, int ROW_MASK = 0xF>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, ROW_MASK, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, ROW_MASK, 0xF, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
    v += dpp_f64<kDppXor1>(v);
    v += dpp_f64<kDppXor2>(v);
    v += dpp_f64<kDppHalfMirror>(v);
    v += dpp_f64<kDppMirror>(v);
    v += dpp_f64<kDppBcast15, 0xA>(v);
    v += dpp_f64<kDppBcast31, 0xC>(v);
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), 63), hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), 63);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// 1 / sqrt(x) to the last places: the instruction's estimate and two Newton steps (of 0 and infinity the estimate is the result).
__device__ __forceinline__ double rsqrt_f64(double x) {
    const double e = __builtin_amdgcn_rsq(x);
    double y = fma(e * 0.5, fma(-x * e, e, 1.0), e);
    y = fma(y * 0.5, fma(-x * y, y, 1.0), y);
    return x == 0.0 || x == static_cast<double>(INFINITY) ? e : y;
}

// A cell's value in binary16, by way of float32 (the compiler would fold the two conversions into one).
__device__ __forceinline__ __half cell_value(double v) {
    float f = static_cast<float>(v);
    asm("" : "+v"(f));
    return __float2half_rn(f);
}

template <int D>
struct Row {  // a lane's dims of one head's row: VEC * lane ..
    static constexpr int VEC = D / 64;
    float x[VEC];
    __device__ __forceinline__ void load(const float *p, int lane) {
        if constexpr (VEC == 4) {
            const float4 v = *reinterpret_cast<const float4 *>(p + 4 * lane);
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else if constexpr (VEC == 2) {
            const float2 v = *reinterpret_cast<const float2 *>(p + 2 * lane);
            x[0] = v.x; x[1] = v.y;
        } else {
            x[0] = p[lane];
        }
    }
};

// The rotation of a lane's dims at a position, x' = x c + other s: of a pair the first is x0 cos - x1 sin, the second x1 cos + x0 sin, and
// a dim that does not turn has c = 1, s = 0.  (Lanes without a rotated dim read the first's factors: no branch around loads.)
template <int D>
struct Turn {
    static constexpr int VEC = D / 64;
    Row<D> c, s;
    int partner, at;
    bool turns, first;
    __device__ __forceinline__ Turn(int rope_dims, int lane) {
        const int half = rope_dims / 2, e = VEC * lane;
        turns = e < rope_dims;
        first = e < half;
        at = !turns ? 0 : first ? lane : lane - half / VEC;
        partner = !turns ? lane : first ? lane + half / VEC : at;
    }
    __device__ __forceinline__ void load(const float *table, int rope_dims) {
        c.load(table, at);
        s.load(table + rope_dims / 2, at);
    }
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            c.x[v] = turns ? c.x[v] : 1.f;
            s.x[v] = turns ? (first ? -s.x[v] : s.x[v]) : 0.f;
        }
    }
};

// Largest and sum over the four lanes (n, 0..3) that share a query row.
__device__ __forceinline__ float max_over_q(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_q(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// A row's key, normed and rotated, as the lane's dims' halves.
template <int D>
__device__ __forceinline__ void cell_key(const Row<D> &k, const Row<D> &gamma, const Turn<D> &turn, int rope_dims, float eps, uint16_t (&out)[D / 64]) {
    double ss = 0;
#pragma unroll
    for (int v = 0; v < D / 64; v++) ss = fma(static_cast<double>(k.x[v]), static_cast<double>(k.x[v]), ss);
    const double sc = rsqrt_f64(fma(wave_sum_f64(ss), 1.0 / D, static_cast<double>(eps)));
#pragma unroll
    for (int v = 0; v < D / 64; v++) {
        double y = k.x[v] * sc * gamma.x[v];
        if (rope_dims > 0) y = y * turn.c.x[v] + __shfl(y, turn.partner, 64) * turn.s.x[v];
        out[v] = __half_as_ushort(cell_value(y));
    }
}
// A query row as large and small halves.
template <int D>
__device__ __forceinline__ void split_row(const float (&y)[D / 64], _Float16 (&hi)[D / 64], _Float16 (&lo)[D / 64]) {
#pragma unroll
    for (int v = 0; v < D / 64; v++) {
        hi[v] = static_cast<_Float16>(y[v]);
        lo[v] = static_cast<_Float16>(fmaf(static_cast<float>(hi[v]), -1.f, y[v]));
    }
}
template <int BYTES, typename T>
__device__ __forceinline__ void put_bytes(void *to, const T *from) { __builtin_memcpy(__builtin_assume_aligned(to, BYTES), from, BYTES); }

}  // namespace shv
