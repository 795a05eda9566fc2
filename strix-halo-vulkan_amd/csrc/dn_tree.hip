// The gated delta rule over a tree of drafted tokens, and the state behind the branch that is kept.
//
// Row i's state would be S_i = g_i S_parent + k_i delta_i^T.  Written out down to the committed state S0, with G_i the sum of
// log g from the root to i,
//     delta_i = beta_i (v_i - e^(G_i) S0^T k_i) - sum over ancestors j of beta_i e^(G_i - G_j) (k_j . k_i) delta_j
//     out_i   = (e^(G_i) S0^T q_i + sum over ancestors j and i itself of e^(G_i - G_j) (k_j . q_i) delta_j) / sqrt(d)
// so no row needs a state of its own: S0 is read once, whatever the tree's shape, and the deltas are a triangular solve whose
// matrix is masked by ancestry.
// What bounds it, of 16 key and 32 value heads: its chain of steps, each waiting for the one before.  In thousands of cycles of a block's first wave, 5
// rows of one sequence / 64 of each of eight: the sequence's words and parents 4 / 6, gates 1.5 / 5, rows 1.5 / 13 and the wait for the slowest wave's 0.5 / 2,
// products of rows 2.3 / 2.5, inverse and the products below the diagonal 0.1 / 3.3, products with the state 2.1 / 7.5, solve and outputs 2.1 / 10
// (14 and 49: 7.0 us, whose 2.5 MB would take 0.5, and 26; with up to 64 rows 22, whose 36 MB would take 8).
#include <atomic>

#include "shv_device.hpp"
#include "shv_internal.hpp"
#include "tree.hpp"

namespace {

using namespace shv;

constexpr int kBlock = 256;
constexpr int kD = 128;
constexpr int kRows = SHV_TREE_MAX_ROWS;
constexpr int kWaves = 8;

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float softplus_ref(float x) {
    // the add inside the log is float32 on purpose, as in the step's kernels: below about -16.6 it returns exactly 0
    return x > 20.f ? x : logf(1.f + expf(x));
}

// float32 operands enter the matrix cores as two binary16 values, the small one scaled by 2^11 so that it stays normal, three products
// a term: about 22 bits of each operand, accumulated in float32.
constexpr float kLoScale = 2048.f, kLoInv = 1.f / 2048.f;
__device__ __forceinline__ void split(float x, _Float16 &hi, _Float16 &lo) {
    hi = static_cast<_Float16>(x);
    lo = static_cast<_Float16>(fmaf(static_cast<float>(hi), -1.f, x) * kLoScale);
}
__device__ __forceinline__ void mma32(half8_t xh, half8_t xl, half8_t yh, half8_t yl, float4_t &main, float4_t &low) {
    main = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, yh, main, 0, 0, 0);
    low = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, yl, low, 0, 0, 0);
    low = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl, yh, low, 0, 0, 0);
}
// acc + X Y for 16 x 16 tiles in float32: lane (n, g) holds X[n][4g ..] and Y[4g ..][n], the sum's own layout.
__device__ __forceinline__ float4_t mma16(float4_t x, float4_t y, float4_t acc) {
#pragma unroll
    for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
    return acc;
}
__device__ __forceinline__ float max_over_g(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ uint32_t or_over_g(uint32_t v) {
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = r[0] | r[1];
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return r[0] | r[1];
}
// e to this is 0 in float32 beside anything it may be a factor of, the growth of other rows by up to e^800 included.
constexpr float kForgets = -1000.f;
// Sum over each half of the wave, in every lane of it.
__device__ __forceinline__ float sum32(float v) {
    v += dpp_f32<kDppXor1>(v);
    v += dpp_f32<kDppXor2>(v);
    v += dpp_f32<kDppHalfMirror>(v);
    v += dpp_f32<kDppMirror>(v);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The power of two that brings values of up to m to about 1 (of 0 and of what is no number, 1), and its inverse.
struct Scale {
    float down, up;
    __device__ __forceinline__ explicit Scale(float m) {
        int e = static_cast<int>(__float_as_uint(m) >> 23) - 126;  // m < 2^e
        e = m > 0.f && m < INFINITY ? min(max(e, -120), 126) : 0;  // (what is left over, a factor of four at most, the halves hold)
        down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    }
};

constexpr int kKS = kD + 8;      // halves between rows of the [64][128] operands (272 B: 16 rows cover all banks)
constexpr int kAS = kRows + 4;   // floats between rows of the [64][64] ones (272 B as well)
constexpr int kTS = 20;          // floats between rows of a 16 x 16 inverse
template <int CT>
struct TreeLds {
    _Float16 kh[kRows][kKS], kl[kRows][kKS], qh[kRows][kKS], ql[kRows][kKS];
    float a[kRows][kAS], m[kRows][kAS];  // -A below the diagonal blocks, and M
    float t[4][16][kTS];                 // the inverses of the diagonal blocks of I + A
    float adiag[4][16][17];
    float v[kRows][16 * CT + 4];
    double G[kRows];  // (differences of two of them are what counts: in float32 a row that forgets, log g = -100, would cost those behind it 2^-18)
    float beta[kRows];
    uint64_t anc[kRows];
    int lost[kRows];  // bit 0: A's row holds what is no number, bit 1: M's
};

// grid: (8 / CT, n_head_v, n_seq), eight waves: a value head's rows against CT tiles of 16 of its 128 value columns.
//   1  conv, SiLU and norm of q and k, conv and SiLU of v, a row a wave at a time, into LDS as operands
//   2  P = K K^T and R = Q K^T in tiles of 16 x 16 on and below the diagonal, A and M from them where the column's row is an
//      ancestor of the row's; the diagonal blocks of I + A inverted by substitution, a lane a column; and, a column tile a wave,
//      K and Q against the state, which goes from memory to registers once
//   3  a column tile a wave: the block rows' solve, the outputs.  A product's result is laid out as the next one's second operand,
//      so a column tile never leaves its wave
// The state enters the products scaled by a power of two a column, any float32: what binary16 cannot hold of it beside the column's largest, 2^-35 of that, is
// below the rounding of a sum of 128 products with them.  The deltas of one column are of different branches, of which one may be of any size beside another, so the solve's
// products are float32's own: where a row is no ancestor the weight is 0, and what it would add is exactly 0.  (With deltas as two binary16 values under a
// common scale the rows beside a branch 2^40 times theirs were off by 0.2.)
// A row whose delta is no number must reach its descendants alone, and the products are of whole tiles: A, M, B and the deltas are cleaned of such values
// first, and the outputs of rows that stand on one are made NaN at the end.
template <int CT>
__global__ __launch_bounds__(64 * kWaves, 2) void dn_tree_kernel(shv_dn_tree_args a) {
    extern __shared__ __align__(16) char raw[];
    TreeLds<CT> &L = *reinterpret_cast<TreeLds<CT> *>(raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int slab = blockIdx.x, h = blockIdx.y, seq = blockIdx.z, hk = h % a.n_head_k;
    const int qk = a.n_head_k * kD, vw = a.n_head_v * kD;
    const TreeWords words(a.count, a.pos, a.slot, a.parent, a.conv1d, seq, a.rows, lane);
    const float *x = a.x + static_cast<size_t>(seq) * a.rows * a.x_stride;
    // asked for before anything is known: each lane's row's gates, the convs' taps, the state's columns
    const float *gates = x + static_cast<size_t>(lane < a.rows ? lane : 0) * a.x_stride + 2 * qk + 2 * vw;
    const float alpha = gates[h], write = gates[a.n_head_v + h], dt_bias = load_in_turn(a.dt_bias + h), decay = load_in_turn(a.a + h);
    const int ch = lane < 32 ? hk * kD + 4 * lane : qk + hk * kD + 4 * (lane - 32);
    constexpr int VC = CT == 8 ? 2 : 1;  // columns of v a lane takes
    const int vcol = VC * (CT == 8 ? lane : lane & (16 * CT - 1)), vch = 2 * qk + h * kD + slab * 16 * CT + vcol;
    float4_t tap[4], vtap[VC];
#pragma unroll
    for (int c = 0; c < 4; c++) tap[c] = *reinterpret_cast<const float4_t *>(a.conv1d + static_cast<size_t>(ch + c) * 4);
#pragma unroll
    for (int c = 0; c < VC; c++) vtap[c] = *reinterpret_cast<const float4_t *>(a.conv1d + static_cast<size_t>(vch + c) * 4);
    const int slot = __builtin_amdgcn_readfirstlane(words.slot), pos = __builtin_amdgcn_readfirstlane(words.pos), rows = __builtin_amdgcn_readfirstlane(words.count);
    if (rows == 0) return;
    const int planes = a.n_planes > 1 ? a.n_planes : 1;
    const int cur = a.plane && planes > 1 ? static_cast<int>(static_cast<unsigned>(a.plane[slot]) % static_cast<unsigned>(planes)) : 0;
    const bool has_tile = wave < CT;  // of value columns
    float4_t S[4][2];
    if (has_tile) {
        const float *state = a.state + ((static_cast<size_t>(slot) * planes + cur) * a.n_head_v + h) * kD * kD + static_cast<size_t>((slab * CT + wave) * 16 + n) * kD + 8 * g;
#pragma unroll
        for (int ks = 0; ks < 4; ks++)
#pragma unroll
            for (int e = 0; e < 2; e++) S[ks][e] = *reinterpret_cast<const float4_t *>(state + 32 * ks + 4 * e);
    }
    const TreeRow t = tree_row(rows, words.parent, a.rows, lane);
    const int tiles = (rows + 15) / 16;
    const float *ring = a.ring + static_cast<size_t>(slot) * a.ring_slots * a.ring_stride;

    // ---- 1 ----
    struct Taps {
        float4_t qk[4];
        float v[4][VC];
    };
    // Where a lane's row's taps are: the row, its parent, grandparent and the one above it; behind the root the ring's rows.  Each is read as a buffer
    // of the conv's channels, and of none before the sequence's start, where loads give zeros: nothing waits to put them there, and a
    // row's loads stay on their way under the row before (where a select put the zeros, 64 rows of one sequence took 2 us more).
    const uint32_t width = static_cast<uint32_t>(2 * qk + vw) * 4;
    const float *from[3];
    uint64_t there[3];
    {
        int up = t.parent, back = 0;
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const int next = __shfl(t.parent, up < 0 ? 0 : up, 64);
            back += up < 0;
            const int p = pos - back;
            const uint32_t behind = p < 0 ? 0 : static_cast<uint32_t>(p) % static_cast<uint32_t>(a.ring_slots);
            from[k] = up < 0 ? ring + static_cast<size_t>(behind) * a.ring_stride : x + static_cast<size_t>(up) * a.x_stride;
            there[k] = __ballot(up >= 0 || p >= 0);
            up = up < 0 ? -1 : next;
        }
    }
    const auto load = [&](Taps &f, int r) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float *row = x + static_cast<size_t>(r) * a.x_stride;
            uint32_t bytes = width;
            if (k > 0) {
                const uint64_t at = reinterpret_cast<uint64_t>(from[k - 1]);
                const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(at), r), hi = __builtin_amdgcn_readlane(static_cast<int>(at >> 32), r);
                row = reinterpret_cast<const float *>(static_cast<uint64_t>(hi) << 32 | lo);
                bytes = there[k - 1] >> r & 1 ? width : 0;
            }
            const __amdgpu_buffer_rsrc_t buf = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(row), 0, bytes, 0x00027000);
            f.qk[k] = __builtin_bit_cast(float4_t, __builtin_amdgcn_raw_buffer_load_b128(buf, ch * 4, 0, 0));
            if constexpr (VC == 2) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b64(buf, vch * 4, 0, 0);
                f.v[k][0] = __uint_as_float(v[0]);
                f.v[k][1] = __uint_as_float(v[1]);
            } else {
                f.v[k][0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(buf, vch * 4, 0, 0));
            }
        }
    };
    Taps even, odd;
    if (wave < rows) load(even, wave);
    // One wave forms what all need of the gates, another leaves what shv_dn_keep does.
    if (wave == 0 || (wave == kWaves - 1 && slab == 0)) {
        const float log_g = lane < rows ? softplus_ref(alpha + dt_bias) * decay : 0.f;
        // Between rows a log g below kForgets, infinite perhaps, counts as kForgets: the sums stay numbers whose differences say what lies between them.
        const bool forgets = log_g < kForgets;
        const double G = tree_sum(t, forgets && wave == 0 ? kForgets : log_g, a.rows, lane);
        if (wave == 0) {
            L.G[lane] = G;
            L.beta[lane] = lane < rows ? sigmoid_exact(write) : 0.f;
            L.anc[lane] = t.ancestors;
            L.lost[lane] = 0;
        } else if (lane < rows) {
            const size_t at = (static_cast<size_t>(seq) * a.rows + lane) * a.n_head_v + h;
            a.decay[at] = static_cast<float>(G);
            if (a.log_g) a.log_g[at] = log_g;
        }
    }
    const auto silu = [](float c) { return c * __builtin_amdgcn_rcpf(1.f + __expf(-c)); };
    // a row of a wave's, and the loads of its next one under it
    const auto prepare = [&](Taps &now, Taps &next, int r) {
        float y[4], v[VC];
        if (r < rows) {
            if (r + kWaves < rows) load(next, r + kWaves);
            float ss = 0.f;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                float s = now.qk[3][c] * tap[c].x;
                s = fmaf(now.qk[2][c], tap[c].y, s);
                s = fmaf(now.qk[1][c], tap[c].z, s);
                y[c] = silu(fmaf(now.qk[0][c], tap[c].w, s));
                ss = fmaf(y[c], y[c], ss);
            }
#pragma unroll
            for (int c = 0; c < VC; c++) {
                float s = now.v[3][c] * vtap[c].x;
                s = fmaf(now.v[2][c], vtap[c].y, s);
                s = fmaf(now.v[1][c], vtap[c].z, s);
                v[c] = silu(fmaf(now.v[0][c], vtap[c].w, s));
            }
            ss = sum32(ss);
            const float nrm = a.qk_norm_max ? 1.f / fmaxf(sqrtf(ss), a.eps) : __builtin_amdgcn_rsqf(ss + a.eps);
#pragma unroll
            for (int c = 0; c < 4; c++) y[c] *= nrm;
            if (slab == 0 && h < a.n_head_k && lane >= 32)
                *reinterpret_cast<float4_t *>(a.kn + (static_cast<size_t>(seq) * a.rows + r) * qk + hk * kD + 4 * (lane - 32)) = float4_t{y[0], y[1], y[2], y[3]};
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) y[c] = 0.f;
#pragma unroll
            for (int c = 0; c < VC; c++) v[c] = 0.f;
        }
        half4_t hi, lo;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            _Float16 p, q;
            split(y[c], p, q);
            hi[c] = p;
            lo[c] = q;
        }
        *reinterpret_cast<half4_t *>(lane < 32 ? &L.qh[r][4 * lane] : &L.kh[r][4 * (lane - 32)]) = hi;
        *reinterpret_cast<half4_t *>(lane < 32 ? &L.ql[r][4 * lane] : &L.kl[r][4 * (lane - 32)]) = lo;
        if (CT == 8 || lane < 16 * CT) {
#pragma unroll
            for (int c = 0; c < VC; c++) L.v[r][vcol + c] = v[c];
        }
    };
    for (int r = wave; r < 16 * tiles; r += 2 * kWaves) {
        prepare(even, odd, r);
        prepare(odd, even, r + kWaves);
    }
    __syncthreads();

    // ---- 2 ----
    const auto tile = [&](int tt, int st) {
        float4_t pm = {0.f, 0.f, 0.f, 0.f}, pl = pm, rm = pm, rl = pm;
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            const int c = 32 * ks + 8 * g;
            const half8_t bh = *reinterpret_cast<const half8_t *>(&L.kh[16 * st + n][c]), bl = *reinterpret_cast<const half8_t *>(&L.kl[16 * st + n][c]);
            mma32(*reinterpret_cast<const half8_t *>(&L.kh[16 * tt + n][c]), *reinterpret_cast<const half8_t *>(&L.kl[16 * tt + n][c]), bh, bl, pm, pl);
            mma32(*reinterpret_cast<const half8_t *>(&L.qh[16 * tt + n][c]), *reinterpret_cast<const half8_t *>(&L.ql[16 * tt + n][c]), bh, bl, rm, rl);
        }
        const int s = 16 * st + n;
        const double Gs = L.G[s];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = 16 * tt + 4 * g + r;
            const bool above = (L.anc[row] >> s & 1) != 0;
            const float dec = __expf(static_cast<float>(L.G[row] - Gs));
            float av = above && s != row ? L.beta[row] * dec * fmaf(pl[r], kLoInv, pm[r]) : 0.f;
            float mv = above ? dec * fmaf(rl[r], kLoInv, rm[r]) : 0.f;
            if (!(fabsf(av) < INFINITY)) {
                atomicOr(&L.lost[row], 1);
                av = 0.f;
            }
            if (!(fabsf(mv) < INFINITY)) {
                atomicOr(&L.lost[row], 2);
                mv = 0.f;
            }
            if (st == tt) L.adiag[tt][4 * g + r][n] = av;
            else L.a[row][s] = -av;
            L.m[row][s] = mv;
        }
    };
    if (wave < tiles) tile(wave, wave);
    __syncthreads();
    if (wave == kWaves - 1) {
        // lane (block g, column n): its column of (I + A_gg)^-1, by forward substitution
        if (g < tiles) {
            float T[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float s0 = i == n ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
                for (int j = 0; j < i; j++) {
                    const float av = L.adiag[g][i][j];
                    if (j & 1) s1 = fmaf(-av, T[j], s1);
                    else s0 = fmaf(-av, T[j], s0);
                }
                T[i] = s0 + s1;
                L.t[g][i][n] = T[i];
            }
        }
    } else {
        // the tiles below the diagonal: (1,0) (2,0) (2,1) (3,0) (3,1) (3,2), one a wave
        const int tt = wave < 1 ? 1 : wave < 3 ? 2 : 3, st = wave < 1 ? 0 : wave < 3 ? wave - 1 : wave - 3;
        if (wave < 6 && tt < tiles) tile(tt, st);
    }
    float4_t B[4], O[4];  // of a row tile: B, and e^G Q S0
    uint32_t bad_lo = 0, bad_hi = 0;
    if (has_tile) {
        float m = 0.f;
#pragma unroll
        for (int ks = 0; ks < 4; ks++)
#pragma unroll
            for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(S[ks][e >> 2][e & 3]));
        const Scale scale(max_over_g(m));
        half8_t sh[4], sl[4];
#pragma unroll
        for (int ks = 0; ks < 4; ks++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                _Float16 hi, lo;
                split(S[ks][e >> 2][e & 3] * scale.down, hi, lo);
                sh[ks][e] = hi;
                sl[ks][e] = lo;
            }
#pragma unroll
        for (int tt = 0; tt < 4; tt++) {
            B[tt] = O[tt] = float4_t{0.f, 0.f, 0.f, 0.f};
            if (tt >= tiles) continue;
            float4_t km = {0.f, 0.f, 0.f, 0.f}, kl = km, qm = km, ql = km;
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
                const int c = 32 * ks + 8 * g;
                mma32(*reinterpret_cast<const half8_t *>(&L.kh[16 * tt + n][c]), *reinterpret_cast<const half8_t *>(&L.kl[16 * tt + n][c]), sh[ks], sl[ks], km, kl);
                mma32(*reinterpret_cast<const half8_t *>(&L.qh[16 * tt + n][c]), *reinterpret_cast<const half8_t *>(&L.ql[16 * tt + n][c]), sh[ks], sl[ks], qm, ql);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * tt + 4 * g + r;
                const float fall = __expf(static_cast<float>(L.G[row])) * scale.up;
                float b = L.beta[row] * (L.v[row][16 * wave + n] - fall * fmaf(kl[r], kLoInv, km[r]));
                if (!(fabsf(b) < INFINITY)) {
                    if (row < 32) bad_lo |= 1u << row;
                    else bad_hi |= 1u << (row - 32);
                    b = 0.f;
                }
                B[tt][r] = b;
                O[tt][r] = fall * fmaf(ql[r], kLoInv, qm[r]);
            }
        }
    }
    __syncthreads();
    if (!has_tile) return;

    // ---- 3 ----
    const int lost_here = L.lost[lane];
    uint64_t bad = (static_cast<uint64_t>(or_over_g(bad_hi)) << 32 | or_over_g(bad_lo)) | __ballot((lost_here & 1) != 0);
    const uint64_t bad_out = __ballot((lost_here & 2) != 0);
    const auto clean = [&](float4_t &of, int tt) {  // of sums past float32's range
        uint32_t over = 0;
#pragma unroll
        for (int r = 0; r < 4; r++) over |= fabsf(of[r]) < INFINITY ? 0u : 1u << (4 * g + r);
        if (__ballot(over != 0) == 0ull) return;
        bad |= static_cast<uint64_t>(or_over_g(over)) << (16 * tt);
#pragma unroll
        for (int r = 0; r < 4; r++) of[r] = over >> (4 * g + r) & 1 ? 0.f : of[r];
    };
    float4_t u[4];
    const float root = 1.f / sqrtf(static_cast<float>(kD));
#pragma unroll
    for (int tt = 0; tt < 4; tt++) {
        if (tt >= tiles) continue;
        // U_t = T_tt (B_t - sum over s < t of A_ts U_s)
        float4_t rest = B[tt];
#pragma unroll
        for (int st = 0; st < tt; st++) rest = mma16(*reinterpret_cast<const float4_t *>(&L.a[16 * tt + n][16 * st + 4 * g]), u[st], rest);
        clean(rest, tt);
        u[tt] = mma16(*reinterpret_cast<const float4_t *>(&L.t[tt][n][4 * g]), rest, float4_t{0.f, 0.f, 0.f, 0.f});
        clean(u[tt], tt);
        float4_t om = O[tt];
#pragma unroll
        for (int st = 0; st <= tt; st++) om = mma16(*reinterpret_cast<const float4_t *>(&L.m[16 * tt + n][16 * st + 4 * g]), u[st], om);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = 16 * tt + 4 * g + r;
            if (row >= rows) continue;
            const bool lost = (L.anc[row] & bad) != 0, lost_out = lost || (bad_out >> row & 1) != 0;
            const size_t at = (static_cast<size_t>(seq) * a.rows + row) * vw + static_cast<size_t>(h) * kD + (slab * CT + wave) * 16 + n;
            a.out[at] = lost_out ? __int_as_float(0x7fc00000) : om[r] * root;
            a.delta[at] = lost ? __int_as_float(0x7fc00000) : u[tt][r];
        }
    }
}

template <int CT>
int launch_tree(shv_ctx *ctx, const shv_dn_tree_args &a) {
    static std::atomic<uint64_t> raised{0};  // by device
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (!(raised.load(std::memory_order_acquire) & bit)) {
        SHV_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&dn_tree_kernel<CT>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(TreeLds<CT>))));
        raised.fetch_or(bit, std::memory_order_release);
    }
    SHV_LAUNCH(ctx, dn_tree_kernel<CT>, dim3(8 / CT, a.n_head_v, a.n_seq), dim3(64 * kWaves), sizeof(TreeLds<CT>), a);
    return SHV_OK;
}

// grid: (8 slabs of 16 state rows, n_head_v, n_seq): a thread holds eight values of one row.  Memory-bound: the state is read once
// and written once (twelve sequences of 32 heads, 54 MB: 13.8 us where the last-level cache still holds them, 19.1 from memory; one 3.9 us, the launch
// and two trips to memory).
constexpr int kKeepRows = 16;
// OWN: the rows' own log decays are there.
template <bool OWN>
__global__ __launch_bounds__(kBlock) void dn_keep_kernel(shv_dn_keep_args a) {
    __shared__ float fall[kRows];
    __shared__ int row[kRows];
    __shared__ float all;
    __shared__ int used;
    const int tid = threadIdx.x, lane = tid & 63;
    const int slab = blockIdx.x, h = blockIdx.y, seq = blockIdx.z, hk = h % a.n_head_k;
    const int where = a.slot ? a.slot[seq] : seq, slot = max(where, 0);  // (a sequence that is not there reads the first slot and writes nothing: no branch before the loads)
    const int planes = a.n_planes > 1 ? a.n_planes : 1;
    const int cur = a.plane ? static_cast<int>(static_cast<unsigned>(a.plane[slot]) % static_cast<unsigned>(planes)) : 0;
    const int next = cur + 1 < planes ? cur + 1 : 0;
    const size_t plane_floats = static_cast<size_t>(a.n_head_v) * kD * kD;
    const int j = slab * kKeepRows + tid / 16, i0 = tid % 16 * 4;
    float *at = a.state + static_cast<size_t>(slot) * planes * plane_floats + (static_cast<size_t>(h) * kD + j) * kD + i0;
    float4 s0 = *reinterpret_cast<const float4 *>(at + cur * plane_floats), s1 = *reinterpret_cast<const float4 *>(at + cur * plane_floats + 64);
    const int keep = max(0, min(a.n_keep[seq], a.rows));
    const size_t base = static_cast<size_t>(seq) * a.rows;
    if (tid < 64) {
        const int r = lane < keep ? a.path[base + lane] : -1;
        const bool on = r >= 0 && r < a.rows;
        const float G = on ? (OWN ? a.log_g : a.decay)[(base + r) * a.n_head_v + h] : 0.f;
        const uint64_t there = __ballot(on);
        const int n = __popcll(there);
        float behind, whole;  // log of the decay by the rows behind the lane's, and by all
        if constexpr (OWN) {
            double sum = G;  // from the lane's row to the last: each sum by itself, since of two long ones the difference loses what is short
#pragma unroll
            for (int far = 1; far < 64; far *= 2) {
                const double more = __shfl_down(sum, far, 64);
                sum += lane + far < 64 ? more : 0.0;
            }
            whole = static_cast<float>(__shfl(sum, 0, 64));
            const float next = static_cast<float>(__shfl_down(sum, 1, 64));
            behind = lane < 63 ? next : 0.f;
        } else {
            whole = n ? __shfl(G, 63 - __clzll(there), 64) : 0.f;
            behind = whole - G;
        }
        if (on) {
            const int k = __popcll(there & ((1ull << lane) - 1));
            fall[k] = expf(behind);
            row[k] = r;
        }
        if (lane == 0) {
            all = expf(whole);
            used = n;
        }
    }
    __syncthreads();
    if (where < 0) return;
    const int n = used;
    const float f = all;
    s0.x *= f; s0.y *= f; s0.z *= f; s0.w *= f;
    s1.x *= f; s1.y *= f; s1.z *= f; s1.w *= f;
    for (int e = 0; e < n; e++) {
        const size_t r = base + row[e];
        const float *k = a.kn + (r * a.n_head_k + hk) * kD + i0;
        const float d = a.delta[(r * a.n_head_v + h) * kD + j] * fall[e];
        const float4 k0 = *reinterpret_cast<const float4 *>(k), k1 = *reinterpret_cast<const float4 *>(k + 64);
        s0.x = fmaf(d, k0.x, s0.x); s0.y = fmaf(d, k0.y, s0.y); s0.z = fmaf(d, k0.z, s0.z); s0.w = fmaf(d, k0.w, s0.w);
        s1.x = fmaf(d, k1.x, s1.x); s1.y = fmaf(d, k1.y, s1.y); s1.z = fmaf(d, k1.z, s1.z); s1.w = fmaf(d, k1.w, s1.w);
    }
    *reinterpret_cast<float4 *>(at + next * plane_floats) = s0;
    *reinterpret_cast<float4 *>(at + next * plane_floats + 64) = s1;
    // the last three rows' conv channels, 256 a block
    const int ch = (h * (kD / kKeepRows) + slab) * kBlock + tid, cw = 2 * a.n_head_k * kD + a.n_head_v * kD;
    const int pos = a.pos ? a.pos[seq] : 0;
    if (ch < cw) {
        float *ring = a.ring + static_cast<size_t>(slot) * a.ring_slots * a.ring_stride;
        for (int e = max(0, keep - (a.conv - 1)); e < keep; e++) {
            const int r = a.path[base + e];
            const long long p = static_cast<long long>(pos) + e;
            if (r >= 0 && r < a.rows && p >= 0) ring[static_cast<size_t>(p % a.ring_slots) * a.ring_stride + ch] = a.x[(base + r) * a.x_stride + ch];
        }
    }
}

}  // namespace

int shv_launch_dn_tree(shv_ctx *ctx, const shv_dn_tree_args *pa) {
    const shv_dn_tree_args &a = *pa;
    SHV_REQUIRE(a.x && a.ring && a.conv1d && a.a && a.dt_bias && a.state && a.out && a.kn && a.delta && a.decay, "dn_tree: NULL argument");
    SHV_REQUIRE(a.rows >= 1 && a.rows <= kRows, "dn_tree: %d rows; 1..%d", a.rows, kRows);
    SHV_REQUIRE(a.n_seq >= 1 && a.n_seq <= 65535, "dn_tree: %d sequences", a.n_seq);
    SHV_REQUIRE(a.head_dim == kD, "dn_tree: head_dim %d; built for %d", a.head_dim, kD);
    SHV_REQUIRE(a.conv == 4, "dn_tree: conv kernel %d; built for 4", a.conv);
    SHV_REQUIRE(a.n_head_k >= 1 && a.n_head_v >= a.n_head_k && a.n_head_v % a.n_head_k == 0 && a.n_head_v <= 1024, "dn_tree: heads %d/%d", a.n_head_k, a.n_head_v);
    const int width = 2 * a.n_head_k * kD + 2 * a.n_head_v * kD + 2 * a.n_head_v, cw = 2 * a.n_head_k * kD + a.n_head_v * kD;
    SHV_REQUIRE(a.x_stride >= width, "dn_tree: x_stride %d < row width %d", a.x_stride, width);
    SHV_REQUIRE(a.ring_stride >= cw && a.ring_slots >= a.conv - 1, "dn_tree: a ring of %d rows %d floats apart", a.ring_slots, a.ring_stride);
    SHV_REQUIRE(a.n_planes >= 0 && a.n_planes <= 64, "dn_tree: %d state planes", a.n_planes);
    SHV_REQUIRE(shv_aligned16(a.x) && shv_aligned16(a.state) && shv_aligned16(a.conv1d) && shv_aligned16(a.ring) && shv_aligned16(a.out) &&
                    shv_aligned16(a.kn) && shv_aligned16(a.delta),
                "dn_tree: x, ring, conv1d, state, out, kn and delta must be 16-byte aligned");
    // Columns cut in four, two or not at all: as far as every block still finds a compute unit of its own (a block's rows are prepared anew
    // whatever its columns).  us of 5 / 64 rows of one sequence of 32 value heads cut in four 7.0 / 17.8, in two 7.4 / 17.8, whole
    // 9.3 / 21.5; of four sequences 12.5 / 36, 7.5 / 19.8, 9.4 / 23.6.
    const int heads = a.n_seq * a.n_head_v, units = ctx->prop.multiProcessorCount;
    if (4 * heads <= units) return launch_tree<2>(ctx, a);
    if (2 * heads <= units) return launch_tree<4>(ctx, a);
    return launch_tree<8>(ctx, a);
}

int shv_launch_dn_keep(shv_ctx *ctx, const shv_dn_keep_args *pa) {
    const shv_dn_keep_args &a = *pa;
    SHV_REQUIRE(a.x && a.kn && a.delta && (a.decay || a.log_g) && a.state && a.ring && a.path && a.n_keep, "dn_keep: NULL argument");
    SHV_REQUIRE(a.rows >= 1 && a.rows <= kRows, "dn_keep: %d rows; 1..%d", a.rows, kRows);
    SHV_REQUIRE(a.n_seq >= 1 && a.n_seq <= 65535, "dn_keep: %d sequences", a.n_seq);
    SHV_REQUIRE(a.head_dim == kD, "dn_keep: head_dim %d; built for %d", a.head_dim, kD);
    SHV_REQUIRE(a.conv == 4, "dn_keep: conv kernel %d; built for 4", a.conv);
    SHV_REQUIRE(a.n_head_k >= 1 && a.n_head_v >= a.n_head_k && a.n_head_v % a.n_head_k == 0 && a.n_head_v <= 1024, "dn_keep: heads %d/%d", a.n_head_k, a.n_head_v);
    const int cw = 2 * a.n_head_k * kD + a.n_head_v * kD;
    SHV_REQUIRE(a.x_stride >= cw, "dn_keep: x_stride %d < %d conv channels", a.x_stride, cw);
    SHV_REQUIRE(a.ring_stride >= cw && a.ring_slots >= a.conv - 1, "dn_keep: a ring of %d rows %d floats apart", a.ring_slots, a.ring_stride);
    SHV_REQUIRE(a.n_planes >= 0 && a.n_planes <= 64, "dn_keep: %d state planes", a.n_planes);
    SHV_REQUIRE(shv_aligned16(a.state) && shv_aligned16(a.kn), "dn_keep: state and kn must be 16-byte aligned");
    const dim3 grid(kD / kKeepRows, a.n_head_v, a.n_seq);
    if (a.log_g) SHV_LAUNCH(ctx, dn_keep_kernel<true>, grid, dim3(kBlock), 0, a);
    else SHV_LAUNCH(ctx, dn_keep_kernel<false>, grid, dim3(kBlock), 0, a);
    return SHV_OK;
}
