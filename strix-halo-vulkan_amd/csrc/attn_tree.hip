// Full attention over a tree of drafted tokens, and the kept branch's cells into the cache.
#include <atomic>

#include "shv_device.hpp"
#include "shv_internal.hpp"
#include "tree.hpp"

namespace {

using namespace shv;

constexpr int kBlock = 256;
constexpr int kTile = 32;  // cells of a tile of V
constexpr int kMaxSplits = 512;

// Whether a sequence's rows fit behind what it has kept; the others are left alone.
__device__ __forceinline__ bool fits(int pos, int n, int max_cells) { return n > 0 && pos >= 0 && pos <= max_cells - n; }

// Sum over a wave, in every lane.
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// A cell's value in binary16, by way of float32 (the compiler would fold the two conversions into one).
__device__ __forceinline__ __half cell_value(double v) {
    float f = static_cast<float>(v);
    asm("" : "+v"(f));
    return __float2half_rn(f);
}

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void *lds_ptr_t;

constexpr int kChunk = 64 * 16;
constexpr int kStages = 4, kAhead = kStages - 1;
constexpr int kMinTiles = 4;  // tiles a slice gets at least

// Which tiles of 32 cells a sequence's rows look at: the sinks', then those the window of the first row reaches.
struct Tiles {
    int sinks, first, all;
    __device__ __forceinline__ Tiles(const shv_attn_tree_args &a, int pos) {
        const int end = (pos + kTile - 1) / kTile;
        sinks = first = 0;
        if (a.window > 0) {
            sinks = (min(a.sinks, pos) + kTile - 1) / kTile;
            first = max(sinks, max(0, pos - a.window + 1) / kTile);
        }
        all = sinks + max(0, end - first);
    }
    __device__ __forceinline__ int at(int i) const { return i < sinks ? i : i - sinks + first; }
};

// How a call's sequences are cut: slices of `len` tiles as many as the call has blocks for, and behind them one for the rows
// themselves; where a call has one slice, it holds both.
struct Cut {
    int len, cache, all;  // tiles of a slice, slices of the cache, slices
    __device__ __forceinline__ Cut(const shv_attn_tree_args &a, int tiles, int slots, int lane) {
        long long total = 0;
        for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
            const int s = s0 + lane;
            int t = 0;
            if (s < a.n_seq) {
                const int pos = a.pos ? a.pos[s] : 0;
                const int n = tree_rows(a.count, s, a.rows);
                t = fits(pos, n, a.max_cells) ? Tiles(a, pos).all : 0;
            }
            int sum = t;
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
            total += sum;
        }
        if (a.n_splits == 1) {
            len = tiles;
            cache = 0;
            all = 1;
            return;
        }
        len = max(kMinTiles, static_cast<int>((total + slots - 1) / slots));
        len = max(len, (tiles + a.n_splits - 2) / (a.n_splits - 1));
        cache = (tiles + len - 1) / len;
        all = cache + 1;
    }
};

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

// The rotary factors of a lane's dims, of a position.
template <int D>
struct Turn {
    static constexpr int VEC = D / 64;
    float c[VEC], s[VEC];
    int partner;
    bool turns, first;
    __device__ __forceinline__ Turn(int rope_dims, int lane) {
        const int half = rope_dims / 2, e = VEC * lane;
        turns = e < rope_dims;
        first = e < half;
        partner = !turns ? lane : first ? lane + half / VEC : lane - half / VEC;
    }
    __device__ __forceinline__ void load(const float *table, int rope_dims, int lane) {
        const int half = rope_dims / 2, e = VEC * lane;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            c[v] = turns ? table[(first ? e : e - half) + v] : 1.f;
            s[v] = turns ? table[(first ? e + half : e) + v] : 0.f;
        }
    }
    template <typename T>
    __device__ __forceinline__ T of(T x, T other, int v) const {
        // first of the pair: x0' = x0 cos - x1 sin; second: x1' = x0 sin + x1 cos
        const T r = first ? x * static_cast<T>(c[v]) - other * static_cast<T>(s[v]) : other * static_cast<T>(s[v]) + x * static_cast<T>(c[v]);
        return turns ? r : x;
    }
};

// A tile in LDS: 1 KB chunks that a wave reads 16 bytes a lane.  K chunk T * (D/32) + i: lane (n, q) = cell 8 (n / 4) + 4 T + n % 4, dims
// 32 i + 8 q ..; V chunk db behind them: lane (n, q) = dim 16 db + n, cells 8 q ...  After S^T = K Q^T lane (n, q) then holds query row n's
// scores of cells 8 q + 4 T + 0..3, T = 0, 1: the eight cells of its operand of the second product.
template <int D>
__device__ __forceinline__ int k_byte(int cell, int dim) {
    const int T = (cell >> 2) & 1, n = (cell >> 3) * 4 + (cell & 3);
    return (T * (D / 32) + dim / 32) * kChunk + (16 * ((dim & 31) >> 3) + n) * 16 + (dim & 7) * 2;
}
template <int D>
__device__ __forceinline__ int v_byte(int cell, int dim) {
    return (D / 16 + (dim >> 4)) * kChunk + (16 * (cell >> 3) + (dim & 15)) * 16 + (cell & 7) * 2;
}

template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <int D, int W>
struct TreeSmem {
    char ring[kStages][D / 8 * kChunk];
    float p[W][16 * kTile];  // a wave's weights of a tile, where its values are not all finite
};

// grid: (slices rounded up to 8, times query blocks; n_head_kv; n_seq), W waves.  A wave holds 16 query rows: query row r of a KV head is
// head r % rep of tree row r / rep.
template <int D, int W>
__global__ __launch_bounds__(64 * W, D == 256 ? 2 : 4) void tree_attn_kernel(shv_attn_tree_args a, int q_blocks, int slots) {
    constexpr int VEC = D / 64, KI = D / 32, DB = D / 16;
    constexpr int kPer = D / 8 / W;  // chunks of a tile a wave asks for
    extern __shared__ __align__(16) char raw[];
    TreeSmem<D, W> &sm = *reinterpret_cast<TreeSmem<D, W> *>(raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, q = lane >> 4;
    // blocks of one slice lie on one die (workgroups go to the dies in turn) and find its tiles in the die's L2
    const int split = blockIdx.x / (8 * q_blocks) * 8 + (blockIdx.x & 7), qb = blockIdx.x / 8 % q_blocks;
    const int kvh = blockIdx.y, seq = blockIdx.z;
    const int rep = a.n_head / a.n_head_kv;
    const int slot = a.slot ? a.slot[seq] : seq, pos = a.pos ? a.pos[seq] : 0;
    const TreeRow t = tree_row(a.parent, a.count, seq, a.rows, lane);
    if (!fits(pos, t.n, a.max_cells) || qb * W * 16 >= t.n * rep) return;
    const Tiles tiles(a, pos);
    const Cut cut(a, tiles.all, slots, lane);
    if (split >= cut.all) return;
    const bool with_rows = split == cut.all - 1;
    const int t0 = with_rows && cut.all > 1 ? 0 : split * cut.len;
    const int t1 = with_rows && cut.all > 1 ? 0 : min(t0 + cut.len, tiles.all);

    const size_t kvw = static_cast<size_t>(a.n_head_kv) * D;
    const uint16_t *kc = static_cast<const uint16_t *>(a.kcache) + static_cast<size_t>(slot) * a.max_cells * kvw + kvh * D;
    const uint16_t *vc = static_cast<const uint16_t *>(a.vcache) + static_cast<size_t>(slot) * a.max_cells * kvw + static_cast<size_t>(kvh) * D * kTile;

    // ---- the wave's query rows are asked for, then the first two tiles ----
    const int r0 = (qb * W + wave) * 16, r_end = t.n * rep;  // rows past the last repeat it and are dropped
    Row<D> qx[16];
    const float *qkv = a.qkv + static_cast<size_t>(seq) * a.rows * a.qkv_stride;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int r = min(r0 + i, r_end - 1), tr = r / rep;
        qx[i].load(qkv + static_cast<size_t>(tr) * a.qkv_stride + static_cast<size_t>(kvh * rep + r - tr * rep) * 2 * D, lane);
    }
    Row<D> gq;
    gq.load(a.q_norm, lane);
    const bool keys = wave < W / 2;
    const int first = (keys ? wave : wave - W / 2) * kPer;  // of the wave's chunks among K's or V's
    const uint32_t from = keys ? static_cast<uint32_t>((8 * (n >> 2) + 4 * (first / KI) + (n & 3)) * kvw + 32 * (first % KI) + 8 * q) * 2
                               : static_cast<uint32_t>((16 * first + n) * kTile + 8 * q) * 2;
    auto ask = [&](int i) {
        const size_t at = static_cast<size_t>(tiles.at(i)) * kTile * kvw;
        const __amdgpu_buffer_rsrc_t bytes = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>((keys ? kc : vc) + at), 0, static_cast<uint32_t>(kTile * kvw) * 2, 0x00027000);
        char *to = sm.ring[(i - t0) & (kStages - 1)] + (wave * kPer) * kChunk;
#pragma unroll
        for (int u = 0; u < kPer; u++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(bytes, (lds_ptr_t)(to + u * kChunk), 16, from, u * (keys ? 64 : 1024), 0, 0);
    };
    if (t0 < t1) ask(t0);
    if (t0 + 1 < t1) ask(t0 + 1);

    // ---- queries: norm, rotation, operand order by way of the last two stages, half of the dims at a time ----
    half8_t qh[KI], ql[KI];
    {
        const Turn<D> shape(a.rope_dims, lane);
        Turn<D> turn = shape;
        int at_row = -1;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int r = min(r0 + i, r_end - 1), tr = r / rep;
            if (tr != at_row && a.rope_dims > 0) turn.load(a.rope + static_cast<size_t>(pos + __builtin_amdgcn_readlane(t.depth, tr)) * a.rope_dims, a.rope_dims, lane);
            at_row = tr;
            float ss = 0.f;
#pragma unroll
            for (int v = 0; v < VEC; v++) ss = fmaf(qx[i].x[v], qx[i].x[v], ss);
            const float sc = 1.f / sqrtf(wave_sum_all(ss) / static_cast<float>(D) + a.eps);
            float y[VEC], o[VEC];
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                y[v] = qx[i].x[v] * sc * gq.x[v];
                o[v] = __shfl(y[v], turn.partner, 64);
            }
#pragma unroll
            for (int v = 0; v < VEC; v++) qx[i].x[v] = a.rope_dims > 0 ? turn.of(y[v], o[v], v) : y[v];
        }
        // a wave's share: [dim step of the half][hi, lo][lane] 16 bytes
        char *mine = sm.ring[2] + wave * (KI / 2 * 2 * kChunk);
        static_assert(W * KI * kChunk <= 2 * (D / 8) * kChunk, "the last two stages hold all waves' shares");
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if ((lane >> 5) == h) {
                const int e = VEC * (lane & 31);  // dim within the half
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    _Float16 hi[VEC], lo[VEC];
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
                        hi[v] = static_cast<_Float16>(qx[i].x[v]);
                        lo[v] = static_cast<_Float16>(qx[i].x[v] - static_cast<float>(hi[v]));
                    }
                    char *dst = mine + (e / 32) * 2 * kChunk + (16 * ((e & 31) >> 3) + i) * 16 + (e & 7) * 2;
                    __builtin_memcpy(__builtin_assume_aligned(dst, 2 * VEC), hi, sizeof(hi));
                    __builtin_memcpy(__builtin_assume_aligned(dst + kChunk, 2 * VEC), lo, sizeof(lo));
                }
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < KI / 2; i++) {
                qh[h * (KI / 2) + i] = *reinterpret_cast<const half8_t *>(mine + (2 * i) * kChunk + lane * 16);
                ql[h * (KI / 2) + i] = *reinterpret_cast<const half8_t *>(mine + (2 * i + 1) * kChunk + lane * 16);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
    const bool working = r0 < r_end;
    const int my_tr = min(r0 + n, r_end - 1) / rep;                 // the lane's query row's tree row
    const int my_pos = pos + __shfl(t.depth, my_tr, 64);
    const int my_first = a.window > 0 ? my_pos - a.window + 1 : 0;  // sees sinks and positions from here on
    const float c2 = 1.44269504088896f / sqrtf(static_cast<float>(D));

    float4_t o[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) o[db] = float4_t{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;  // of the scores as they are, before their scale

    // one tile; sees(c): whether the lane's row sees cell c of it, asked where `part` says that some row may not see some cell
    auto tile = [&](const char *kt, bool part, auto sees) {
        const char *vt = kt + 2 * KI * kChunk;
        float4_t st[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, lo[2] = {st[0], st[0]};
#pragma unroll
        for (int i = 0; i < KI; i++)
#pragma unroll
            for (int T = 0; T < 2; T++) {
                const half8_t k = *reinterpret_cast<const half8_t *>(kt + (T * KI + i) * kChunk + lane * 16);
                st[T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[i], st[T], 0, 0, 0);
                lo[T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[i], lo[T], 0, 0, 0);
            }
        float mx = -INFINITY;
        uint32_t seen = 0xFF;
        if (part) {
            seen = 0;
#pragma unroll
            for (int T = 0; T < 2; T++)
#pragma unroll
                for (int i = 0; i < 4; i++) seen |= sees(8 * q + 4 * T + i) ? 1u << (4 * T + i) : 0u;
        }
#pragma unroll
        for (int T = 0; T < 2; T++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                st[T][i] += lo[T][i];
                if (part) st[T][i] = seen >> (4 * T + i) & 1 ? st[T][i] : -INFINITY;
                mx = fmaxf(mx, st[T][i]);
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(m_run, mx);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        const float m2 = m_use * c2;
        float sum = 0.f, pv[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            pv[e] = __builtin_amdgcn_exp2f(fmaf(st[e >> 2][e & 3], c2, -m2));
            sum += pv[e];
        }
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        const float alpha = __builtin_amdgcn_exp2f(fmaf(m_run, c2, -m2));
        l_run = l_run * alpha + sum;
        m_run = m_new;
        if (__ballot(alpha != 1.f) != 0ull) {
            float av[4];
#pragma unroll
            for (int i = 0; i < 4; i++) av[i] = __shfl(alpha, 4 * q + i, 64);
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[db][i] *= av[i];
        }
        if (part) {
            // a value that is not finite meets the weight 0 of rows that do not see it: such a tile is multiplied by hand
            bool odd = false;
#pragma unroll
            for (int db = 0; db < DB; db++) {
                const uint4 v = *reinterpret_cast<const uint4 *>(vt + db * kChunk + lane * 16);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; e++) odd = odd || (w[e] & 0x7C00u) == 0x7C00u || (w[e] & 0x7C000000u) == 0x7C000000u;
            }
            if (__ballot(odd) != 0ull) {
                float *p = sm.p[wave];
#pragma unroll
                for (int e = 0; e < 8; e++) p[n * kTile + 8 * q + e] = seen >> e & 1 ? pv[e] : -1.f;
                __builtin_amdgcn_wave_barrier();
                for (int c = 0; c < kTile; c++) {
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = p[(4 * q + i) * kTile + c];
#pragma unroll
                    for (int db = 0; db < DB; db++) {
                        const float v = static_cast<float>(*reinterpret_cast<const _Float16 *>(vt + db * kChunk + (16 * (c >> 3) + n) * 16 + (c & 7) * 2));
#pragma unroll
                        for (int i = 0; i < 4; i++) o[db][i] = w[i] < 0.f ? o[db][i] : fmaf(w[i], v, o[db][i]);
                    }
                }
                __builtin_amdgcn_wave_barrier();
                return;
            }
        }
        half8_t ph, pl;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            ph[e] = static_cast<_Float16>(pv[e]);
            pl[e] = static_cast<_Float16>(pv[e] - static_cast<float>(ph[e]));
        }
#pragma unroll
        for (int db = 0; db < DB; db++) {
            const half8_t v = *reinterpret_cast<const half8_t *>(vt + db * kChunk + lane * 16);
            o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, v, o[db], 0, 0, 0);
            o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, v, o[db], 0, 0, 0);
        }
    };

    // ---- the slice's tiles: three on their way while one is multiplied; one barrier a tile ----
    __syncthreads();  // every wave holds its queries: the last two stages are free
    if (t0 + 2 < t1) ask(t0 + 2);
    for (int i = t0; i < t1; i++) {
        // a wave's loads complete in order: this tile's have landed when no more are out than those behind it
        if (i + 2 < t1) wait_loads<2 * kPer>();
        else if (i + 1 < t1) wait_loads<kPer>();
        else wait_loads<0>();
        asm volatile("s_barrier" ::: "memory");  // everyone's: this tile is whole, and the stage of the one before is free
        if (i + kAhead < t1) ask(i + kAhead);
        if (!working) continue;
        const int c0 = tiles.at(i) * kTile;
        const bool part = c0 + kTile > pos || (a.window > 0 && c0 + kTile > a.sinks && c0 < pos + t.n - a.window);
        tile(sm.ring[(i - t0) & (kStages - 1)], part, [&](int c) {
            c += c0;
            return c < pos && (a.window == 0 || c < a.sinks || c >= my_first);
        });
    }
    if (with_rows) {
        // ---- the rows' own cells: normed, rotated and rounded into two more tiles, and left for whoever keeps them ----
        __syncthreads();
        const int n_tiles = (t.n + kTile - 1) / kTile;
        const Turn<D> shape(a.rope_dims, lane);
        Row<D> gk;
        gk.load(a.k_norm, lane);
        for (int j = wave; j < n_tiles * kTile; j += W) {
            char *to = sm.ring[j / kTile];
            uint16_t kx[VEC], vx[VEC];
#pragma unroll
            for (int v = 0; v < VEC; v++) kx[v] = vx[v] = 0;
            if (j < t.n) {
                const float *src = qkv + static_cast<size_t>(j) * a.qkv_stride + static_cast<size_t>(a.n_head) * 2 * D + kvh * D;
                Row<D> k, val;
                k.load(src, lane);
                val.load(src + kvw, lane);
                Turn<D> turn = shape;
                if (a.rope_dims > 0) turn.load(a.rope + static_cast<size_t>(pos + __builtin_amdgcn_readlane(t.depth, j)) * a.rope_dims, a.rope_dims, lane);
                double ss = 0;
#pragma unroll
                for (int v = 0; v < VEC; v++) ss += static_cast<double>(k.x[v]) * k.x[v];
                const double sc = 1.0 / sqrt(wave_sum_f64(ss) / D + a.eps);
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    const double y = k.x[v] * sc * gk.x[v], other = __shfl(y, turn.partner, 64);
                    kx[v] = __half_as_ushort(cell_value(a.rope_dims > 0 ? turn.of(y, other, v) : y));
                    vx[v] = __half_as_ushort(__float2half_rn(val.x[v]));
                }
                if (qb == 0) {
                    const size_t cell = (static_cast<size_t>(seq) * a.rows + j) * kvw + kvh * D + VEC * lane;
                    __builtin_memcpy(__builtin_assume_aligned(static_cast<uint16_t *>(a.kcells) + cell, 2 * VEC), kx, sizeof(kx));
                    __builtin_memcpy(__builtin_assume_aligned(static_cast<uint16_t *>(a.vcells) + cell, 2 * VEC), vx, sizeof(vx));
                }
            }
            __builtin_memcpy(__builtin_assume_aligned(to + k_byte<D>(j % kTile, VEC * lane), 2 * VEC), kx, sizeof(kx));
#pragma unroll
            for (int v = 0; v < VEC; v++) *reinterpret_cast<uint16_t *>(to + v_byte<D>(j % kTile, VEC * lane + v)) = vx[v];
        }
        __syncthreads();
        uint64_t see = static_cast<uint64_t>(__shfl(static_cast<uint32_t>(t.ancestors >> 32), my_tr, 64)) << 32 | __shfl(static_cast<uint32_t>(t.ancestors), my_tr, 64);
        if (a.window > 0 && a.window < t.n) {
            uint64_t in = 0;
            for (int j = 0; j < t.n; j++) {
                const int p = pos + __builtin_amdgcn_readlane(t.depth, j);
                in |= p < a.sinks || p >= my_first ? 1ull << j : 0ull;
            }
            see &= in;
        }
        if (working)
            for (int i = 0; i < n_tiles; i++) tile(sm.ring[i], true, [&](int c) { return (see >> (i * kTile + c) & 1) != 0; });
    }
    if (!working) return;
    if (cut.all == 1) {
        float lr[4];
#pragma unroll
        for (int i = 0; i < 4; i++) lr[i] = __shfl(l_run, 4 * q + i, 64);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = r0 + 4 * q + i, tr = r / rep;
            if (r >= r_end) continue;
            float *dst = a.out + ((static_cast<size_t>(seq) * a.rows + tr) * a.n_head + kvh * rep + r - tr * rep) * D;
#pragma unroll
            for (int db = 0; db < DB; db++) dst[16 * db + n] = o[db][i] / lr[i];
        }
        return;
    }
    // the slice's record of each query row: unnormalised sums, then (max, sum)
    float *rec = a.partial + ((static_cast<size_t>(seq) * a.n_head_kv + kvh) * a.n_splits + split) * (a.rows * rep) * (D + 2);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = r0 + 4 * q + i;
        if (r >= r_end) continue;
#pragma unroll
        for (int db = 0; db < DB; db++) rec[static_cast<size_t>(r) * (D + 2) + 16 * db + n] = o[db][i];
    }
    if (q == 0 && r0 + n < r_end) *reinterpret_cast<float2 *>(rec + static_cast<size_t>(r0 + n) * (D + 2) + D) = make_float2(m_run, l_run);
}

// grid: (n_head * D / 64, rows, n_seq), a block 64 dims of a row's head: its waves share the slices' records, each folds its share with all of a
// batch's loads on their way together, and the first wave folds their results.
constexpr int kMergeWaves = 8;
template <int D>
__global__ __launch_bounds__(64 * kMergeWaves) void tree_merge_kernel(shv_attn_tree_args a, int slots) {
    __shared__ float red[3][kMergeWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int head = blockIdx.x / (D / 64), d = blockIdx.x % (D / 64) * 64 + lane, row = blockIdx.y, seq = blockIdx.z;
    const int rep = a.n_head / a.n_head_kv, kvh = head / rep;
    const int pos = a.pos ? a.pos[seq] : 0, rows = tree_rows(a.count, seq, a.rows);
    if (row >= rows || !fits(pos, rows, a.max_cells)) return;
    const Cut cut(a, Tiles(a, pos).all, slots, lane);
    if (cut.all == 1) return;  // put straight out
    const float c2 = 1.44269504088896f / sqrtf(static_cast<float>(D));
    const size_t step = static_cast<size_t>(a.rows) * rep * (D + 2);
    const float *from = a.partial + (static_cast<size_t>(seq) * a.n_head_kv + kvh) * a.n_splits * step + static_cast<size_t>(row * rep + head % rep) * (D + 2);
    constexpr int MB = 16;
    float num = 0.f, den = 0.f, M = -INFINITY;
    for (int s0 = wave; s0 < cut.all; s0 += kMergeWaves * MB) {
        float v[MB];
        float2 ml[MB];
#pragma unroll
        for (int u = 0; u < MB; u++) {
            const int s = s0 + kMergeWaves * u < cut.all ? s0 + kMergeWaves * u : s0;
            v[u] = from[s * step + d];
            ml[u] = *reinterpret_cast<const float2 *>(from + s * step + D);
        }
#pragma unroll
        for (int u = 0; u < MB; u++) asm volatile("" : "+v"(v[u]));  // asked for together, not each behind the one before's test
#pragma unroll
        for (int u = 0; u < MB; u++) {
            if (s0 + kMergeWaves * u >= cut.all || (ml[u].x == -INFINITY && ml[u].y == 0.f)) continue;  // (sees nothing; a sum of NaN stays)
            const float Mn = fmaxf(M, ml[u].x);
            const float shrink = __builtin_amdgcn_exp2f((M - Mn) * c2), w = __builtin_amdgcn_exp2f((ml[u].x - Mn) * c2);
            den = fmaf(den, shrink, w * ml[u].y);
            num = fmaf(num, shrink, w * v[u]);
            M = Mn;
        }
    }
    red[0][wave][lane] = M;
    red[1][wave][lane] = den;
    red[2][wave][lane] = num;
    __syncthreads();
    if (wave != 0) return;
    float Mt = red[0][0][lane];
#pragma unroll
    for (int k = 1; k < kMergeWaves; k++) Mt = fmaxf(Mt, red[0][k][lane]);
    float nt = 0.f, dt = 0.f;
#pragma unroll
    for (int k = 0; k < kMergeWaves; k++) {
        const float mk = red[0][k][lane];
        if (mk == -INFINITY && red[1][k][lane] == 0.f) continue;
        const float w = __builtin_amdgcn_exp2f((mk - Mt) * c2);
        dt = fmaf(w, red[1][k][lane], dt);
        nt = fmaf(w, red[2][k][lane], nt);
    }
    a.out[((static_cast<size_t>(seq) * a.rows + row) * a.n_head + head) * D + d] = nt / dt;
}

template <int D, int W>
int launch_tree(shv_ctx *ctx, const shv_attn_tree_args &a) {
    const int rep = a.n_head / a.n_head_kv;
    const int q_blocks = (a.rows * rep + 16 * W - 1) / (16 * W);
    constexpr int kBlocksPerUnit = D == 256 ? 1 : 2;
    // slices of the cache all sequences have together: as many blocks as the chip holds at once
    int slots = ctx->prop.multiProcessorCount * kBlocksPerUnit / (a.n_head_kv * q_blocks) - a.n_seq;
    if (slots < 1) slots = 1;
    static std::atomic<uint64_t> raised{0};  // by device
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (!(raised.load(std::memory_order_acquire) & bit)) {
        SHV_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&tree_attn_kernel<D, W>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(TreeSmem<D, W>))));
        raised.fetch_or(bit, std::memory_order_release);
    }
    // a sequence may have all the slices of the cache to itself, and those its share leaves over
    const int most = a.n_splits < slots + 1 + a.n_seq ? a.n_splits : slots + 1 + a.n_seq;
    shv_attn_tree_args b = a;
    b.n_splits = most;
    SHV_LAUNCH(ctx, (tree_attn_kernel<D, W>), dim3((most + 7) / 8 * 8 * q_blocks, a.n_head_kv, a.n_seq), dim3(64 * W), sizeof(TreeSmem<D, W>), b, q_blocks, slots);
    if (most > 1) SHV_LAUNCH(ctx, tree_merge_kernel<D>, dim3(a.n_head * (D / 64), a.rows, a.n_seq), dim3(64 * kMergeWaves), 0, b, slots);
    return SHV_OK;
}

template <int D>
int launch_tree(shv_ctx *ctx, const shv_attn_tree_args &a) {
    return a.rows * (a.n_head / a.n_head_kv) <= 64 ? launch_tree<D, 4>(ctx, a) : launch_tree<D, 8>(ctx, a);
}

// grid: (rows, n_seq): one kept row; the cells' keys lie as they will, their values go to their places in a tile of 32 cells.
__global__ __launch_bounds__(kBlock) void attn_keep_kernel(shv_attn_keep_args a) {
    const int j = blockIdx.x, seq = blockIdx.y, d = a.head_dim, kvw = a.n_head_kv * d;
    const int keep = min(a.n_keep[seq], a.rows);
    const int row = a.path[static_cast<size_t>(seq) * a.rows + j];
    const int slot = a.slot ? a.slot[seq] : seq;
    const long long c = (a.pos ? a.pos[seq] : 0) + static_cast<long long>(j);
    if (j >= keep || row < 0 || row >= a.rows || c < 0 || c >= a.max_cells) return;
    const size_t from = (static_cast<size_t>(seq) * a.rows + row) * kvw;
    const uint4 *k = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.kcells) + from);
    const uint16_t *v = static_cast<const uint16_t *>(a.vcells) + from;
    uint4 *kd = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.kcache) + (static_cast<size_t>(slot) * a.max_cells + c) * kvw);
    uint16_t *vd = static_cast<uint16_t *>(a.vcache) + (static_cast<size_t>(slot) * a.max_cells + c / kTile * kTile) * kvw + c % kTile;
    for (int i = threadIdx.x; i < kvw / 8; i += kBlock) kd[i] = k[i];
    for (int i = threadIdx.x; i < kvw; i += kBlock) vd[static_cast<size_t>(i) * kTile] = v[i];
}

}  // namespace

int shv_launch_attn_tree(shv_ctx *ctx, const shv_attn_tree_args *pa) {
    const shv_attn_tree_args &a = *pa;
    SHV_REQUIRE(a.qkv && a.q_norm && a.k_norm && a.kcache && a.vcache && a.kcells && a.vcells && a.partial && a.out, "attn_tree: NULL argument");
    SHV_REQUIRE(a.rows >= 1 && a.rows <= SHV_TREE_MAX_ROWS, "attn_tree: %d rows; 1..%d", a.rows, SHV_TREE_MAX_ROWS);
    SHV_REQUIRE(a.n_seq >= 1 && a.n_seq <= 65535, "attn_tree: %d sequences", a.n_seq);
    SHV_REQUIRE(a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256, "attn_tree: head_dim %d; 64, 128 or 256", a.head_dim);
    SHV_REQUIRE(a.n_head_kv >= 1 && a.n_head >= 1 && a.n_head % a.n_head_kv == 0 && a.n_head / a.n_head_kv <= 64 && a.n_head <= 1024,
                "attn_tree: %d query heads over %d KV heads; 1..64 per KV head, 1024 in all", a.n_head, a.n_head_kv);
    SHV_REQUIRE(a.rope_dims >= 0 && a.rope_dims <= a.head_dim && a.rope_dims % (a.head_dim / 32) == 0,
                "attn_tree: rope_dims %d; a multiple of %d up to %d", a.rope_dims, a.head_dim / 32, a.head_dim);
    SHV_REQUIRE(a.rope || a.rope_dims == 0, "attn_tree: NULL rotary table");
    SHV_REQUIRE(a.max_cells >= kTile && a.max_cells % kTile == 0, "attn_tree: max_cells %d; a multiple of %d", a.max_cells, kTile);
    SHV_REQUIRE(a.qkv_stride >= (a.n_head + a.n_head_kv) * 2 * a.head_dim && a.qkv_stride % 4 == 0, "attn_tree: qkv_stride %d", a.qkv_stride);
    SHV_REQUIRE(a.n_splits >= 1 && a.n_splits <= kMaxSplits, "attn_tree: %d slices; 1..%d", a.n_splits, kMaxSplits);
    SHV_REQUIRE(a.window >= 0 && a.sinks >= 0, "attn_tree: window %d, sinks %d", a.window, a.sinks);
    SHV_REQUIRE(shv_aligned16(a.qkv) && shv_aligned16(a.kcache) && shv_aligned16(a.vcache) && shv_aligned16(a.kcells) && shv_aligned16(a.vcells) &&
                    shv_aligned16(a.q_norm) && shv_aligned16(a.k_norm) && shv_aligned16(a.out) && shv_aligned16(a.partial),
                "attn_tree: qkv, norms, caches, cells, partial and out must be 16-byte aligned");
    if (a.head_dim == 256) return launch_tree<256>(ctx, a);
    if (a.head_dim == 128) return launch_tree<128>(ctx, a);
    return launch_tree<64>(ctx, a);
}

int shv_launch_attn_keep(shv_ctx *ctx, const shv_attn_keep_args *pa) {
    const shv_attn_keep_args &a = *pa;
    SHV_REQUIRE(a.kcells && a.vcells && a.kcache && a.vcache && a.path && a.n_keep, "attn_keep: NULL argument");
    SHV_REQUIRE(a.rows >= 1 && a.rows <= SHV_TREE_MAX_ROWS, "attn_keep: %d rows; 1..%d", a.rows, SHV_TREE_MAX_ROWS);
    SHV_REQUIRE(a.n_seq >= 1 && a.n_seq <= 65535, "attn_keep: %d sequences", a.n_seq);
    SHV_REQUIRE(a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256, "attn_keep: head_dim %d; 64, 128 or 256", a.head_dim);
    SHV_REQUIRE(a.n_head_kv >= 1 && a.n_head_kv <= 1024, "attn_keep: %d KV heads", a.n_head_kv);
    SHV_REQUIRE(a.max_cells >= kTile && a.max_cells % kTile == 0, "attn_keep: max_cells %d; a multiple of %d", a.max_cells, kTile);
    SHV_REQUIRE(shv_aligned16(a.kcells) && shv_aligned16(a.vcells) && shv_aligned16(a.kcache) && shv_aligned16(a.vcache), "attn_keep: cells and caches must be 16-byte aligned");
    SHV_LAUNCH(ctx, attn_keep_kernel, dim3(a.rows, a.n_seq), dim3(kBlock), 0, a);
    return SHV_OK;
}
