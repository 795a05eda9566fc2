// Full attention over a tree of drafted tokens, and the kept branch's cells into the cache.
//
// Row i of a tree, at position p_i = pos + depth_i, sees the cells c < pos, the rows on its way to the root and itself; with a window those of
// them alone whose position is below `sinks` or above p_i - window:
//     out_i = sum over them of softmax(q_i . k_j / sqrt(d)) v_j
// q and k normed over a head and rotated at their positions.  A block takes one KV head, a slice of the cache in tiles of 32 cells and up to
// 64 or 128 query rows (query row r is head r % rep of tree row r / rep), 16 a wave, on v_mfma_f32_16x16x32_f16:
//     S^T = K Q^T   the cache's binary16 keys against the queries as two halves; a lane then holds eight cells of one query row, the operand
//                   of the second product
//     O  += P V     weights as two halves against values, which the cache holds by dim
// with a running maximum and sum.  Tiles go from memory to LDS past the registers, three ahead.  The rows' own keys and values never enter the
// cache here: one more block of a KV head forms their cells, attends over them by the ancestors' bits, and leaves them for attn_keep.  A second
// launch joins the slices.
// What bounds it: one or two rows behind a long cache the cache's bytes (131000 cells 53 us, 5.1 TB/s of K and V, much of it from the last-level cache); 64 rows products and their
// operands' reads from LDS, each half of the cycles at its rate, with the softmax on the vector units between them (64 rows of 16 heads behind 131000
// cells 258 us, 1.06 PFLOP/s of binary16 products, where a large library product reaches 1.18); short
// caches the chain of trips to memory before the first product (2 rows behind 700 cells 9 us and 4 for the join).
#include <atomic>

#include "shv_device.hpp"
#include "shv_internal.hpp"
#include "tree.hpp"

namespace {

using namespace shv;

constexpr int kBlock = 256;
constexpr int kTile = 32;  // cells of a tile of V
constexpr int kMaxSplits = 512;

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

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void *lds_ptr_t;

constexpr int kChunk = 64 * 16;
constexpr int kStages = 4, kAhead = kStages - 1;
// Weights are e^(s - m) 2^kLift, and m stands until a score is more than kSlack powers of two above it: up to 2^15.9, which the larger half holds (2^16 is too
// much), and down to 2^-35 of the largest with the smaller half's last place, to which it is rounded and not cut: behind a first cell that takes nearly all and has
// no value, as models have it, the output is what small weights make of theirs (3000 cells of 2^-20 in one slice, cut off at 2^-31, 2.4e-4 low).
// Behind 131000 cells / the windowed batch, us: lift 7 and slack 8 264 / 38.0, 11 and 4.9 264 / 37.9, 11 and 4 265 / 38.3, 12 and 3 269 / 39.6, 14 and 1 272 / 39.5.
constexpr float kLift = 11.f, kSlack = 4.9f;
constexpr int kLeastNarrow = 2, kLeastWide = 3;  // tiles a slice gets at least: launch_tree has the figures
// Waves that join the slices of 256 dims' rows: one where there are many such pieces, eight where there are some, four where there are few.  us
// by one / four / eight waves: 32 pieces of 13 slices 3.9 / 4.2 / 5.4 (of 130 slices one wave would go to memory nine times in a row), 192 of
// 95 14.5 / 8.6 / 7.6, 1024 of 32 10.8 / 11.9 / 19, 2016 of 11 6.0 / 10.7 / 21.  Whole calls of 128 dims: 256 pieces 31.0 / 27.0 / 27.7, 1024 45.8 / 47.0 /
// 53.6; of 64 dims: 64 pieces 28.4 / 21.7 / 20.8, 256 31.6 / 27.3 / 28.1, 1024 47.2 / 48.9 / 56.7 (one line for all widths costs their middle 0.8).
constexpr int kMergeMany = 512, kMergeSome = 64;

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

// What the launcher works out once.
struct Plan {
    int q_blocks;        // blocks that share a slice, 16 query rows a wave
    int least;           // tiles a slice gets at least
    int slots;           // full slices of the cache that all sequences may have together: with the others as many blocks as the chip holds at once
    int32_t *len;        // of several sequences, where the slices' length is left for the join
    uint32_t rep_magic;  // r / rep = r * rep_magic >> 20 for r < 4096 and rep <= 64: off by less than r / 2^20 <= 1 / 256 before it is cut
};
__device__ __forceinline__ int over_rep(const Plan &plan, int r) { return static_cast<int>(static_cast<uint32_t>(r) * plan.rep_magic >> 20); }

// Tiles that sequence s looks at; -1: it is left alone, as any behind the last is.
__device__ __forceinline__ int tiles_of(const shv_attn_tree_args &a, int s) {
    if (s >= a.n_seq) return -1;
    const int pos = a.pos ? a.pos[s] : 0;
    return tree_fits(pos, tree_rows(a.count, s, a.rows), a.max_cells) ? Tiles(a, pos).all : -1;
}

// Tiles that all sequences look at.
__device__ __forceinline__ uint32_t all_tiles(const shv_attn_tree_args &a, int lane) {
    uint32_t total = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
        uint32_t sum = max(tiles_of(a, s0 + lane), 0);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
        total = min(total + sum, 1u << 30);  // (64 sequences have at most 2^32 / 2^6 tiles)
    }
    return __builtin_amdgcn_readfirstlane(total);
}

// Of several sequences, tiles a slice may have: the least for which all slices of the cache find a block.  Slices as long as the full ones
// alone call for, 1 / slots of all tiles, are enough whatever the sequences' remainders; 1 / (slots + n_seq) is the least that could be.  A lane tries a
// length between (longest 62 steps apart), by float32 quotients that are exact below 2^21.  Not tried
// where it could take off an eighth or less (us of eight sequences of up to 54 rows of 32 heads behind up to 1872 cells 70, so 62; of 20 rows behind up
// to 16000 116, so 104; six windows that it does not change 38.0 either way, 38.6 with the trial).
__device__ __forceinline__ int call_len(const shv_attn_tree_args &a, const Plan &plan, int lane) {
    const uint32_t total = all_tiles(a, lane), most = plan.slots + a.n_seq;
    const int hi = max(static_cast<int>((total + plan.slots - 1) / plan.slots), plan.least), lo = max(static_cast<int>((total + most - 1) / most), plan.least);
    if (hi - lo <= hi / 8 || total >= 1u << 20) return hi;
    const int mine = lane == 63 ? hi : min(hi, lo + lane * ((hi - lo + 62) / 63));
    const float inv = 1.f / static_cast<float>(mine), up = static_cast<float>(mine) - 0.5f;
    uint32_t slices = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
        const float tiles = static_cast<float>(max(tiles_of(a, s0 + lane), 0));
        for (int s = 0; s < min(64, a.n_seq - s0); s++) slices += static_cast<uint32_t>((__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(tiles), s)) + up) * inv);
    }
    return __builtin_amdgcn_readlane(mine, __ffsll(static_cast<unsigned long long>(__ballot(slices <= most || lane == 63))) - 1);
}

// How a call's sequences are cut: slices, of several sequences of equal length, as many as the call has blocks for, and behind them one for the rows
// themselves; where a call has one slice, it holds both.  most: call_len of several sequences.
template <bool MANY>
struct Cut {
    int len, cache, all;  // tiles of a slice, slices of the cache, slices
    __device__ __forceinline__ Cut(const shv_attn_tree_args &a, int tiles, int most, const Plan &plan) {
        if (a.n_splits == 1) {
            len = tiles;
            cache = 0;
            all = 1;
            return;
        }
        const uint32_t slots = plan.slots, least = plan.least, share = (tiles + slots - 1) / slots, room = a.n_splits - 1;
        uint32_t l = MANY ? most : share > least ? share : least;
        if (l * static_cast<uint64_t>(room) < static_cast<uint32_t>(tiles)) l = (tiles + room - 1) / room;
        cache = (tiles + l - 1) / l;
        len = MANY && cache > 1 ? (tiles + cache - 1) / cache : l;  // (one sequence's last slice may be short: a division less)
        all = cache + 1;
    }
};

// The `work`-th slice of all the call's: whose it is and which of its own; seq -1: there are fewer.  The slices stand in a row, without gaps for
// sequences that have fewer of them: blocks that find nothing to do and end, one in seven between those that work, leave the latter on
// few compute units (six windows of 9 slices in a grid of 64 a sequence 66 us, of 72 40, in a row 24, and 27 with the count of all that makes them of like length).
template <bool MANY>
struct Slice {
    int seq, split;
    __device__ __forceinline__ Slice(const shv_attn_tree_args &a, int work, int most, const Plan &plan, int lane) {
        seq = MANY ? -1 : 0;
        split = work;
        if (!MANY) return;
        int before = 0;
        for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
            const int tiles = tiles_of(a, s0 + lane);
            const int mine = tiles < 0 ? 0 : Cut<true>(a, tiles, most, plan).all;
            int upto = mine;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int less = __shfl_up(upto, off, 64);
                if (lane >= off) upto += less;
            }
            const uint64_t past = __ballot(before + upto > work);
            if (past != 0) {
                const int l = __ffsll(static_cast<unsigned long long>(past)) - 1;
                seq = s0 + l;
                split = work - before - __builtin_amdgcn_readlane(upto - mine, l);
                return;
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
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

// ---- the same work for the launch before a wide call's, and inside a narrow one's --------------------------------------------------
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

// Where the rows' operands of a wide call lie: of group g (16 query rows, fewer in a KV head's last) of a KV head, [dim step][large, small]
// [dims 8 q ..][row] 16 bytes.  As many bytes as the rows have floats.
__device__ __forceinline__ char *staged(char *stage, const shv_attn_tree_args &a, int seq, int kvh, int rows, int rep, int g, int D) {
    return stage + (static_cast<size_t>(seq) * a.rows * a.n_head + static_cast<size_t>(kvh) * rows * rep + 16 * g) * D * 4;
}

// A wide call's query rows as operands, and its rows' cells.  grid: (ceil((rows * n_head + rows * n_head_kv) / 4), n_seq), a wave a query row or a
// row's cell of a KV head.  Bound by its chain of trips to memory (parents, then the position's rotation): 4 us whatever its size.
template <int D>
__global__ __launch_bounds__(256) void tree_prep_kernel(shv_attn_tree_args a, Plan plan, char *stage) {
    constexpr int VEC = D / 64, KI = D / 32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), seq = blockIdx.y;
    const int rep = a.n_head / a.n_head_kv;
    const TreeWords words(a.count, a.pos, a.slot, a.parent, a.q_norm, seq, a.rows, lane);
    const int item = blockIdx.x * 4 + wave, cell0 = a.rows * a.n_head;
    if (item >= cell0 + a.rows * a.n_head_kv) return;
    const bool query = item < cell0;
    const int per = query ? a.n_head : a.n_head_kv, i = query ? item : item - cell0;
    const int row = static_cast<int>(static_cast<uint32_t>(i) / static_cast<uint32_t>(per)), head = i - row * per;
    const float *src = a.qkv + (static_cast<size_t>(seq) * a.rows + row) * a.qkv_stride + static_cast<size_t>(query ? head : a.n_head) * 2 * D + (query ? 0 : head * D);
    Row<D> x, gamma, val;
    x.load(src, lane);
    val.load(query ? src : src + static_cast<size_t>(a.n_head_kv) * D, lane);
    gamma.load(query ? a.q_norm : a.k_norm, lane);
    const int pos = __builtin_amdgcn_readfirstlane(words.pos), rows = __builtin_amdgcn_readfirstlane(words.count);
    if (row >= rows || !tree_fits(pos, rows, a.max_cells)) return;
    const TreeRow t = tree_row(rows, words.parent, a.rows, lane);
    Turn<D> turn(a.rope_dims, lane);
    if (a.rope_dims > 0) {
        turn.load(a.rope + static_cast<size_t>(pos + __builtin_amdgcn_readlane(t.depth, row)) * a.rope_dims, a.rope_dims);
        turn.settle();
    }
    if (!query) {
        uint16_t kx[VEC], vx[VEC];
        cell_key<D>(x, gamma, turn, a.rope_dims, a.eps, kx);
#pragma unroll
        for (int v = 0; v < VEC; v++) vx[v] = __half_as_ushort(__float2half_rn(val.x[v]));
        const size_t cell = ((static_cast<size_t>(seq) * a.rows + row) * a.n_head_kv + head) * D + VEC * lane;
        put_bytes<2 * VEC>(static_cast<uint16_t *>(a.kcells) + cell, kx);
        put_bytes<2 * VEC>(static_cast<uint16_t *>(a.vcells) + cell, vx);
        return;
    }
    float ss = 0.f, y[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) ss = fmaf(x.x[v], x.x[v], ss);
    const float sc = __builtin_amdgcn_rsqf(fmaf(wave_sum_all(ss), 1.f / static_cast<float>(D), a.eps));
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        y[v] = x.x[v] * sc * gamma.x[v];
        if (a.rope_dims > 0) y[v] = fmaf(__shfl(y[v], turn.partner, 64), turn.s.x[v], y[v] * turn.c.x[v]);
    }
    _Float16 hi[VEC], lo[VEC];
    split_row<D>(y, hi, lo);
    const int kvh = over_rep(plan, head), r = row * rep + head - kvh * rep, g = r >> 4, here = min(16, rows * rep - 16 * g), e = VEC * lane;
    char *dst = staged(stage, a, seq, kvh, rows, rep, g, D) + ((e / 32) * 8 + ((e & 31) >> 3)) * here * 16 + (r & 15) * 16 + (e & 7) * 2;
    put_bytes<2 * VEC>(dst, hi);
    put_bytes<2 * VEC>(dst + 4 * here * 16, lo);
    static_assert(KI * 32 == D, "whole steps");
}

// Floats of all records' sums.
__device__ __forceinline__ size_t record_floats(const shv_attn_tree_args &a, int D) { return static_cast<size_t>(a.n_seq) * a.rows * a.n_head * a.n_splits * D; }

template <int D, int W>
struct TreeSmem {
    char ring[kStages][D / 8 * kChunk];
    float p[W][16 * kTile / 2];  // a wave's weights of half a tile, where its values are not all finite (a whole one's would leave a unit one block of D 128)
};

// grid: (slices rounded up to 8, times query blocks; n_head_kv), W waves of 16 query rows.  MANY: several sequences; of one the slices are known
// without counting (one kernel for both costs a call of one 0.2 to 0.5 us).  Four waves: calls of up to 64 query rows a KV head, whose
// rows every block norms and turns itself, the waves sharing the rows of however few groups there are.  Eight: wider ones, whose rows a
// launch before (tree_prep_kernel) has left as operands.  There every block would have 128 rows to prepare, 5 us before its first product,
// and the launch costs 4 (us of 12 rows behind 9000 cells so / with the launch 31.7 / 30.1, a batch of six windows 68 / 54, before the steps that brought
// these to 26 and 38).  Of 128 dims eight waves hold 128 registers each, so that two blocks share a unit, and 10 more stand in scratch memory, 36 bytes a lane.
// Tried beside it: two groups a wave, so that an operand read serves both (512 registers a lane do not hold them: 1130 us where this takes
// 260); a tile's keys multiplied under the weights of the one before (275 for 260); half of the waves half a tile behind the others (263, and a
// batch of six windows 43 for 37).
template <int D, int W, bool MANY>
__global__ __launch_bounds__(64 * W, W == 4 || D == 256 ? 2 : 4) void tree_attn_kernel(shv_attn_tree_args a, Plan plan, char *stage) {
    constexpr bool kWide = W == 8;
    constexpr int VEC = D / 64, KI = D / 32, DB = D / 16;
    constexpr int kPer = D / 8 / W;  // chunks of a tile a wave asks for
    extern __shared__ __align__(16) char raw[];
    TreeSmem<D, W> &sm = *reinterpret_cast<TreeSmem<D, W> *>(raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, q = lane >> 4;
    // blocks of one slice lie on one die (workgroups go to the dies in turn) and find its tiles in the die's L2
    const int eight = blockIdx.x >> 3, of_eight = static_cast<int>(static_cast<uint32_t>(eight) / static_cast<uint32_t>(plan.q_blocks));
    const int work = of_eight * 8 + (blockIdx.x & 7), qb = eight - of_eight * plan.q_blocks;
    const int kvh = blockIdx.y;
    const int most = MANY && a.n_splits > 1 ? call_len(a, plan, lane) : 0;
    if (MANY && blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) *plan.len = most;
    const Slice<MANY> slice(a, work, most, plan, lane);
    if (slice.seq < 0) return;
    const int seq = __builtin_amdgcn_readfirstlane(slice.seq), split = __builtin_amdgcn_readfirstlane(slice.split);
    const int rep = a.n_head / a.n_head_kv;
    const TreeWords words(a.count, a.pos, a.slot, a.parent, a.q_norm, seq, a.rows, lane);
    const float *qkv = a.qkv + static_cast<size_t>(seq) * a.rows * a.qkv_stride;
    // ---- GW 1: what depends on nothing, the first query rows this wave prepares.  The waves share the rows of all groups (there is often one),
    //      four rows of a group each ----
    const int groups_here = !kWide ? (a.rows * rep + 15) / 16 : 0;
    const auto row_of = [&](int f, int u) { return 16 * f + 4 * u + wave; };
    const auto load_four = [&](Row<D>(&x)[4], int f) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int r = min(row_of(f, u), a.rows * rep - 1), tr = over_rep(plan, r);  // (rows past the last repeat it and are dropped)
            x[u].load(qkv + static_cast<size_t>(tr) * a.qkv_stride + static_cast<size_t>(kvh * rep + r - tr * rep) * 2 * D, lane);
        }
    };
    Row<D> qx[4], gq;
    if constexpr (!kWide) {
        load_four(qx, 0);
        gq.load(a.q_norm, lane);
    }
    const int slot = words.slot, pos = __builtin_amdgcn_readfirstlane(words.pos), rows = __builtin_amdgcn_readfirstlane(words.count);
    const int r_end = rows * rep;
    if (!tree_fits(pos, rows, a.max_cells) || qb * W * 16 >= r_end) return;
    const Tiles tiles(a, pos);
    const Cut<MANY> cut(a, tiles.all, most, plan);
    if (split >= cut.all) return;
    const bool with_rows = split == cut.all - 1;
    const int t0 = with_rows && cut.all > 1 ? 0 : split * cut.len;
    const int t1 = with_rows && cut.all > 1 ? 0 : min(t0 + cut.len, tiles.all);

    const size_t kvw = static_cast<size_t>(a.n_head_kv) * D;
    const uint16_t *kc = static_cast<const uint16_t *>(a.kcache) + static_cast<size_t>(slot) * a.max_cells * kvw + kvh * D;
    const uint16_t *vc = static_cast<const uint16_t *>(a.vcache) + static_cast<size_t>(slot) * a.max_cells * kvw + static_cast<size_t>(kvh) * D * kTile;
    const bool keys = wave < W / 2;
    const int first = (keys ? wave : wave - W / 2) * kPer;  // of the wave's chunks among K's or V's
    const uint32_t from = keys ? static_cast<uint32_t>((8 * (n >> 2) + 4 * (first / KI) + (n & 3)) * kvw + 32 * (first % KI) + 8 * q) * 2
                               : static_cast<uint32_t>((16 * first + n) * kTile + 8 * q) * 2;
    // The block's tiles in a row: the rows' own, n_own of them, then the slice's.  Tile j lies in stage j % kStages.
    const int n_own = with_rows ? (rows + kTile - 1) / kTile : 0, n_tiles = n_own + t1 - t0;
    const auto ask = [&](int j) {
        const size_t at = static_cast<size_t>(tiles.at(t0 + j - n_own)) * kTile * kvw;
        const __amdgpu_buffer_rsrc_t bytes = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>((keys ? kc : vc) + at), 0, static_cast<uint32_t>(kTile * kvw) * 2, 0x00027000);
        char *to = sm.ring[j & (kStages - 1)] + (wave * kPer) * kChunk;
#pragma unroll
        for (int u = 0; u < kPer; u++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(bytes, (lds_ptr_t)(to + u * kChunk), 16, from, u * (keys ? 64 : 1024), 0, 0);
    };
    // (loads complete in order: what the prologue needs goes out before the tiles do)
    const int r0 = (qb * W + wave) * 16;
    const bool working = r0 < r_end;
    half8_t qh[KI], ql[KI];
    if constexpr (kWide) {
        // a group that is not there is the last one again, and dropped
        const int g = min(r0, r_end - 1) / 16, here = min(16, r_end - 16 * g);
        const char *mine = staged(stage, a, seq, kvh, rows, rep, g, D) + (q * here + min(n, here - 1)) * 16;
#pragma unroll
        for (int i = 0; i < KI; i++) {
            qh[i] = *reinterpret_cast<const half8_t *>(mine + (i * 8) * here * 16);
            ql[i] = *reinterpret_cast<const half8_t *>(mine + (i * 8 + 4) * here * 16);
        }
    }
    // (a wide call's slice of the cache has no use for the tree but for a window's edge: 2 of its 24 thousand cycles)
    TreeRow t{rows, -1, 0, 0};
    if (!kWide || with_rows || a.window > 0) t = tree_row(rows, words.parent, a.rows, lane);
    const Turn<D> shape(a.rope_dims, lane);
    const auto load_turn = [&](Turn<D> &turn, int row) { turn.load(a.rope + static_cast<size_t>(pos + __builtin_amdgcn_readlane(t.depth, row)) * a.rope_dims, a.rope_dims); };
    const auto turn_four = [&](Turn<D>(&turn)[4], int f) {
        if (a.rope_dims == 0) return;
#pragma unroll
        for (int u = 0; u < 4; u++) load_turn(turn[u], min(over_rep(plan, row_of(f, u)), rows - 1));
    };
    Turn<D> q_turn[4] = {shape, shape, shape, shape};
    if constexpr (!kWide) turn_four(q_turn, 0);
    if (!with_rows) {
        ask(0);
        if (1 < n_tiles) ask(1);
    }
    if (with_rows) {
        // ---- the rows' own cells go into the first two stages; GW 1: normed, rotated and rounded here, and left for whoever keeps them ----
        if (rows % kTile != 0) {
            // behind the last row the second product wants something finite
            uint4 *v = reinterpret_cast<uint4 *>(sm.ring[n_own - 1] + 2 * KI * kChunk);
            for (int i = tid; i < DB * 64; i += 64 * W) v[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
        }
        const auto place = [&](int j, const uint16_t(&kx)[VEC], const uint16_t(&vx)[VEC]) {
            char *to = sm.ring[j / kTile];
            put_bytes<2 * VEC>(to + k_byte<D>(j % kTile, VEC * lane), kx);
#pragma unroll
            for (int v = 0; v < VEC; v++) *reinterpret_cast<uint16_t *>(to + v_byte<D>(j % kTile, VEC * lane + v)) = vx[v];
        };
        const size_t cell0 = static_cast<size_t>(seq) * a.rows * kvw + kvh * D + VEC * lane;
        if constexpr (kWide) {
            for (int j0 = wave; j0 < rows; j0 += 4 * W) {
                uint16_t kx[4][VEC], vx[4][VEC];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const size_t cell = cell0 + min(j0 + u * W, rows - 1) * kvw;
                    put_bytes<2 * VEC>(kx[u], static_cast<const uint16_t *>(__builtin_assume_aligned(static_cast<const uint16_t *>(a.kcells) + cell, 2 * VEC)));
                    put_bytes<2 * VEC>(vx[u], static_cast<const uint16_t *>(__builtin_assume_aligned(static_cast<const uint16_t *>(a.vcells) + cell, 2 * VEC)));
                }
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (j0 + u * W < rows) place(j0 + u * W, kx[u], vx[u]);
            }
        } else {
            Row<D> gk, k, val;
            gk.load(a.k_norm, lane);
            Turn<D> turn = shape;
            const auto load = [&](int j) {
                const float *src = qkv + static_cast<size_t>(j) * a.qkv_stride + static_cast<size_t>(a.n_head) * 2 * D + kvh * D;
                k.load(src, lane);
                val.load(src + kvw, lane);
                if (a.rope_dims > 0) load_turn(turn, j);
            };
            if (wave < rows) load(wave);
            for (int j = wave; j < rows; j += W) {
                if (a.rope_dims > 0) turn.settle();
                uint16_t kx[VEC], vx[VEC];
                cell_key<D>(k, gk, turn, a.rope_dims, a.eps, kx);
#pragma unroll
                for (int v = 0; v < VEC; v++) vx[v] = __half_as_ushort(__float2half_rn(val.x[v]));
                if (j + W < rows) load(j + W);  // under the rest of this one
                put_bytes<2 * VEC>(static_cast<uint16_t *>(a.kcells) + cell0 + j * kvw, kx);
                put_bytes<2 * VEC>(static_cast<uint16_t *>(a.vcells) + cell0 + j * kvw, vx);
                place(j, kx, vx);
            }
        }
    }
    if constexpr (!kWide) {
        // ---- queries: norm, rotation, and operand order by way of the last two stages: [group][large, small][dim step][dims 8 q ..][row] 16 bytes ----
        constexpr int kPart = KI * kChunk;
        static_assert(2 * W * kPart <= 2 * (D / 8) * kChunk, "the last two stages hold all groups' operands");
        char *here = sm.ring[2];
        // row i's 16 bytes of dims 32 d + 8 q ..: turned on among the rows' places, since a row, written at once, would ask the same few banks
        const auto place = [&](int i, int d, int q) { return (16 * q + ((i + 4 * d + q) & 15)) * 16; };
        for (int f = 0; f < groups_here; f++) {
            Row<D> next[4];
            Turn<D> next_turn[4] = {shape, shape, shape, shape};
            if (f + 1 < groups_here) {
                load_four(next, f + 1);
                turn_four(next_turn, f + 1);
            }
            float y[4][VEC], other[4][VEC];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                float ss = 0.f;
#pragma unroll
                for (int v = 0; v < VEC; v++) ss = fmaf(qx[u].x[v], qx[u].x[v], ss);
                const float sc = __builtin_amdgcn_rsqf(fmaf(wave_sum_all(ss), 1.f / static_cast<float>(D), a.eps));
#pragma unroll
                for (int v = 0; v < VEC; v++) y[u][v] = qx[u].x[v] * sc * gq.x[v];
            }
            if (a.rope_dims > 0) {
#pragma unroll
                for (int u = 0; u < 4; u++) {
#pragma unroll
                    for (int v = 0; v < VEC; v++) other[u][v] = __shfl(y[u][v], shape.partner, 64);
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    q_turn[u].settle();
#pragma unroll
                    for (int v = 0; v < VEC; v++) y[u][v] = fmaf(other[u][v], q_turn[u].s.x[v], y[u][v] * q_turn[u].c.x[v]);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                _Float16 hi[VEC], lo[VEC];
                split_row<D>(y[u], hi, lo);
                const int e = VEC * lane;
                char *dst = here + 2 * f * kPart + (e / 32) * kChunk + place(4 * u + wave, e / 32, (e & 31) >> 3) + (e & 7) * 2;
                put_bytes<2 * VEC>(dst, hi);
                put_bytes<2 * VEC>(dst + kPart, lo);
            }
#pragma unroll
            for (int u = 0; u < 4; u++) qx[u] = next[u], q_turn[u] = next_turn[u];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KI; i++) {
            qh[i] = *reinterpret_cast<const half8_t *>(here + 2 * wave * kPart + i * kChunk + place(n, i, q));
            ql[i] = *reinterpret_cast<const half8_t *>(here + (2 * wave + 1) * kPart + i * kChunk + place(n, i, q));
        }
    }
    int my_first;    // the first position the lane's row sees, but for the sinks
    uint64_t mates;  // the rows it sees
    {
        const int tr = over_rep(plan, min(r0 + n, r_end - 1));
        my_first = a.window > 0 ? pos + __shfl(t.depth, tr, 64) - a.window + 1 : 0;
        mates = static_cast<uint64_t>(__shfl(static_cast<uint32_t>(t.ancestors >> 32), tr, 64)) << 32 | __shfl(static_cast<uint32_t>(t.ancestors), tr, 64);
        if (a.window > 0 && a.window < rows) {
            uint64_t in = 0;
            for (int j = 0; j < rows; j++) {
                const int p = pos + __builtin_amdgcn_readlane(t.depth, j);
                in |= p < a.sinks || p >= my_first ? 1ull << j : 0ull;
            }
            mates &= in;
        }
    }
    const float c2 = 1.44269504088896f / sqrtf(static_cast<float>(D));

    float4_t o[DB];
    float m_run, l_run;  // of the scores as they are, before their scale; the sums of a lane's own cells
#pragma unroll
    for (int db = 0; db < DB; db++) o[db] = float4_t{0.f, 0.f, 0.f, 0.f};
    m_run = -INFINITY;
    l_run = 0.f;

    // ---- the rows' own tiles, then the slice's: three of these on their way while one is multiplied, one barrier a tile ----
    __syncthreads();  // every wave holds its queries, the rows' cells are there; the last two stages are free
    for (int j = with_rows ? n_own : 2; j < min(n_tiles, 3); j++) ask(j);
    for (int j = 0; j < n_tiles; j++) {
        const char *kt = sm.ring[j & (kStages - 1)];
        uint32_t seen = 0xFF;  // which of the lane's eight cells its query row sees
        bool part;
        // a wave's loads complete in order: this tile's have landed when no more are out than those behind it
        if (j + 2 < n_tiles) wait_loads<2 * kPer>();
        else if (j + 1 < n_tiles) wait_loads<kPer>();
        else wait_loads<0>();
        asm volatile("s_barrier" ::: "memory");  // everyone's: this tile is whole, and the stage of the one before is free
        if (j + kAhead < n_tiles && j + kAhead >= n_own) ask(j + kAhead);
        if (j < n_own) {
            part = true;
            seen = static_cast<uint32_t>(mates >> (kTile * j + 8 * q)) & 0xFF;
        } else {
            const int c0 = tiles.at(t0 + j - n_own) * kTile;
            part = c0 + kTile > pos || (a.window > 0 && c0 + kTile > a.sinks && c0 < pos + rows - a.window);
            if (part) {
                seen = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int c = c0 + 8 * q + e;
                    seen |= c < pos && (a.window == 0 || c < a.sinks || c >= my_first) ? 1u << e : 0u;
                }
            }
        }
        if (!working) continue;
        const char *vt = kt + 2 * KI * kChunk;
        // operands come from LDS four reads ahead of the products that use them
        float4_t st[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, lo[2] = {st[0], st[0]};
        half8_t kb[2][4];
        const auto read_k = [&](half8_t(&to)[4], int g) {
#pragma unroll
            for (int e = 0; e < 4; e++) to[e] = *reinterpret_cast<const half8_t *>(kt + ((e & 1) * KI + 2 * g + (e >> 1)) * kChunk + lane * 16);
        };
        read_k(kb[0], 0);
#pragma unroll
        for (int g = 0; g < KI / 2; g++) {
            if (g + 1 < KI / 2) read_k(kb[(g + 1) & 1], g + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                st[e & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb[g & 1][e], qh[2 * g + (e >> 1)], st[e & 1], 0, 0, 0);
                lo[e & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb[g & 1][e], ql[2 * g + (e >> 1)], lo[e & 1], 0, 0, 0);
            }
        }
        float mx = -INFINITY, s[8];
#pragma unroll
        for (int e = 0; e < 8; e++) s[e] = st[e >> 2][e & 3] + lo[e >> 2][e & 3];
        if (part) {
#pragma unroll
            for (int e = 0; e < 8; e++) s[e] = seen >> e & 1 ? s[e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) mx = fmaxf(mx, s[e]);
        mx = max_over_q(mx);
        // the sums are rescaled a few times a slice instead of whenever some row's maximum moves
        const bool moves = mx * c2 > fmaf(m_run, c2, kSlack);
        if (__ballot(moves) != 0ull) {
            const float m_new = moves ? mx : m_run;
            const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_run - m_new) * c2);
            l_run *= alpha;
            m_run = m_new;
            float av[4];
#pragma unroll
            for (int e = 0; e < 4; e++) av[e] = __shfl(alpha, 4 * q + e, 64);
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[db][e] *= av[e];
        }
        const float m2 = fmaf(m_run == -INFINITY ? 0.f : m_run, c2, -kLift);
        float pv[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            pv[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c2, -m2));
            l_run += pv[e];
        }
        if (part) {
            // a value that is not finite would meet the weight 0 of rows that do not see it: such a tile is multiplied by hand
            uint32_t odd = 0;
#pragma unroll
            for (int db = 0; db < DB; db++) {
                const uint4 v = *reinterpret_cast<const uint4 *>(vt + db * kChunk + lane * 16);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; e++) odd |= ((w[e] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;  // an exponent of ones carries into the sign
            }
            if (__ballot(odd != 0) != 0ull) {
                float *p = sm.p[wave];
#pragma unroll 1
                for (int h = 0; h < 2; h++) {
                    if ((q >> 1) == h) {
#pragma unroll
                        for (int e = 0; e < 8; e++) p[n * (kTile / 2) + 8 * (q & 1) + e] = seen >> e & 1 ? pv[e] : -1.f;
                    }
                    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                    for (int i = 0; i < kTile / 2; i++) {
                        const int c = kTile / 2 * h + i;
                        float w[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] = p[(4 * q + e) * (kTile / 2) + i];
#pragma unroll
                        for (int db = 0; db < DB; db++) {
                            const float v = static_cast<float>(*reinterpret_cast<const _Float16 *>(vt + db * kChunk + (16 * (c >> 3) + n) * 16 + (c & 7) * 2));
#pragma unroll
                            for (int e = 0; e < 4; e++) o[db][e] = w[e] < 0.f ? o[db][e] : fmaf(w[e], v, o[db][e]);
                        }
                    }
                    __builtin_amdgcn_wave_barrier();
                }
                continue;
            }
        }
        // weights as two halves, the large one cut off and not rounded: the small one holds the rest either way, and is rounded to nearest, so that what
        // many cells lose cancels
        half8_t ph, pl;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const half2_t h = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(pv[e], pv[e + 1]));
            const half2_t r = {static_cast<_Float16>(fmaf(static_cast<float>(h[0]), -1.f, pv[e])), static_cast<_Float16>(fmaf(static_cast<float>(h[1]), -1.f, pv[e + 1]))};
            ph[e] = h[0]; ph[e + 1] = h[1];
            pl[e] = r[0]; pl[e + 1] = r[1];
        }
        half8_t vb[2][4];
#pragma unroll
        for (int e = 0; e < 4; e++) vb[0][e] = *reinterpret_cast<const half8_t *>(vt + e * kChunk + lane * 16);
#pragma unroll
        for (int g = 0; g < DB / 4; g++) {
            if (g + 1 < DB / 4) {
#pragma unroll
                for (int e = 0; e < 4; e++) vb[(g + 1) & 1][e] = *reinterpret_cast<const half8_t *>(vt + (4 * (g + 1) + e) * kChunk + lane * 16);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 4; e++) o[4 * g + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, vb[g & 1][e], o[4 * g + e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; e++) o[4 * g + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, vb[g & 1][e], o[4 * g + e], 0, 0, 0);
        }
    }
    if (!working) return;
    const float sum = sum_over_q(l_run);
    if (cut.all == 1) {
        float lr[4];
#pragma unroll
        for (int i = 0; i < 4; i++) lr[i] = __shfl(sum, 4 * q + i, 64);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = r0 + 4 * q + i, tr = over_rep(plan, r);
            if (r >= r_end) continue;
            float *dst = a.out + ((static_cast<size_t>(seq) * a.rows + tr) * a.n_head + kvh * rep + r - tr * rep) * D;
#pragma unroll
            for (int db = 0; db < DB; db++) dst[16 * db + n] = o[db][i] / lr[i];
        }
        return;
    }
    // the slice's record of each query row: unnormalised sums, and behind all records' the (max, sum)
    const size_t base = ((static_cast<size_t>(seq) * a.n_head_kv + kvh) * a.n_splits + split) * (static_cast<size_t>(a.rows) * rep);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = r0 + 4 * q + i;
        if (r >= r_end) continue;
        float *rec = a.partial + (base + r) * D;
#pragma unroll
        for (int db = 0; db < DB; db++) rec[16 * db + n] = o[db][i];
    }
    if (q == 0 && r0 + n < r_end) reinterpret_cast<float2 *>(a.partial + record_floats(a, D))[base + r0 + n] = make_float2(m_run, sum);
}

// The slices' records of a row and head joined, a lane four dims.  NW waves share the records of 256 / D rows' heads, each folds its share with
// all of a batch's loads on their way together, and the first wave folds their results.  grid: (ceil(rows * n_head * D / 256), n_seq).
template <int D, int NW, bool MANY>
__global__ __launch_bounds__(64 * NW) void tree_merge_kernel(shv_attn_tree_args a, Plan plan) {
    __shared__ float4_t sums[NW][64];
    __shared__ float2 of[NW][64];
    constexpr int kLanes = D / 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, seq = blockIdx.y;
    const int rep = a.n_head / a.n_head_kv;
    const int most = MANY ? *plan.len : 0, pos = a.pos ? a.pos[seq] : 0, rows = tree_rows(a.count, seq, a.rows);
    const uint32_t unit = blockIdx.x * (64 / kLanes) + lane / kLanes;
    const int row = static_cast<int>(unit / static_cast<uint32_t>(a.n_head)), head = static_cast<int>(unit) - row * a.n_head;
    const bool there = row < rows;
    if (!tree_fits(pos, rows, a.max_cells) || __ballot(there) == 0ull) return;
    const int tiles = Tiles(a, pos).all;
    const Cut<MANY> cut(a, tiles, most, plan);
    if (cut.all == 1) return;  // put straight out
    const float c2 = 1.44269504088896f / sqrtf(static_cast<float>(D));
    const int kvh = over_rep(plan, head), r = there ? row * rep + head - kvh * rep : 0;
    const size_t per = static_cast<size_t>(a.rows) * rep, base = (static_cast<size_t>(seq) * a.n_head_kv + kvh) * a.n_splits * per + r;
    const float4_t *from = reinterpret_cast<const float4_t *>(a.partial + base * D) + lane % kLanes;
    const float2 *from_of = reinterpret_cast<const float2 *>(a.partial + record_floats(a, D)) + base;
    constexpr int MB = 16;
    float4_t num = {0.f, 0.f, 0.f, 0.f};
    float den = 0.f, M = -INFINITY;
    const auto fold = [&](const float4_t &v, float2 ml) {
        if (ml.x == -INFINITY && ml.y == 0.f) return;  // (sees nothing; a sum of NaN stays)
        const float Mn = fmaxf(M, ml.x);
        const float shrink = __builtin_amdgcn_exp2f((M - Mn) * c2), w = __builtin_amdgcn_exp2f((ml.x - Mn) * c2);
        den = fmaf(den, shrink, w * ml.y);
#pragma unroll
        for (int e = 0; e < 4; e++) num[e] = fmaf(num[e], shrink, w * v[e]);
        M = Mn;
    };
    for (int s0 = wave; s0 < cut.all; s0 += NW * MB) {
        float4_t v[MB];
        float2 ml[MB];
#pragma unroll
        for (int u = 0; u < MB; u++) {
            const size_t s = s0 + NW * u < cut.all ? s0 + NW * u : s0;
            v[u] = from[s * per * kLanes];
            ml[u] = from_of[s * per];
        }
#pragma unroll
        for (int u = 0; u < MB; u++) asm volatile("" : "+v"(v[u]));  // asked for together, not each behind the one before's test
#pragma unroll
        for (int u = 0; u < MB; u++)
            if (s0 + NW * u < cut.all) fold(v[u], ml[u]);
    }
    if constexpr (NW > 1) {
        sums[wave][lane] = num;
        of[wave][lane] = make_float2(M, den);
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int k = 1; k < NW; k++) fold(sums[k][lane], of[k][lane]);
    }
    if (there) {
        float4_t y;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = num[e] / den;
        *(reinterpret_cast<float4_t *>(a.out + ((static_cast<size_t>(seq) * a.rows + row) * a.n_head + head) * D) + lane % kLanes) = y;
    }
}

template <int D, int W, bool MANY>
int launch_tree(shv_ctx *ctx, const shv_attn_tree_args &a) {
    const int rep = a.n_head / a.n_head_kv;
    constexpr int kBlocksPerUnit = D == 256 ? 1 : 2;
    Plan plan;
    plan.q_blocks = (a.rows * rep + 16 * W - 1) / (16 * W);
    // Beside them every sequence has a slice for its rows and, of several, one that is not full.  Each counts as a block for the whole call, though it ends soon: from
    // about ten wide sequences on part of the chip idles (64 rows behind 9000 cells each: eight sequences 201 us, ten 265, sixteen 494), and beside many
    // sequences a long one gets too few slices (sixteen of 64 rows, one behind 131000 cells and the others behind 500, 3050 us, where that one alone takes 274).
    plan.slots = ctx->prop.multiProcessorCount * kBlocksPerUnit / (a.n_head_kv * plan.q_blocks) - (MANY ? 2 : 1) * a.n_seq;
    if (plan.slots < 1) plan.slots = 1;
    plan.len = ctx->tree_len;
    // us with slices of 1 / 2 / 3 / 4 / 6 tiles at least: 2 rows behind 700 cells 12.4 / 12.6 / 13.2 / 14.0 / 16.2, 8 behind 3000 25.4 / 22.2 / 22.1 /
    // 22.9 / 24.0 (a slice more is a record more of every row to join); 32 behind 4000 (wide) - / 36.0 / 33.5 / 33.3 / 33.6.  Of 128 dims (rep 4) 12.0 / 12.2 / 12.0 /
    // 12.7 / 14.1, 18.0 / 18.1 / 17.9 / 18.0 / 18.9 and 32.8 / 32.7 / 31.1 / 31.9 / 32.0; of 64 (rep 8) 10.1 / 10.4 / 10.9 / 11.2 / 12.4, 17.2 / 15.1 / 15.3 / 16.1 / 17.4 and
    // 24.5 / 20.7 / 20.5 / 20.7 / 22.3
    plan.least = W == 4 ? kLeastNarrow : kLeastWide;
    plan.rep_magic = ((1u << 20) + rep - 1) / rep;
    static std::atomic<uint64_t> raised{0};  // by device
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (!(raised.load(std::memory_order_acquire) & bit)) {
        SHV_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&tree_attn_kernel<D, W, MANY>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(TreeSmem<D, W>))));
        raised.fetch_or(bit, std::memory_order_release);
    }
    // A sequence may have all the slices of the cache to itself, and those its share leaves over.  Of a wide call the last slice's records
    // (all there are, with one slice) are where the rows' operands lie: D floats of each record's D + 2.
    shv_attn_tree_args b = a;
    char *stage = nullptr;
    if (W == 8) {
        b.n_splits = a.n_splits > 1 ? a.n_splits - 1 : 1;
        const size_t records = static_cast<size_t>(a.n_seq) * a.rows * a.n_head * (D + 2) * (a.n_splits - 1);
        stage = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(a.partial + records) + 15) & ~static_cast<uintptr_t>(15));
        const int items = a.rows * (a.n_head + a.n_head_kv);
        SHV_LAUNCH(ctx, tree_prep_kernel<D>, dim3((items + 3) / 4, a.n_seq), dim3(256), 0, a, plan, stage);
    }
    if (b.n_splits > plan.slots + a.n_seq + 1) b.n_splits = plan.slots + a.n_seq + 1;  // no sequence is cut into more
    // slots + n_seq slices of the cache at most (call_len), and each sequence's of its rows
    const long long slices = b.n_splits == 1 ? a.n_seq : plan.slots + 2ll * a.n_seq;
    SHV_LAUNCH(ctx, (tree_attn_kernel<D, W, MANY>), dim3(static_cast<unsigned>((slices + 7) / 8 * 8 * plan.q_blocks), a.n_head_kv), dim3(64 * W), sizeof(TreeSmem<D, W>), b, plan, stage);
    if (b.n_splits > 1) {
        const int units = (a.rows * a.n_head * D + 255) / 256;
        const dim3 grid(units, a.n_seq);
        if (units * a.n_seq >= kMergeMany) SHV_LAUNCH(ctx, (tree_merge_kernel<D, 1, MANY>), grid, dim3(64), 0, b, plan);
        else if (units * a.n_seq >= kMergeSome) SHV_LAUNCH(ctx, (tree_merge_kernel<D, 8, MANY>), grid, dim3(512), 0, b, plan);
        else SHV_LAUNCH(ctx, (tree_merge_kernel<D, 4, MANY>), grid, dim3(256), 0, b, plan);
    }
    return SHV_OK;
}

template <int D>
int launch_tree(shv_ctx *ctx, const shv_attn_tree_args &a) {
    const bool narrow = a.rows * (a.n_head / a.n_head_kv) <= 64;
    if (a.n_seq == 1) return narrow ? launch_tree<D, 4, false>(ctx, a) : launch_tree<D, 8, false>(ctx, a);
    return narrow ? launch_tree<D, 4, true>(ctx, a) : launch_tree<D, 8, true>(ctx, a);
}

// grid: (rows, n_seq): one kept row; the cells' keys lie as they will, their values go to their places in a tile of 32 cells.  Bound by the
// launch and two trips to memory: 3.7 us of one sequence and of 24, whose 0.5 MB are nothing.
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
    SHV_REQUIRE(shv_aligned16(a.rope), "attn_tree: the rotary table must be 16-byte aligned");
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
