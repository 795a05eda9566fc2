// Full attention over a tree of drafted tokens, and the kept branch's cells into the cache.
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

// grid: (n_head_kv, rows, n_seq): the rows' cells.
__global__ __launch_bounds__(kBlock) void tree_cells_kernel(shv_attn_tree_args a) {
    __shared__ double kd[256];
    const int tid = threadIdx.x, lane = tid & 63;
    const int kvh = blockIdx.x, row = blockIdx.y, seq = blockIdx.z, d = a.head_dim;
    const int pos = a.pos ? a.pos[seq] : 0;
    const TreeRow t = tree_row(a.parent, a.count, seq, a.rows, lane);
    if (row >= t.n || !fits(pos, t.n, a.max_cells)) return;
    const int p = pos + __shfl(t.depth, row, 64);
    const float *qkv = a.qkv + (static_cast<size_t>(seq) * a.rows + row) * a.qkv_stride + static_cast<size_t>(a.n_head) * 2 * d + kvh * d;
    const size_t cell = ((static_cast<size_t>(seq) * a.rows + row) * a.n_head_kv + kvh) * d;
    if (tid < d) static_cast<__half *>(a.vcells)[cell + tid] = __float2half_rn(qkv[a.n_head_kv * d + tid]);
    if (tid >= 64) return;
    double ss = 0;
    for (int i = lane; i < d; i += 64) ss += static_cast<double>(qkv[i]) * qkv[i];
    const double sc = 1.0 / sqrt(wave_sum_f64(ss) / d + a.eps);
    for (int i = lane; i < d; i += 64) kd[i] = qkv[i] * sc * a.k_norm[i];
    __builtin_amdgcn_wave_barrier();
    const int half = a.rope_dims / 2;
    const float *table = a.rope + static_cast<size_t>(p) * a.rope_dims;
    for (int i = lane; i < d; i += 64) {
        double v = kd[i];
        if (i < half) v = kd[i] * table[i] - kd[i + half] * table[half + i];
        else if (i < a.rope_dims) v = kd[i - half] * table[i] + kd[i] * table[i - half];
        static_cast<__half *>(a.kcells)[cell + i] = cell_value(v);
    }
}

// grid: (n_head, rows, n_seq): one row and head, 256 cells at a time.
__global__ __launch_bounds__(kBlock) void tree_attn_kernel(shv_attn_tree_args a) {
    __shared__ float q[256];
    __shared__ float red[4];
    __shared__ float w[kBlock];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, d = a.head_dim;
    const int head = blockIdx.x, row = blockIdx.y, seq = blockIdx.z;
    const int rep = a.n_head / a.n_head_kv, kvh = head / rep;
    const int pos = a.pos ? a.pos[seq] : 0, slot = a.slot ? a.slot[seq] : seq;
    const TreeRow t = tree_row(a.parent, a.count, seq, a.rows, lane);
    if (row >= t.n || !fits(pos, t.n, a.max_cells)) return;
    const uint64_t anc = static_cast<uint64_t>(__shfl(static_cast<uint32_t>(t.ancestors >> 32), row, 64)) << 32 | __shfl(static_cast<uint32_t>(t.ancestors), row, 64);
    const int p = pos + __shfl(t.depth, row, 64);
    const float *src = a.qkv + (static_cast<size_t>(seq) * a.rows + row) * a.qkv_stride + static_cast<size_t>(head) * 2 * d;
    float ss = 0.f;
    for (int i = lane; i < d; i += 64) ss = fmaf(src[i], src[i], ss);
    const float sc = 1.f / sqrtf(wave_sum_all(ss) / d + a.eps);
    const int half = a.rope_dims / 2;
    const float *table = a.rope + static_cast<size_t>(p) * a.rope_dims;
    if (tid < d) {
        const auto x = [&](int i) { return src[i] * sc * a.q_norm[i]; };
        float v = x(tid);
        if (tid < half) v = x(tid) * table[tid] - x(tid + half) * table[half + tid];
        else if (tid < a.rope_dims) v = x(tid - half) * table[tid] + x(tid) * table[tid - half];
        q[tid] = v / sqrtf(static_cast<float>(d));
    }
    __syncthreads();
    const size_t kvw = static_cast<size_t>(a.n_head_kv) * d;
    const __half *kc = static_cast<const __half *>(a.kcache) + static_cast<size_t>(slot) * a.max_cells * kvw + kvh * d;
    const __half *vt = static_cast<const __half *>(a.vcache) + static_cast<size_t>(slot) * a.max_cells * kvw + static_cast<size_t>(kvh) * d * kTile;
    const __half *kt = static_cast<const __half *>(a.kcells) + static_cast<size_t>(seq) * a.rows * kvw + kvh * d;
    const __half *vx = static_cast<const __half *>(a.vcells) + static_cast<size_t>(seq) * a.rows * kvw + kvh * d;
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int c0 = 0; c0 < pos + t.n; c0 += kBlock) {
        const int c = c0 + tid;
        const int depth = __shfl(t.depth, (c - pos) & 63, 64);
        bool see = false;
        float s = -INFINITY;
        if (c < pos + t.n) {
            const int at = c < pos ? c : pos + depth;
            see = (c < pos || ((anc >> (c - pos)) & 1)) && (a.window == 0 || at < a.sinks || p - at < a.window);
            if (see) {
                const __half *k = c < pos ? kc + c * kvw : kt + (c - pos) * kvw;
                s = 0.f;
                for (int i = 0; i < d; i++) s = fmaf(q[i], __half2float(k[i]), s);
            }
        }
        const float mw = wave_max_all(s);
        __syncthreads();
        if (lane == 0) red[wave] = mw;
        __syncthreads();
        const float m_new = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float use = m_new == -INFINITY ? 0.f : m_new;
        const float e = see ? expf(s - use) : 0.f;
        w[tid] = see ? e : -1.f;
        const float sum = wave_sum_all(e);
        __syncthreads();
        if (lane == 0) red[wave] = sum;
        __syncthreads();
        const float fall = expf(m - use);
        l = l * fall + (red[0] + red[1] + red[2] + red[3]);
        m = m_new;
        if (tid < d) {
            o *= fall;
            for (int i = 0; i < kBlock; i++) {
                if (w[i] < 0.f) continue;  // a cell the row does not see may hold anything
                const int cc = c0 + i;
                const __half v = cc < pos ? vt[static_cast<size_t>(cc / kTile) * kvw * kTile + tid * kTile + cc % kTile] : vx[(cc - pos) * kvw + tid];
                o = fmaf(w[i], __half2float(v), o);
            }
        }
    }
    if (tid < d) a.out[((static_cast<size_t>(seq) * a.rows + row) * a.n_head + head) * d + tid] = o / l;
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
    SHV_REQUIRE(a.rope_dims >= 0 && a.rope_dims <= a.head_dim && a.rope_dims % 2 == 0, "attn_tree: rope_dims %d; even, up to head_dim %d", a.rope_dims, a.head_dim);
    SHV_REQUIRE(a.rope || a.rope_dims == 0, "attn_tree: NULL rotary table");
    SHV_REQUIRE(a.max_cells >= kTile && a.max_cells % kTile == 0, "attn_tree: max_cells %d; a multiple of %d", a.max_cells, kTile);
    SHV_REQUIRE(a.qkv_stride >= (a.n_head + a.n_head_kv) * 2 * a.head_dim && a.qkv_stride % 4 == 0, "attn_tree: qkv_stride %d", a.qkv_stride);
    SHV_REQUIRE(a.n_splits >= 1 && a.n_splits <= kMaxSplits, "attn_tree: %d slices; 1..%d", a.n_splits, kMaxSplits);
    SHV_REQUIRE(a.window >= 0 && a.sinks >= 0, "attn_tree: window %d, sinks %d", a.window, a.sinks);
    SHV_REQUIRE(shv_aligned16(a.qkv) && shv_aligned16(a.kcache) && shv_aligned16(a.vcache) && shv_aligned16(a.kcells) && shv_aligned16(a.vcells) &&
                    shv_aligned16(a.q_norm) && shv_aligned16(a.k_norm) && shv_aligned16(a.out) && shv_aligned16(a.partial),
                "attn_tree: qkv, norms, caches, cells, partial and out must be 16-byte aligned");
    SHV_LAUNCH(ctx, tree_cells_kernel, dim3(a.n_head_kv, a.rows, a.n_seq), dim3(kBlock), 0, a);
    SHV_LAUNCH(ctx, tree_attn_kernel, dim3(a.n_head, a.rows, a.n_seq), dim3(kBlock), 0, a);
    return SHV_OK;
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
